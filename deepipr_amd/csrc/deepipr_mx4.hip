// deepipr_mx4.hip -- translation unit of libdeepipr_hip.so: matrices in microscaled 4-bit floating point ("MX4") and their products.
//
// The format (the open MX specification's MXFP4): 32 neighbouring values of a row share a power of two X = 2^(code - 127), held in one
// byte (E8M0; 255 = not a number); each value is a 4-bit float E2M1 -- sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- times X.
// Quantising: code = max(0, biased exponent of max|block| - 2), so max|block| / X lies in [4, 8); values are rounded to the nearest code,
// ties to the even one, and saturate at 6.  Division by X is exact, so every value's code is a function of its block alone.
// A block that holds a NaN or an infinity gets code 255: all of it reads as NaN.
//
// In memory a quantised matrix of R rows and K columns, Kp = K rounded up to 128:
//   codes   [Kp / 128][R][64] bytes: 128 columns of a row are 64 bytes, neighbouring rows' neighbours in memory (a tile of a product
//           is then whole cache lines however few columns it takes); the value with the lower index in the low half byte; the columns
//           behind K are zero;
//   scales  [Kp / 128][ceil(R / 64)][64] words of 4 bytes: word 32 (b % 2) + r % 32 of a 64-row group holds the scales of the blocks b % 2
//           and 2 + b % 2 (of the four of these 128 columns) of the rows r % 32 and 32 + r % 32; byte 2 (b / 2) + r / 32.  That is the order
//           in which the lanes of v_mfma_scale_f32_32x32x64_f8f6f4 take them: one coalesced 256-byte load serves 64 rows x 128 columns.
//
// Times in this file, unless they say otherwise: launches back to back in a replayed graph on the same operands (what fits stays in the
// 256 MB cache).  A pass with other work around it takes longer: 1 x 4096 x 9216 6.8 us where the graph gives 5.6, 253 x 4096 x 9216 15.6 / 13.6, the
// codes of 8192 x 8192 bf16 40 / 26, of 200 704 x 1021 141 / 113 to 124.
#include <cmath>

#include "deepipr_host.h"

namespace {

enum { F32 = DEEPIPR_F32, BF16 = DEEPIPR_BF16, F16 = DEEPIPR_F16 };
constexpr int kThreads = 256;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

__host__ __device__ inline long long round_up(long long v, long long m) { return (v + m - 1) / m * m; }
__host__ __device__ inline long long row_groups(long long rows) { return (rows + 63) / 64; }

// ------------------------------------------------------------------------------------------------------------ element types
__device__ __forceinline__ float bf16_to_f32(unsigned h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ unsigned f32_to_bf16(float f) {                // nearest, ties to even; NaN stays NaN
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ float f16_to_f32(unsigned h) {
    const unsigned short s = static_cast<unsigned short>(h);
    _Float16 v;
    __builtin_memcpy(&v, &s, 2);
    return static_cast<float>(v);
}
__device__ __forceinline__ unsigned f32_to_f16(float f) {
    const _Float16 v = static_cast<_Float16>(f);
    unsigned short h;
    __builtin_memcpy(&h, &v, 2);
    return h;
}
template <int T> __device__ __forceinline__ float load1(const void *p, long long i) {
    if (T == F32) return static_cast<const float *>(p)[i];
    const unsigned h = static_cast<const unsigned short *>(p)[i];
    return T == BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
template <int T> __device__ __forceinline__ void store1(void *p, long long i, float v) {
    if (T == F32) static_cast<float *>(p)[i] = v;
    else static_cast<unsigned short *>(p)[i] = static_cast<unsigned short>(T == BF16 ? f32_to_bf16(v) : f32_to_f16(v));
}
// Four neighbours at once, on whatever address their type allows (the card takes vector accesses at any element); gfx950 converts pairs,
// to nearest, ties to even.
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef bf16x4 bf16x4_any __attribute__((aligned(2)));
typedef f16x4 f16x4_any __attribute__((aligned(2)));
template <int T> __device__ __forceinline__ void store4(void *p, f32x4 v) {
    if (T == F32) *static_cast<f32x4_any *>(p) = v;
    else if (T == BF16) *static_cast<bf16x4_any *>(p) = __builtin_convertvector(v, bf16x4);
    else *static_cast<f16x4_any *>(p) = __builtin_convertvector(v, f16x4);
}
// 16 bytes of elements (the caller checked the alignment)
template <int T> __device__ __forceinline__ u32x4 load16(const void *p, long long i) {
    return *reinterpret_cast<const u32x4 *>(static_cast<const char *>(p) + i * (T == F32 ? 4 : 2));
}
template <int T> __device__ __forceinline__ void *element(void *p, long long i) { return static_cast<char *>(p) + i * (T == F32 ? 4 : 2); }

// ------------------------------------------------------------------------------------------------------- one block of 32 values
// `top`: the largest magnitude's bits (NaN and infinity compare above every finite value as integers).  -> the scale byte
__device__ __forceinline__ unsigned scale_code(unsigned top) {
    const int e = static_cast<int>(top >> 23);
    return e == 255 ? 255u : static_cast<unsigned>(max(e - 2, 0));
}
// 1 / X as a float: 2^(127 - code), code 0 .. 252: always a normal number
__device__ __forceinline__ float inverse_scale(unsigned code) { return __uint_as_float((254u - code) << 23); }
__device__ __forceinline__ float scale_value(unsigned code) {
    if (code == 255u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(code ? code << 23 : 0x00400000u);              // 2^-127 is a subnormal float
}
// eight values, already divided by X, as eight 4-bit codes
__device__ __forceinline__ unsigned pack8(const float *v) {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
    return w;
}
// -> the block's 16 bytes of codes; `code`: its scale byte
__device__ __forceinline__ u32x4 quantise32(float *v, unsigned &code) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    code = scale_code(top);
    if (code == 255u) return u32x4{0u, 0u, 0u, 0u};
    const float inv = inverse_scale(code);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= inv;
    return u32x4{pack8(v), pack8(v + 8), pack8(v + 16), pack8(v + 24)};
}

// ------------------------------------------------------------------------------------------------------------------- quantise
// One pass over x [R][C] (row stride in elements, columns contiguous): ROW writes x with blocks along its rows, COL writes x's
// transpose with blocks along x's columns, SUM the sums of 64 rows of every column (the bias gradient).
// A workgroup takes 64 x 128 values through LDS as floats; every thread then owns one block of 32 in each direction.
// Bound by bytes: each value is read from HBM once for both directions.
constexpr int kQR = 64, kQC = 128, kQP = kQC + 4;        // pitch: 16-byte rows shifted by four banks each

struct Matrix {
    const void *x;
    long long R, C, stride;
    int vec;                                             // rows start on 16-byte boundaries
    unsigned char *row_codes, *col_codes;
    unsigned *row_scales, *col_scales;
    float *sums;
};
// `first` workgroups take matrix A, the others B (a layer's input and weight in one launch)
template <int T, bool ROW, bool COL, bool SUM>
__global__ __launch_bounds__(kThreads) void k_mx4_quantise(const Matrix A, const Matrix B, unsigned first) {
    const Matrix &m = blockIdx.x < first ? A : B;
    int id = static_cast<int>(blockIdx.x < first ? blockIdx.x : blockIdx.x - first);
    // Tiles that end inside a cache line of x share it with their neighbours: those meet in one XCD's L2 (200 704 x 1016 bf16 137 -> 105 us);
    // whole lines are better off spread (8192 x 8192 bf16 25 us, 30 in that order).
    if (m.C % kQC) id = dipr_xcd_contiguous(id, static_cast<int>(blockIdx.x < first ? first : gridDim.x - first));
    const void *__restrict__ x = m.x;
    const long long R = m.R, C = m.C, stride = m.stride;
    const int vec = m.vec;
    unsigned char *__restrict__ row_codes = m.row_codes, *__restrict__ col_codes = m.col_codes;
    unsigned *__restrict__ row_scales = m.row_scales, *__restrict__ col_scales = m.col_scales;
    float *__restrict__ sums = m.sums;
    __shared__ float s[kQR * kQP];
    __shared__ unsigned char sc[2][256];
    const long long tiles_c = (C + kQC - 1) / kQC;
    const long long r0 = id / tiles_c * kQR, c0 = id % tiles_c * kQC;
    const int tid = threadIdx.x;
    constexpr int V = T == F32 ? 4 : 8, PER = kQC / V, LOADS = kQR * PER / kThreads;      // 16-byte pieces
    const auto put = [&](int i, u32x4 q) {
        float *d = s + i / PER * kQP + i % PER * V;
        if (T == F32) {
            *reinterpret_cast<u32x4 *>(d) = q;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                f32x4 f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f[2 * e] = T == BF16 ? __uint_as_float(q[k + e] << 16) : f16_to_f32(q[k + e] & 0xffffu);
                    f[2 * e + 1] = T == BF16 ? __uint_as_float(q[k + e] & 0xffff0000u) : f16_to_f32(q[k + e] >> 16);
                }
                *reinterpret_cast<f32x4 *>(d + 2 * k) = f;
            }
        }
    };
    if (vec && r0 + kQR <= R && c0 + kQC <= C) {
        u32x4 q[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int i = j * kThreads + tid;
            q[j] = load16<T>(x, (r0 + i / PER) * stride + c0 + i % PER * V);
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) put(j * kThreads + tid, q[j]);
    } else if (vec && C % V == 0) {                                      // the last rows or columns, in whole pieces
        u32x4 q[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int i = j * kThreads + tid;
            const long long r = r0 + i / PER, c = c0 + i % PER * V;
            q[j] = r < R && c < C ? load16<T>(x, r * stride + c) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) put(j * kThreads + tid, q[j]);
    } else if (T == F32) {
        // rows off the 16-byte grid (a wave's single elements are contiguous whatever the alignment: 200 704 x 1021 takes 179 us this way
        // and 293 by unaligned 16-byte loads), and the matrix's last rows and columns
        const int c = tid & 127, h = tid >> 7;
        const long long left = c0 + c < C ? R - r0 - h : 0;              // rows h, h + 2, ... that exist
        float e[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) e[j] = 2 * j < left ? load1<T>(x, (r0 + h + 2 * j) * stride + c0 + c) : 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) s[(h + 2 * j) * kQP + c] = e[j];
    } else if (r0 + kQR <= R && c0 + kQC <= C) {
        // rows of 16-bit elements off the grid: eight of them out of the two aligned pieces that hold them (200 704 x 1021 bf16 124 us, 151 by
        // aligned words).  Both pieces hold an element of the row: nothing outside its last aligned piece is read.
        u32x4 lo[LOADS], hi[LOADS];
        const auto at = [&](int j) {
            const int i = j * kThreads + tid;
            return static_cast<const char *>(x) + ((r0 + i / PER) * stride + c0 + i % PER * V) * 2;
        };
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int by = static_cast<int>(reinterpret_cast<uintptr_t>(at(j)) & 15);        // (pointers stay pointers: global loads)
            lo[j] = *reinterpret_cast<const u32x4 *>(at(j) - by);
            hi[j] = *reinterpret_cast<const u32x4 *>(at(j) + (by ? 16 - by : 0));
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int by = static_cast<int>(reinterpret_cast<uintptr_t>(at(j)) >> 1 & 7);   // elements
            u32x4 l = lo[j], h = hi[j];
            if (by & 2) l = u32x4{l.y, l.z, l.w, h.x}, h = u32x4{h.y, h.z, h.w, h.w};
            if (by & 4) l = u32x4{l.z, l.w, h.x, h.y}, h.x = h.z;
            if (by & 1) l = u32x4{l.x >> 16 | l.y << 16, l.y >> 16 | l.z << 16, l.z >> 16 | l.w << 16, l.w >> 16 | h.x << 16};
            put(j * kThreads + tid, l);
        }
    } else {
        // the last rows and columns, two elements to an aligned word (loads of single ones are four times slower); a row that starts in the middle
        // of a word is off by one: its first and last words hold one element of it, and what else they hold is not used
        const int lane = tid & 63, row0 = (tid >> 6) * 16;
        const auto row_at = [&](int r) { return static_cast<const char *>(x) + ((r0 + r) * stride + c0) * 2; };
        const auto odd_at = [&](int r) { return static_cast<int>(reinterpret_cast<uintptr_t>(row_at(r)) >> 1 & 1); };
        const auto value = [&](unsigned h) { return T == BF16 ? bf16_to_f32(h) : f16_to_f32(h); };
        unsigned w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int odd = odd_at(row0 + j);
            w[j] = r0 + row0 + j < R && c0 + 2 * lane - odd < C ? *reinterpret_cast<const unsigned *>(row_at(row0 + j) - 2 * odd + 4 * lane) : 0u;
            if (c0 + 2 * lane - odd + 1 >= C) w[j] &= 0xffffu;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int odd = odd_at(row0 + j);
            float *d = s + (row0 + j) * kQP + 2 * lane - odd;
            if (odd == 0) {
                *reinterpret_cast<f32x2 *>(d) = f32x2{value(w[j] & 0xffffu), value(w[j] >> 16)};
            } else {
                if (lane) d[0] = value(w[j] & 0xffffu);
                d[1] = value(w[j] >> 16);
            }
        }
        if (tid < kQR && odd_at(tid))                         // the 128th column of a row that is off by one
            s[tid * kQP + 127] = r0 + tid < R && c0 + 127 < C ? load1<T>(x, (r0 + tid) * stride + c0 + 127) : 0.0f;
    }
    __syncthreads();
    float v[32];
    if (ROW) {
        const int r = tid >> 2, b = tid & 3;
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<f32x4 *>(v + 4 * k) = *reinterpret_cast<const f32x4 *>(s + r * kQP + b * 32 + 4 * k);
        unsigned code;
        const u32x4 q = quantise32(v, code);
        if (r0 + r < R) *reinterpret_cast<u32x4 *>(row_codes + (c0 / 128 * R + r0 + r) * 64 + b * 16) = q;
        sc[0][((b & 1) * 32 + (r & 31)) * 4 + (b >> 1) * 2 + (r >> 5)] = static_cast<unsigned char>(code);
    }
    if (COL) {
        const int c = tid & 127, h = tid >> 7;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
            v[k] = s[(h * 32 + k) * kQP + c];
            if (SUM) sum += v[k];
        }
        unsigned code;
        const u32x4 q = quantise32(v, code);
        if (c0 + c < C) *reinterpret_cast<u32x4 *>(col_codes + (r0 / 128 * C + c0 + c) * 64 + (r0 / 64 & 1) * 32 + h * 16) = q;
        sc[1][(c >> 6) * 128 + (h * 32 + (c & 31)) * 2 + (c >> 5 & 1)] = static_cast<unsigned char>(code);
        if (SUM) {
            __syncthreads();                             // the tile has been read: its first row takes the upper half's sums
            if (h == 1) s[c] = sum;
            __syncthreads();
            if (h == 0 && c0 + c < C) sums[r0 / kQR * C + c0 + c] = sum + s[c];
        }
    }
    __syncthreads();
    // (with the column direction the grid covers the rows' padding too: row groups that do not exist there)
    if (ROW && tid < 64 && r0 < R) row_scales[(c0 / 128 * row_groups(R) + r0 / 64) * 64 + tid] = reinterpret_cast<const unsigned *>(sc[0])[tid];
    if (COL && tid < 128) {                              // these 64 rows are one half (two of four blocks) of every word
        const long long rg = c0 / 64 + (tid >> 6);
        if (rg < row_groups(C))
            reinterpret_cast<unsigned short *>(col_scales)[((r0 / 128 * row_groups(C) + rg) * 64 + (tid & 63)) * 2 + (r0 / 64 & 1)] =
                reinterpret_cast<const unsigned short *>(sc[1])[tid];
    }
}

// Adds up groups of 128 tiles' sums of each column, in 64 bits: eight threads a column, each every eighth tile in order, then the eight in
// order.  The first pass reads sums [tiles][C] in 32 bits.  With more than one group a group's sum takes the place of its first two rows
// (low and high word; a group has at least two: the tiles come in pairs), which only this workgroup has read, and the next pass adds up
// those: its item t lies in rows t * step and t * step + 1.  The last pass rounds once, to `out`.
constexpr int kSumTiles = 128;
template <bool FIRST>
__global__ __launch_bounds__(kThreads) void k_mx4_colsum(float *sums, long long items, long long step, long long C, float *out) {
    __shared__ double red[8][32];
    const long long t0 = static_cast<long long>(blockIdx.y) * kSumTiles;
    const int n = static_cast<int>(min(items - t0, static_cast<long long>(kSumTiles)));
    const int col = threadIdx.x & 31, part = threadIdx.x >> 5;
    const long long c = static_cast<long long>(blockIdx.x) * 32 + col;
    float *at = sums + t0 * step * C + c;
    double v = 0.0;
    if (c < C) {
#pragma unroll 4
        for (int t = part; t < n; t += 8) {
            const float *p = at + t * step * C;
            v += FIRST ? static_cast<double>(p[0]) : __hiloint2double(__float_as_int(p[C]), __float_as_int(p[0]));
        }
    }
    red[part][col] = v;
    __syncthreads();
    if (part == 0 && c < C) {
#pragma unroll
        for (int i = 1; i < 8; ++i) v += red[i][col];
        if (gridDim.y == 1) {
            out[c] = static_cast<float>(v);
        } else {
            at[0] = __int_as_float(__double2loint(v));
            at[C] = __int_as_float(__double2hiint(v));
        }
    }
}

// ----------------------------------------------------------------------------------------------------------------- dequantise
// The matrix [R][K] of values, or its transpose [K][R].
__device__ __forceinline__ unsigned scale_at(const unsigned *scales, long long rows, long long r, long long b) {
    const unsigned w = scales[((b >> 2) * row_groups(rows) + (r >> 6)) * 64 + (b & 1) * 32 + (r & 31)];
    return w >> (((b >> 1 & 1) * 2 + (r >> 5 & 1)) * 8) & 0xffu;
}
__device__ __forceinline__ void decode8(unsigned w, float x, float *v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a.x * x; v[1] = a.y * x; v[2] = b.x * x; v[3] = b.y * x;
    v[4] = c.x * x; v[5] = c.y * x; v[6] = d.x * x; v[7] = d.y * x;
}

// a workgroup takes 64 rows x 128 columns; 32 lanes write one row's 128 values
template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_dequantise(const unsigned char *__restrict__ codes, const unsigned *__restrict__ scales,
                                                             long long R, long long K, void *__restrict__ out) {
    const long long panels = (K + 127) / 128;
    const int id = dipr_xcd_contiguous(blockIdx.x, gridDim.x);           // neighbours share cache lines of `out` where rows are off the grid
    const long long r0 = id / panels * 64, p = id % panels;
    const int c = (threadIdx.x & 31) * 4;
    const long long k = p * 128 + c;
    if (k >= K) return;
#pragma unroll 4
    for (int i = threadIdx.x >> 5; i < 64; i += kThreads / 32) {
        const long long r = r0 + i;
        if (r >= R) break;
        const unsigned w = *reinterpret_cast<const unsigned short *>(codes + (p * R + r) * 64 + c / 2);
        const float x = scale_value(scale_at(scales, R, r, p * 4 + (c >> 5)));
        const f32x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
        const f32x4 v = f32x4{lo.x, lo.y, hi.x, hi.y} * x;
        if (k + 4 <= K) {
            store4<T>(element<T>(out, r * K + k), v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k + j < K) store1<T>(out, r * K + k + j, v[j]);
        }
    }
}

// out [K][R]: a workgroup takes 64 rows x 128 columns of the matrix, a thread one block; 64 values of each output row go out together
template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_dequantise_t(const unsigned char *__restrict__ codes, const unsigned *__restrict__ scales,
                                                               long long R, long long K, void *__restrict__ out) {
    constexpr int P = 68;
    __shared__ __align__(16) float s[128 * P];
    const long long tiles_r = (R + 63) / 64;
    const int id = dipr_xcd_contiguous(blockIdx.x, gridDim.x);
    const long long r0 = id % tiles_r * 64, k0 = id / tiles_r * 128;
    const int r = threadIdx.x & 63, b = threadIdx.x >> 6;
    if (r0 + r < R) {                                    // columns behind K lie in the padding: zero codes
        const u32x4 q = *reinterpret_cast<const u32x4 *>(codes + (k0 / 128 * R + r0 + r) * 64 + b * 16);
        const float x = scale_value(scale_at(scales, R, r0 + r, k0 / 32 + b));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float v[8];
            decode8(q[w], x, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[(b * 32 + w * 8 + j) * P + r] = v[j];
        }
    }
    __syncthreads();
    const int c = threadIdx.x & 15;                      // four neighbouring rows of the matrix
#pragma unroll 4
    for (int k = threadIdx.x >> 4; k < 128; k += kThreads / 16) {
        if (k0 + k >= K) break;
        const f32x4 v = *reinterpret_cast<const f32x4 *>(s + k * P + c * 4);
        const long long at = (k0 + k) * R + r0 + c * 4;
        if (r0 + c * 4 + 4 <= R) {
            store4<T>(element<T>(out, at), v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r0 + c * 4 + j < R) store1<T>(out, at + j, v[j]);
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------- product
// out[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]), A [M][K] and B [N][K] quantised.  v_mfma_scale_f32_32x32x64_f8f6f4: lane l gives 32
// codes of row l % 32 (block l / 32 of 64 columns) and that block's scale, a byte of a word; B is the instruction's first operand, so
// that a lane holds four times four neighbouring n of one m.  Products and sums in 32 bits.
// (Measured: one wave per SIMD issues these at 9.1 PFLOP/s over the card, v_mfma_scale_f32_16x16x128_f8f6f4 at 5.2.)
__device__ __forceinline__ float bias_at(const void *bias, int type, long long n) {
    return type == F32 ? load1<F32>(bias, n) : type == BF16 ? load1<BF16>(bias, n) : load1<F16>(bias, n);
}

template <int SA, int SB>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, unsigned sa, unsigned sb) {
    const i32x8 av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
    const i32x8 bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, SA, static_cast<int>(sa), SB, static_cast<int>(sb));
}

// The outputs of a wave, TM x TN tiles of 32 x 32 (acc[n tile][m tile]; a lane holds n = 8 q + 4 (lane / 32) .. + 3 of m = lane % 32), to
// rows m0 .. of `out`, 32 rows at a time through `strip` (32 rows of 32 TN + 4 floats of this wave's own): whole cache lines per row.
template <int T, int TM, int TN>
__device__ __forceinline__ void store_tiles(const f32x16 (&acc)[TN][TM], float *strip, const void *bias, int bias_type, long long m0, long long n0,
                                            long long M, long long N, void *out) {
    constexpr int P = 32 * TN + 4, PER = 8 * TN, STEP = 64 / PER;          // lanes per row (a lane keeps its columns), rows per pass
    const int lane = threadIdx.x & 63, row = lane / PER;
    const long long n = n0 + lane % PER * 4;
    f32x4 add = {};
    if (bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < N) add[j] = bias_at(bias, bias_type, n + j);
    }
    const bool whole = m0 + 32 * TM <= M && n0 + 32 * TN <= N;      // uniform: nearly every tile of a large product
    const float *from = strip + row * P + lane % PER * 4;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4 *>(strip + (lane & 31) * P + i * 32 + q * 8 + (lane >> 5) * 4) =
                    f32x4{acc[i][t][4 * q], acc[i][t][4 * q + 1], acc[i][t][4 * q + 2], acc[i][t][4 * q + 3]};
        if (whole) {
            char *to = static_cast<char *>(element<T>(out, (m0 + t * 32 + row) * N + n));
            const long long step = N * (STEP * (T == F32 ? 4 : 2));
#pragma unroll
            for (int r = 0; r < 32; r += STEP) {
                store4<T>(to, *reinterpret_cast<const f32x4 *>(from + r * P) + add);
                to += step;
            }
        } else {
            for (int r = 0; r < 32; r += STEP) {
                const long long m = m0 + t * 32 + row + r;
                const f32x4 v = *reinterpret_cast<const f32x4 *>(from + r * P) + add;
                if (m >= M) continue;
                if (n + 4 <= N) {
                    store4<T>(element<T>(out, m * N + n), v);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (n + j < N) store1<T>(out, m * N + n + j, v[j]);
                }
            }
        }
    }
}

struct Product {
    const unsigned char *a, *b;                          // [kt][M][64], [kt][N][64]
    const unsigned *sa, *sb;
    const void *bias;
    int bias_type;
    long long M, N;                                      // of the operands in memory
    long long first, last;                               // rows first .. last - 1 of the output (first a multiple of 64)
    int kt, splits;                                      // splits > 1: out is float [splits][M][N], split i adds up its share of the steps
    void *out;
    long long K;                                         // columns
    const void *x;                                       // a in its own type instead of a / sa (k_mx4_gemm_rows with X >= 0)
    long long x_stride;
    int x_vec;                                           // its rows start on 16-byte boundaries
};

// 32 values of a row from column k on, zero behind K
template <int X> __device__ __forceinline__ void load_block(const void *x, long long at, long long k, long long K, int vec, float *v) {
    if (vec && k + 32 <= K) {
#pragma unroll
        for (int i = 0; i < 32; i += X == F32 ? 4 : 8) {
            const u32x4 q = load16<X>(x, at + i);
            if (X == F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] = __uint_as_float(q[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[(i + 2 * j) & 31] = X == BF16 ? __uint_as_float(q[j] << 16) : f16_to_f32(q[j] & 0xffffu);
                    v[(i + 2 * j + 1) & 31] = X == BF16 ? __uint_as_float(q[j] & 0xffff0000u) : f16_to_f32(q[j] >> 16);
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = k + i < K ? load1<X>(x, at + i) : 0.0f;
    }
}

// Few rows or small tiles: a workgroup of eight waves takes 16 MT rows of a and 16 NT of b; wave i the steps i, i + 8, ... of the columns, a few
// of them on their way at once, straight to registers; the waves' sums are added through LDS in wave order.
// v_mfma_scale_f32_16x16x128_f8f6f4: 16 lanes give one of the four blocks of 16 rows each.
//   NT = 1, all of a in one workgroup (at most 64 rows): bound by reading b once; with 16 rows of b a workgroup, 4096 rows fill 256 CUs and all
//           of b is asked for at once.
//   NT = 2, 4 (64 x 32 and 64 x 64 outputs): up to a few hundred rows, where 128 x 128 tiles would leave CUs free or need the columns shared
//           out over workgroups and a second launch to add up.  Bound by waiting for the L2s: at 253 x 4096 x 9216 every operand goes to the CUs once a
//           tile, 161 MB (counted: 1.26 M reads of 128 bytes, 81 % of them hits) in 13.6 us; the matrix cores are busy 14 % of that.  Measured in us, this /
//           the larger tiles at their best: 253 x 4096 x 9216 13.6 / 21.9, 256 x 1000 x 2048 4.4 / 9.9, 128 x 4096 x 4096 6.2 / 12.1, 1000^3
//           4.7 / 8.0; 512 x 4096 x 4096 14.2 / 13.4, 2048^3 18.4 / 10.4.  Each step's place refilled at once instead of two steps
//           together: 13.6 / 15.1, and 14.9 / 22.8 with b out of HBM.
// X >= 0 (MT = NT = 1): a comes in its own type X and the workgroup first quantises all of it into LDS, one block a thread and turn, while its
// first fetches of b are on their way.  Every workgroup does so again, but a launch is saved (3 us of the host's time, 2 of the card's).
// Measured (us, fused / apart): 1 x 4096 x 9216 fp32 5.5 / 8.6, 4 x: 8.3 / 8.5, 8 x 4096 x 4096 7.0 / 6.9; 16 x 4096 x 4096 bf16 6.9 / 8.0,
// fp32 10.9 / 7.0: up to 4096 bytes x blocks.
constexpr int kFusedBlocks = 2048;
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, unsigned sa, int ha, unsigned sb, int hb) {
    const i32x8 av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
    const i32x8 bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
    const int x = static_cast<int>(sa), y = static_cast<int>(sb);           // the halves' bytes (ha, hb are constants of the unrolled loops)
    if (ha == 0 && hb == 0) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, x, 0, y);
    if (ha == 0) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, x, 1, y);
    if (hb == 0) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 1, x, 0, y);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 1, x, 1, y);
}
// Out of word l of a 64-row group in lane l: [i] = the words of the rows 16 i + l % 16 (and 32 more) for all four blocks
template <int TILES> __device__ __forceinline__ u32x2 words(unsigned w, int shift) {
    if (TILES == 1) return u32x2{w >> shift, 0};
    const u32x2 v = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return u32x2{v.x >> shift, v.y >> shift};
}
template <int T, int MT, int NT, int X>
__global__ __launch_bounds__(512) void k_mx4_gemm_rows(const Product A, const Product B, unsigned first) {
    constexpr int U = NT == 1 ? 4 : 2;
    __shared__ f32x4 red[8][MT * NT][64];
    __shared__ u32x4 codes[X >= 0 ? kFusedBlocks : 1];
    __shared__ unsigned char scales[X >= 0 ? kFusedBlocks : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool of_a = blockIdx.x < first;
    const Product &P = of_a ? A : B;
    // neighbours share their rows of b: with NT > 1 they meet in one XCD's L2
    const int index = of_a ? blockIdx.x : blockIdx.x - first, count = of_a ? first : gridDim.x - first;
    const int id = NT == 1 ? index : dipr_xcd_contiguous(index, count);
    const int tiles_m = static_cast<int>((P.last - P.first + 16 * MT - 1) / (16 * MT));
    const long long n0 = static_cast<long long>(id / tiles_m) * (16 * NT), m0 = P.first + id % tiles_m * (16 * MT);
    const int r = lane & 15, blk = (lane >> 4 & 1) * 2 + (lane >> 5);      // (any order of the four blocks will do that a and b share)
    // A single tile's lane loads the scale word of its own row and block.  Two or four tiles are half of or a whole 64-row group: lane l loads
    // the group's word l, and a swap of rows of 16 lanes hands every tile its words.
    const unsigned char *pb[NT], *pa[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) pb[i] = P.b + min(n0 + i * 16 + r, P.N - 1) * 64 + blk * 16;
    const auto word_of = [&](long long row, int tiles) {
        return row / 64 * 64 + (tiles > 1 ? lane : (blk & 1) * 32 + static_cast<int>((row + r) & 31));
    };
    const auto shift_of = [&](long long row) { return (blk >> 1) * 16 + static_cast<int>(row >> 5 & 1) * 8; };
    const unsigned *qb = P.sb + word_of(n0, NT), *qa = nullptr;
    const int hb = shift_of(n0);
    int ha = 0;
    if (X < 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) pa[t] = P.a + min(m0 + t * 16 + r, P.last - 1) * 64 + blk * 16;
        qa = P.sa + word_of(m0, MT);
        ha = shift_of(m0);
    }
    const long long gm = row_groups(P.M) * 64, gn = row_groups(P.N) * 64;
    f32x4 acc[NT][MT] = {};
    u32x4 fb[U][NT], fa[U][MT];
    unsigned wb[U], wa[U];
    const auto fetch = [&](int u, int step) {             // (behind the last step: that one again)
        const long long k = min(step, P.kt - 1);
        wb[u] = qb[k * gn];
        if (X < 0) wa[u] = qa[k * gm];
#pragma unroll
        for (int i = 0; i < NT; ++i) fb[u][i] = *reinterpret_cast<const u32x4 *>(pb[i] + k * P.N * 64);
        if (X < 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) fa[u][t] = *reinterpret_cast<const u32x4 *>(pa[t] + k * P.M * 64);
        }
    };
    if (NT == 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) fetch(u, wave + 8 * u);
    }
    if (X >= 0) {
        const int per = P.kt * 4, blocks = static_cast<int>(P.M) * per;
        for (int i = threadIdx.x; i < blocks; i += 512) {
            const int row = i / per;
            const long long k = static_cast<long long>(i - row * per) * 32;
            float v[32];
            load_block<X < 0 ? 0 : X>(P.x, row * P.x_stride + k, k, P.K, P.x_vec, v);
            unsigned code;
            codes[i] = quantise32(v, code);
            scales[i] = static_cast<unsigned char>(code);
        }
        __syncthreads();
    }
    const auto multiply = [&](int u, int step) {
        if (X >= 0) {
            const int at = (r * P.kt + step) * 4 + blk;
            const bool mine = r < static_cast<int>(P.M);
            fa[u][0] = mine ? codes[at] : u32x4{0, 0, 0, 0};
            wa[u] = mine ? scales[at] : 0;
        }
        const u32x2 sb = words<NT>(wb[u], hb), sa = words<MT>(wa[u], ha);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[i][t] = mfma16(fb[u][i], fa[u][t], acc[i][t], sb[i & 1], i >> 1, sa[t & 1], t >> 1);
    };
    int k = wave;
    if (NT > 1 && k + 8 * (2 * U - 1) < P.kt) {          // each step's place is refilled at once
#pragma unroll
        for (int u = 0; u < U; ++u) fetch(u, k + 8 * u);
        for (; k + 8 * (2 * U - 1) < P.kt; k += 8 * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                multiply(u, k + 8 * u);
                fetch(u, k + 8 * (U + u));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) multiply(u, k + 8 * u);
        k += 8 * U;
    }
    for (; k < P.kt; k += 8 * U) {                       // the last steps, and all of a short or narrow product's
        if (NT > 1 || k != wave) {
#pragma unroll
            for (int u = 0; u < U; ++u) fetch(u, k + 8 * u);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + 8 * u >= P.kt) break;
            multiply(u, k + 8 * u);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[wave][i * MT + t][lane] = acc[i][t];
    __syncthreads();
    for (int tile = wave; tile < MT * NT; tile += 8) {
        f32x4 v = red[0][tile][lane];
#pragma unroll
        for (int i = 1; i < 8; ++i) v += red[i][tile][lane];
        const long long m = m0 + tile % MT * 16 + r, n = n0 + tile / MT * 16 + (lane >> 4) * 4;
        if (m >= P.last) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (P.bias && n + j < P.N) v[j] += bias_at(P.bias, P.bias_type, n + j);
        if (n + 4 <= P.N) {
            store4<T>(element<T>(P.out, m * P.N + n), v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < P.N) store1<T>(P.out, m * P.N + n + j, v[j]);
        }
    }
}

// The splits' sums, in order: out [M][N] = sum_i part[i][M][N] + bias
template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_gemm_sum(const float *__restrict__ part, int splits, const void *__restrict__ bias, int bias_type,
                                                           long long M, long long N, void *__restrict__ out) {
    const long long per = (N + 3) / 4, n = M * per;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long row = i / per, c = i % per * 4, at = row * N + c;
        f32x4 v = {};
        if (c + 4 <= N) {
#pragma unroll 4
            for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4_any *>(part + s * M * N + at);
        } else {
            for (int s = 0; s < splits; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < N) v[j] += part[s * M * N + at + j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (bias && c + j < N) v[j] += bias_at(bias, bias_type, c + j);
        if (c + 4 <= N) {
            store4<T>(element<T>(out, at), v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < N) store1<T>(out, at + j, v[j]);
        }
    }
}

// Large products: a workgroup of four waves takes a tile of 64 TM x 64 TN outputs, a wave 32 TM x 32 TN of it (TM, TN even).
// A step is 128 columns.  Its codes and scales go to LDS without passing registers, into a ring of STAGES stages and as many steps ahead
// of their use (three: 128 x 128 tiles then sit three to a CU, 5 % faster than two with four stages; 256 x 256 tiles take the same time
// with three and four); the fragments of the next 64 columns are read from LDS while the matrix cores work on these.  Fetches and reads
// stand between the matrix instructions, a few behind every fourth: a wave issues in order, and a run of fetches would hold up what
// comes behind it (measured on 8192^3: a step's fetches in one run 295 us, spread out 253).
//   codes in LDS: 64 bytes a row, the 16-byte block b of row r at slot b ^ (r / 4 % 4): the 16 lanes that LDS serves at once (rows
//   0-3, 12-15, 20-27 or 4-11, 16-19, 28-31 of a fragment) touch every bank once (measured: no bank conflicts).
// Per step and workgroup (TM = TN = 4): 32 matrix instructions of 32 cycles on each of four SIMDs = 1024 cycles, 64 KB of LDS reads
// (256 cycles at 256 B per cycle) and 34 KB from the caches.
typedef __attribute__((address_space(3))) void *lptr;
__device__ __forceinline__ unsigned lds_offset(const void *p) { return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lptr)p)); }
// 16 (4) bytes per lane from `src` to LDS offset `to` + 16 (4) * lane.  Written as assembly because the compiler would wait for ALL of
// them in front of every LDS read; there is no result register, the kernel counts and waits itself.
__device__ __forceinline__ void to_lds16(const void *src, unsigned to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(const void *src, unsigned to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(to) : "memory", "m0");
}

template <int TM, int TN, int STAGES> struct Tile {
    static constexpr int BM = 64 * TM, BN = 64 * TN;
    static constexpr int kCodes = (BM + BN) * 64, kStage = kCodes + (BM + BN) * 4, kStages = STAGES;
    static constexpr int kCodeLoads = (BM + BN) / 64, kWordLoads = ((BM + BN) / 64 + 3) / 4;   // 1 KB and 256 B pieces per wave and step
    static constexpr int kLoads = kCodeLoads + kWordLoads;
    static constexpr int kGroups = TM * TN / 4;                                             // of four matrix instructions, per 64 columns
};

__device__ __forceinline__ int slot_of(int r, int b) { return b ^ (r >> 2 & 3); }

template <int T, int TM, int TN, int STAGES>
__global__ __launch_bounds__(kThreads, 1) void k_mx4_gemm_tiled(const Product A, const Product B, unsigned first_tiles) {
    typedef Tile<TM, TN, STAGES> G;
    static_assert(G::kStages * G::kStage >= 4 * 32 * (32 * TN + 4) * 4, "the waves' output strips take the stages' place");
    __shared__ __align__(16) unsigned char lds[G::kStages * G::kStage];
    // the first workgroups are product A's; in each, one XCD's workgroups walk neighbouring tiles, 8 tile rows at a time: operands meet in
    // its L2
    const bool of_a = blockIdx.x < first_tiles;
    const Product &P = of_a ? A : B;
    const int all = of_a ? dipr_xcd_contiguous(blockIdx.x, first_tiles) : dipr_xcd_contiguous(blockIdx.x - first_tiles, gridDim.x - first_tiles);
    const long long M = P.M, N = P.N;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_m = static_cast<int>((P.last - P.first + G::BM - 1) / G::BM), tiles_n = static_cast<int>((N + G::BN - 1) / G::BN);
    const int split = all / (tiles_m * tiles_n), id = all % (tiles_m * tiles_n);
    const int group = 8 * tiles_n, first = id / group * 8, high = min(8, tiles_m - first);
    const long long m0 = P.first + static_cast<long long>(first + id % group % high) * G::BM;
    const long long n0 = static_cast<long long>(id % group / high) * G::BN;
    const int k_first = static_cast<int>(static_cast<long long>(P.kt) * split / P.splits);
    const int kt = static_cast<int>(static_cast<long long>(P.kt) * (split + 1) / P.splits) - k_first;
    const unsigned char *a = P.a + k_first * M * 64, *b = P.b + k_first * N * 64;
    const unsigned *sa = P.sa + k_first * row_groups(M) * 64, *sb = P.sb + k_first * row_groups(N) * 64;
    void *out = P.splits > 1 ? static_cast<float *>(P.out) + split * M * N : P.out;

    // this lane's source addresses: code pieces of 16 rows (rows 0 .. BM - 1 of a, then BN of b), scale pieces of 64 rows
    const unsigned char *src[G::kCodeLoads];
    const unsigned *ssrc[G::kWordLoads];
    long long move[G::kCodeLoads], smove[G::kWordLoads];                // uniform: what a step moves them on by
#pragma unroll
    for (int j = 0; j < G::kCodeLoads; ++j) {
        const int piece = wave * G::kCodeLoads + j, r = lane >> 2;
        const bool is_a = piece < G::BM / 16;
        const long long row = is_a ? min(m0 + piece * 16 + r, M - 1) : min(n0 + (piece - G::BM / 16) * 16 + r, N - 1);
        src[j] = (is_a ? a : b) + row * 64 + slot_of(r, lane & 3) * 16;
        move[j] = (is_a ? M : N) * 64;
    }
#pragma unroll
    for (int j = 0; j < G::kWordLoads; ++j) {
        const int piece = min(wave * G::kWordLoads + j, (G::BM + G::BN) / 64 - 1);      // (a spare one fetches the last again)
        const bool is_a = piece < G::BM / 64;
        const long long groups = is_a ? row_groups(M) : row_groups(N);
        const long long g = is_a ? min(m0 / 64 + piece, groups - 1) : min(n0 / 64 + piece - G::BM / 64, groups - 1);
        ssrc[j] = (is_a ? sa : sb) + g * 64 + lane;
        smove[j] = groups * 64;
    }
    const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_offset(lds));
    // piece j of step s, to its stage; the address moves on to the next step (behind the last one: the last one again, so that the number
    // of fetches on their way is the same in every step)
    auto fetch = [&](int s, int stage, int j) {
        const unsigned base = lds0 + stage * G::kStage;
        const bool on = s + 1 < kt;
        if (j < G::kCodeLoads) {
            to_lds16(src[j], base + (wave * G::kCodeLoads + j) * 1024);
            src[j] += on ? move[j] : 0;
        } else {
            const int i = j - G::kCodeLoads;
            to_lds4(ssrc[i], base + G::kCodes + min(wave * G::kWordLoads + i, (G::BM + G::BN) / 64 - 1) * 256);
            ssrc[i] += on ? smove[i] : 0;
        }
    };
    const int wm = (wave >> 1) * TM, wn = (wave & 1) * TN;              // this wave's first 32-row tile of a and of b
    // where this lane's block of the first / second 64 columns lies in a tile of 32 rows
    const int frag[2] = {(lane & 31) * 64 + slot_of(lane & 31, lane >> 5) * 16, (lane & 31) * 64 + slot_of(lane & 31, 2 + (lane >> 5)) * 16};
    struct Frags {
        u32x4 b[TN], a[TM];
    };
    struct Words {
        unsigned b[TN / 2], a[TM / 2];
    };
    // fragment i of the TN + TM ones
    auto read = [&](Frags &f, int stage, int h, int i) {
        const unsigned char *base = lds + stage * G::kStage;
        if (i < TN) f.b[i] = *reinterpret_cast<const u32x4 *>(base + G::BM * 64 + (wn + i) * 2048 + frag[h]);
        else f.a[i - TN] = *reinterpret_cast<const u32x4 *>(base + (wm + i - TN) * 2048 + frag[h]);
    };
    auto read_word = [&](Words &w, int stage, int i) {
        const unsigned char *base = lds + stage * G::kStage + G::kCodes;
        if (i < TN / 2) w.b[i] = reinterpret_cast<const unsigned *>(base + G::BM * 4 + (wn / 2 + i) * 256)[lane];
        else w.a[i - TN / 2] = reinterpret_cast<const unsigned *>(base + (wm / 2 + i - TN / 2) * 256)[lane];
    };
    f32x16 acc[TN][TM] = {};
    // 64 columns, half H of their step: in front of each group of four matrix instructions a share of the next 64 columns' reads (stage NS,
    // half NH) and of the fetches FIRST .. LAST - 1 of step FS to stage FT
#define MX4_COLUMNS(F, W, H, NF, NS, NH, WORDS, NW, FS, FT, FIRST, LAST)                                                           \
    _Pragma("unroll") for (int g = 0; g < G::kGroups; ++g) {                                                                       \
        const int i = g % (TN / 2) * 2, j = g / (TN / 2) * 2;                                                                      \
        if (WORDS) {                                                                                                               \
            _Pragma("unroll") for (int x = (TM + TN) / 2 * g / G::kGroups; x < (TM + TN) / 2 * (g + 1) / G::kGroups; ++x)          \
                read_word(NW, NS, x);                                                                                              \
        }                                                                                                                          \
        _Pragma("unroll") for (int x = (TM + TN) * g / G::kGroups; x < (TM + TN) * (g + 1) / G::kGroups; ++x) read(NF, NS, NH, x); \
        _Pragma("unroll") for (int x = FIRST + (LAST - FIRST) * g / G::kGroups; x < FIRST + (LAST - FIRST) * (g + 1) / G::kGroups; ++x) fetch(FS, FT, x); \
        acc[i][j] = mfma<2 * H, 2 * H>(F.b[i], F.a[j], acc[i][j], W.b[i / 2], W.a[j / 2]);                                         \
        acc[i + 1][j] = mfma<2 * H + 1, 2 * H>(F.b[i + 1], F.a[j], acc[i + 1][j], W.b[i / 2], W.a[j / 2]);                         \
        acc[i][j + 1] = mfma<2 * H, 2 * H + 1>(F.b[i], F.a[j + 1], acc[i][j + 1], W.b[i / 2], W.a[j / 2]);                         \
        acc[i + 1][j + 1] = mfma<2 * H + 1, 2 * H + 1>(F.b[i + 1], F.a[j + 1], acc[i + 1][j + 1], W.b[i / 2], W.a[j / 2]);         \
        __builtin_amdgcn_sched_barrier(0);                                                                                         \
    }
    // waits until at most `steps` fetched steps are still on their way and everything read from LDS is here, then for all waves
#define MX4_ARRIVED(STEPS)                                                                       \
    do {                                                                                         \
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STEPS) * G::kLoads) : "memory");     \
        __builtin_amdgcn_s_barrier();                                                            \
    } while (0)
    constexpr int kHalf = G::kLoads / 2, kAhead = STAGES - 1;
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
        for (int j = 0; j < G::kLoads; ++j) fetch(s, s, j);
#pragma unroll
    for (int j = 0; j < kHalf; ++j) fetch(kAhead, kAhead, j);
    Frags f0, f1;
    Words w, next;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kAhead - 1) * G::kLoads + kHalf) : "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int i = 0; i < TM + TN; ++i) read(f0, 0, 0, i);
#pragma unroll
    for (int i = 0; i < (TM + TN) / 2; ++i) read_word(w, 0, i);
    int here = 0;                                        // the stage of step k
    for (int k = 0; k < kt; ++k) {
        const int after = here + 1 == STAGES ? 0 : here + 1, last = here == 0 ? STAGES - 1 : here - 1;
        MX4_COLUMNS(f0, w, 0, f1, here, 1, false, next, k + kAhead, last, kHalf, G::kLoads)
        // step k + 1 is in LDS (the ones behind it may be on their way); behind the barrier every wave has read stage `here`, which is free
        // for step k + STAGES
        MX4_ARRIVED(STAGES - 2);
        MX4_COLUMNS(f1, w, 1, f0, after, 0, true, next, k + STAGES, here, 0, kHalf)
        w = next;
        here = after;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // nothing may arrive in LDS behind the last use of a stage
#undef MX4_ARRIVED
#undef MX4_COLUMNS

    __syncthreads();                                     // every wave is through with the stages
    store_tiles<T, TM, TN>(acc, reinterpret_cast<float *>(lds) + wave * 32 * (32 * TN + 4), P.bias, P.bias_type, m0 + wm * 32, n0 + wn * 32,
                           P.last, N, out);
}

// ------------------------------------------------------------------------------------------------------------------- host side
inline bool good_dtype(int d) { return d == F32 || d == BF16 || d == F16; }
inline bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int elem_bytes(int d) { return d == F32 ? 4 : 2; }
constexpr long long kMaxSide = 1ll << 28, kMaxGrid = 1ll << 23;       // a launch counts its threads in 32 bits

// blocks down the columns need the padding rows' zeros too
inline long long quantise_tiles(const Matrix &m) {
    return (m.col_codes ? round_up(m.R, 128) / kQR : (m.R + kQR - 1) / kQR) * ((m.C + kQC - 1) / kQC);
}
template <int T> void launch_quantise(DiprProf &prof, const Matrix &m, const Matrix *other, hipStream_t st) {
    const unsigned first = static_cast<unsigned>(quantise_tiles(m));
    const dim3 grid(first + (other ? static_cast<unsigned>(quantise_tiles(*other)) : 0u)), block(kThreads);
    const Matrix &n = other ? *other : m;
#define MX4_QUANTISE(ROW, COL, SUM) DIPR_LAUNCH(prof, (k_mx4_quantise<T, ROW, COL, SUM>), grid, block, st, m, n, first)
    if (m.row_codes && m.col_codes && m.sums) MX4_QUANTISE(true, true, true);
    else if (m.row_codes && m.col_codes) MX4_QUANTISE(true, true, false);
    else if (m.col_codes && m.sums) MX4_QUANTISE(false, true, true);
    else if (m.col_codes) MX4_QUANTISE(false, true, false);
    else MX4_QUANTISE(true, false, false);
#undef MX4_QUANTISE
}

// ---- which kernels a product takes
// Estimated from measured times (ns).  A round of workgroups over the CUs costs its begin and end and its steps of 128 columns:
//   256 x 256 tiles 10 000 + 860 a step; 128 x 128 tiles, up to two on a CU, 6 500 + 200 (on half the CUs), 270 (one a CU) or 690 a step; 64 x 64 tiles 1 500 and
//   2 300 + 140 a step for each round; 64 x 32 tiles 2 000 and 1 000 + 100; 64 rows x 16 columns 2 200 and 700 + 85; a second launch that adds up
//   partial sums 4 000 and their bytes at 4 TB/s.
// Measured (us): 8192^3 251 large, 355 small; 4096 x 4096 x 8200 65 / 78; 2048^3 18.4 / 10.0, 64 x 32 19.5; 512 x 512 x 16384 34.8 small, 15.5 with
// the columns in eight, 64 x 32 15.0; 64 x 8192 x 8192 14.0 by 16 columns, 64 x 32 10.0, 64 x 64 12.2; 64 x 4096 x 9216 8.6 / 9.4 / 11.9;
// 8192 x 300 x 300 7.6 small, 64 x 32 9.2, 64 x 64 10.4; 4096 x 512 x 4096 12.7, 23.1, 17.5.
struct Plan {
    enum { kRows, k64x32, k64x64, kSmall, kLarge } form;
    int splits;                  // kSmall only
    long long tail;              // kLarge only: rows at the end that go to the kernel for few rows (0: none)
    bool strips() const { return form == k64x32 || form == k64x64; }
};
inline long long tiles_of(long long m, long long n, int side) { return ((m + side - 1) / side) * ((n + side - 1) / side); }
inline int cu_count() {
    const int n = dipr_device_cu_count();
    return n > 0 ? n : 256;
}
inline double large_ns(long long m, long long n, long long kt) {
    const long long rounds = (tiles_of(m, n, 256) + cu_count() - 1) / cu_count();
    return static_cast<double>(rounds) * (860.0 * kt + 10000.0);
}
inline double small_ns(long long m, long long n, long long kt, int splits) {
    const double slots = 2.0 * cu_count(), tiles = static_cast<double>(tiles_of(m, n, 128)) * splits;
    const double step = tiles <= slots / 4 ? 200.0 : tiles <= slots / 2 ? 270.0 : 690.0 * (tiles > slots ? tiles / slots : 1.0);
    const double sums = splits > 1 ? 4000.0 + static_cast<double>(splits) * m * n * 8 / 4000.0 : 0.0;
    return step * static_cast<double>((kt + splits - 1) / splits) + 6500.0 + sums;
}
inline long long strips_of(long long m, long long n, int nt) { return ((m + 63) / 64) * ((n + 16 * nt - 1) / (16 * nt)); }
inline double strip_ns(long long m, long long n, long long kt, int nt) {
    const double rounds = static_cast<double>((strips_of(m, n, nt) + cu_count() - 1) / cu_count()), steps = static_cast<double>(kt);
    return nt == 1 ? 2200.0 + rounds * (700.0 + 85.0 * steps) : nt == 2 ? 2000.0 + rounds * (1000.0 + 100.0 * steps) : 1500.0 + rounds * (2300.0 + 140.0 * steps);
}
Plan plan(long long M, long long N, long long kt) {
    Plan p = {Plan::kRows, 1, 0};
    if (M <= 32) return p;
    double best = strip_ns(M, N, kt, 1);
    if (M > 64) {
        p.form = Plan::kLarge;
        best = large_ns(M, N, kt);
    }
    // a few rows behind whole tiles: a tile row of their own could cost a round
    const long long tail = M % 256 <= 64 && M > 256 ? M % 256 : 0;
    if (tail) {
        const double t = large_ns(M - tail, N, kt) + 5000.0 + static_cast<double>(N * kt) / 80.0;
        if (t < best) best = t, p.tail = tail;
    }
    for (int splits = 1; M > 64 && splits <= 16 && splits <= kt; splits += splits < 4 ? 1 : splits / 2) {
        if (splits > 1 && tiles_of(M, N, 128) * splits > 4 * cu_count()) break;
        const double t = small_ns(M, N, kt, splits);
        if (t < best) {
            best = t;
            p.form = Plan::kSmall;
            p.splits = splits;
            p.tail = 0;
        }
    }
    for (int nt = 2; nt <= 4; nt += 2) {
        if (strips_of(M, N, nt) > 8 * cu_count()) continue;
        const double t = strip_ns(M, N, kt, nt);
        if (t < best) {
            best = t;
            p.form = nt == 2 ? Plan::k64x32 : Plan::k64x64;
            p.splits = 1;
            p.tail = 0;
        }
    }
    return p;
}

inline double flops(const Product &P) { return 2.0 * static_cast<double>(P.last - P.first) * static_cast<double>(P.N) * static_cast<double>(P.K); }

// Every launch is timed by itself, with its own operations.
template <int T> void launch_rows(const Product &P, hipStream_t st) {
    DiprProf prof(DEEPIPR_K_MX4_MATMUL);
    prof.bytes = flops(P);
    const dim3 grid(static_cast<unsigned>((P.N + 15) / 16)), block(512);
    const long long rows = P.last - P.first;
    if (rows <= 16) DIPR_LAUNCH(prof, (k_mx4_gemm_rows<T, 1, 1, -1>), grid, block, st, P, P, grid.x);
    else if (rows <= 32) DIPR_LAUNCH(prof, (k_mx4_gemm_rows<T, 2, 1, -1>), grid, block, st, P, P, grid.x);
    else DIPR_LAUNCH(prof, (k_mx4_gemm_rows<T, 4, 1, -1>), grid, block, st, P, P, grid.x);
}

template <int T> void launch_product(Product P, const Product *other, float *part, hipStream_t st) {
    const dim3 block(kThreads);
    const Plan p = plan(P.M, P.N, P.kt);
    if (p.form == Plan::kRows) return launch_rows<T>(P, st);
    if (p.strips()) {
        int nt = p.form == Plan::k64x32 ? 2 : 4;
        if (other)                                       // one width for both
            nt = strip_ns(P.M, P.N, P.kt, 2) + strip_ns(other->M, other->N, other->kt, 2) <=
                         strip_ns(P.M, P.N, P.kt, 4) + strip_ns(other->M, other->N, other->kt, 4) ? 2 : 4;
        const unsigned first = static_cast<unsigned>(strips_of(P.M, P.N, nt));
        const dim3 grid(first + (other ? static_cast<unsigned>(strips_of(other->M, other->N, nt)) : 0u)), wide(512);
        const Product &Q = other ? *other : P;
        DiprProf prof(DEEPIPR_K_MX4_MATMUL);
        prof.bytes = flops(P) + (other ? flops(Q) : 0.0);
        if (nt == 2) DIPR_LAUNCH(prof, (k_mx4_gemm_rows<T, 4, 2, -1>), grid, wide, st, P, Q, first);
        else DIPR_LAUNCH(prof, (k_mx4_gemm_rows<T, 4, 4, -1>), grid, wide, st, P, Q, first);
        return;
    }
    Product O = other ? *other : P;
    const long long tails[2] = {p.tail, other ? plan(O.M, O.N, O.kt).tail : 0};
    Product *both[2] = {&P, &O};
    for (int i = 0; i < 2; ++i)
        if (tails[i]) {
            Product Q = *both[i];
            Q.first = Q.M - tails[i];
            launch_rows<T>(Q, st);
            both[i]->last -= tails[i];
        }
    const int side = p.form == Plan::kLarge ? 256 : 128;
    const unsigned first = static_cast<unsigned>(tiles_of(P.last, P.N, side)) * p.splits;
    const dim3 grid(first + (other ? static_cast<unsigned>(tiles_of(O.last, O.N, side)) : 0u));
    DiprProf prof(DEEPIPR_K_MX4_MATMUL);
    prof.bytes = flops(P) + (other ? flops(O) : 0.0);
    if (p.form == Plan::kLarge) {
        DIPR_LAUNCH(prof, (k_mx4_gemm_tiled<T, 4, 4, 3>), grid, block, st, P, O, first);
    } else if (p.splits == 1) {
        DIPR_LAUNCH(prof, (k_mx4_gemm_tiled<T, 2, 2, 3>), grid, block, st, P, O, first);
    } else {
        Product Q = P;
        Q.splits = p.splits;
        Q.out = part;
        Q.bias = nullptr;
        DIPR_LAUNCH(prof, (k_mx4_gemm_tiled<F32, 2, 2, 3>), grid, block, st, Q, Q, first);
        const long long want = (P.M * ((P.N + 3) / 4) + kThreads - 1) / kThreads;
        DiprProf sum(DEEPIPR_K_MX4_MATMUL);              // time of the product, no operations of its own
        DIPR_LAUNCH(sum, (k_mx4_gemm_sum<T>), dim3(static_cast<unsigned>(want < 8192 ? want : 8192)), block, st, part, p.splits, P.bias,
                    P.bias_type, P.M, P.N, P.out);
    }
}

// ---- the pieces that the C entries share; arguments are checked by then
Matrix matrix_of(const void *x, int dtype, long long R, long long C, long long stride, void *rc, void *rs, void *cc, void *cs, float *sums) {
    Matrix m;
    m.x = x;
    m.R = R;
    m.C = C;
    m.stride = stride;
    m.vec = aligned(x, 16) && (R == 1 || stride * elem_bytes(dtype) % 16 == 0);
    m.row_codes = static_cast<unsigned char *>(rc);
    m.row_scales = static_cast<unsigned *>(rs);
    m.col_codes = static_cast<unsigned char *>(cc);
    m.col_scales = static_cast<unsigned *>(cs);
    m.sums = sums;
    return m;
}
// `other`: a second matrix of the same type and directions, in the same launch
void quantise(int dtype, const Matrix &m, const Matrix *other, hipStream_t st) {
    DiprProf prof(DEEPIPR_K_MX4_QUANTIZE);
    const auto bytes = [&](const Matrix &q) {
        return static_cast<double>(q.R) * static_cast<double>(q.C) * (elem_bytes(dtype) + 0.53125 * ((q.row_codes ? 1 : 0) + (q.col_codes ? 1 : 0)));
    };
    prof.bytes = bytes(m) + (other ? bytes(*other) : 0.0);
    switch (dtype) {
        case F32: launch_quantise<F32>(prof, m, other, st); break;
        case BF16: launch_quantise<BF16>(prof, m, other, st); break;
        default: launch_quantise<F16>(prof, m, other, st); break;
    }
}
void column_sums(const Matrix &m, float *out, hipStream_t st) {
    long long items = round_up(m.R, 128) / kQR, step = 1;
    for (;;) {                                                           // at most 128 items in one go: long batches take a second or third pass
        const long long groups = (items + kSumTiles - 1) / kSumTiles;
        const dim3 grid(static_cast<unsigned>((m.C + 31) / 32), static_cast<unsigned>(groups)), block(kThreads);
        DiprProf prof(DEEPIPR_K_MX4_QUANTIZE);
        prof.bytes = static_cast<double>(items) * static_cast<double>(m.C) * (step == 1 ? 4.0 : 8.0);
        if (step == 1) DIPR_LAUNCH(prof, k_mx4_colsum<true>, grid, block, st, m.sums, items, step, m.C, out);
        else DIPR_LAUNCH(prof, k_mx4_colsum<false>, grid, block, st, m.sums, items, step, m.C, out);
        if (groups == 1) return;
        items = groups;
        step *= kSumTiles;
    }
}
inline size_t sums_bytes(long long R, long long C) {                      // the tiles' sums (and a row for every group of them, which stays free)
    size_t n = 0;
    for (long long tiles = round_up(R, 128) / kQR;; tiles = (tiles + kSumTiles - 1) / kSumTiles) {
        n += static_cast<size_t>(tiles);
        if (tiles <= kSumTiles) return n * static_cast<size_t>(C) * sizeof(float);
    }
}
inline bool quantise_fits(long long R, long long C) {
    // (the grid of the column sums is 65 535 groups of 128 tiles at most)
    return R <= 65535ll * kSumTiles * kQR && C <= kMaxSide && round_up(R, 128) / kQR * ((C + kQC - 1) / kQC) <= kMaxGrid;
}
inline bool product_fits(long long M, long long N, long long K) {
    return M <= kMaxSide && N <= kMaxSide && K <= kMaxSide && tiles_of(M, N, 128) <= kMaxGrid && (N + 15) / 16 < kMaxGrid &&
           round_up(K, 128) / 128 <= kMaxGrid;
}
inline size_t product_bytes(long long M, long long N, long long K) {
    const Plan p = plan(M, N, round_up(K, 128) / 128);
    return p.splits > 1 ? static_cast<size_t>(p.splits) * static_cast<size_t>(M) * static_cast<size_t>(N) * sizeof(float) : 0;
}
Product product_of(const void *a, const void *sa, const void *b, const void *sb, const void *bias, int bias_dtype, long long M, long long N,
                   long long K, void *out) {
    Product P = {};
    P.a = static_cast<const unsigned char *>(a);
    P.b = static_cast<const unsigned char *>(b);
    P.sa = static_cast<const unsigned *>(sa);
    P.sb = static_cast<const unsigned *>(sb);
    P.bias = bias;
    P.bias_type = bias_dtype;
    P.M = P.last = M;
    P.N = N;
    P.K = K;
    P.kt = static_cast<int>(round_up(K, 128) / 128);
    P.splits = 1;
    P.out = out;
    return P;
}
// Whether two products of one output type can share a launch
bool alike(const Product &p, const Product &q) {
    const Plan a = plan(p.M, p.N, p.kt), b = plan(q.M, q.N, q.kt);
    if (a.strips() && b.strips()) return true;
    return a.form == b.form && a.form != Plan::kRows && a.splits == 1 && b.splits == 1 &&
           tiles_of(p.M, p.N, 128) + tiles_of(q.M, q.N, 128) <= kMaxGrid;
}
// `other`: a second product that is alike, in the same launch
void run(const Product &P, const Product *other, int dtype, void *workspace, hipStream_t st) {
    switch (dtype) {
        case F32: launch_product<F32>(P, other, static_cast<float *>(workspace), st); break;
        case BF16: launch_product<BF16>(P, other, static_cast<float *>(workspace), st); break;
        default: launch_product<F16>(P, other, static_cast<float *>(workspace), st); break;
    }
}

// The same with a in its own type, for at most 16 rows (out of a's type): one launch
void product_of_rows(const void *x, int dtype, long long x_stride, const void *b, const void *sb, const void *bias, int bias_dtype, long long M,
                     long long N, long long K, void *out, hipStream_t st) {
    Product P = product_of(nullptr, nullptr, b, sb, bias, bias_dtype, M, N, K, out);
    P.x = x;
    P.x_stride = x_stride;
    P.x_vec = aligned(x, 16) && (M == 1 || x_stride * elem_bytes(dtype) % 16 == 0);
    DiprProf prof(DEEPIPR_K_MX4_MATMUL);
    prof.bytes = flops(P);
    const dim3 grid(static_cast<unsigned>((N + 15) / 16)), block(512);
    switch (dtype) {
        case F32: DIPR_LAUNCH(prof, (k_mx4_gemm_rows<F32, 1, 1, F32>), grid, block, st, P, P, grid.x); break;
        case BF16: DIPR_LAUNCH(prof, (k_mx4_gemm_rows<BF16, 1, 1, BF16>), grid, block, st, P, P, grid.x); break;
        default: DIPR_LAUNCH(prof, (k_mx4_gemm_rows<F16, 1, 1, F16>), grid, block, st, P, P, grid.x); break;
    }
}

// Cuts one buffer into pieces of whole 256-byte units.
struct Cut {
    char *base;
    size_t used = 0;
    explicit Cut(const void *p) : base(static_cast<char *>(const_cast<void *>(p))) {}
    void *take(size_t bytes) {
        void *p = base ? base + used : nullptr;
        used += static_cast<size_t>(round_up(static_cast<long long>(bytes), 256));
        return p;
    }
};
struct Quantised {
    void *codes = nullptr, *scales = nullptr;
};
Quantised take_matrix(Cut &c, long long rows, long long cols) {
    Quantised q;
    q.codes = c.take(deepipr_mx4_code_bytes(rows, cols));
    q.scales = c.take(deepipr_mx4_scale_bytes(rows, cols));
    return q;
}
struct Saved {                   // what a forward pass leaves for its backward pass: blocks along the rows of the batch / the output features
    Quantised x_t, w_t;
    size_t bytes;
    Saved(const void *p, long long M, long long N, long long K, bool dx, bool dw) {
        Cut c(p);
        if (dw) x_t = take_matrix(c, K, M);
        if (dx) w_t = take_matrix(c, K, N);
        bytes = c.used;
    }
};
struct ForwardScratch {
    Quantised x, w;
    void *work;
    size_t bytes;
    ForwardScratch(void *p, long long M, long long N, long long K, bool kept) {
        Cut c(p);
        x = take_matrix(c, M, K);
        if (!kept) w = take_matrix(c, N, K);
        work = c.take(product_bytes(M, N, K));
        bytes = c.used;
    }
};
struct BackwardScratch {
    Quantised y, y_t;
    void *sums, *work;
    size_t bytes;
    BackwardScratch(void *p, long long M, long long N, long long K) {
        Cut c(p);
        y = take_matrix(c, M, N);
        y_t = take_matrix(c, N, M);
        sums = c.take(sums_bytes(M, N));
        const size_t dx = product_bytes(M, K, N), dw = product_bytes(N, K, M);       // one after the other
        work = c.take(dx > dw ? dx : dw);
        bytes = c.used;
    }
};
inline bool linear_fits(long long M, long long N, long long K) {
    return M > 0 && N > 0 && K > 0 && quantise_fits(M, K) && quantise_fits(N, K) && quantise_fits(M, N) && product_fits(M, N, K) &&
           product_fits(M, K, N) && product_fits(N, K, M);
}
// Whether a product on kept weights quantises its rows itself
inline bool is_fused(long long M, long long K, int dtype) { return M <= 16 && M * (round_up(K, 128) / 32) * elem_bytes(dtype) <= 2 * kFusedBlocks; }
inline bool good_matrix(const void *p, int dtype, long long rows, long long cols, long long stride) {
    return p && good_dtype(dtype) && aligned(p, elem_bytes(dtype)) && (rows <= 1 || stride >= cols);
}

}  // namespace

extern "C" {

size_t deepipr_mx4_code_bytes(long long rows, long long cols) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<size_t>(rows) * static_cast<size_t>(round_up(cols, 128) / 2);
}
size_t deepipr_mx4_scale_bytes(long long rows, long long cols) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<size_t>(round_up(cols, 128) / 128) * static_cast<size_t>(row_groups(rows)) * 256;
}
size_t deepipr_mx4_quantize_workspace_bytes(long long rows, long long cols) { return rows <= 0 || cols <= 0 ? 0 : sums_bytes(rows, cols); }

int deepipr_mx4_quantize(const void *x, int dtype, long long rows, long long cols, long long row_stride, void *row_codes, void *row_scales,
                         void *col_codes, void *col_scales, float *col_sums, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "mx4_quantize";
    if (!x || !good_dtype(dtype) || rows <= 0 || cols <= 0 || rows > kMaxSide || cols > kMaxSide || (rows > 1 && row_stride < cols))
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!row_codes != !row_scales || !col_codes != !col_scales || (!row_codes && !col_codes))
        return dipr_fail(DEEPIPR_EINVAL, "%s: codes and scales of at least one direction", what);
    if (col_sums && (!col_codes || !workspace || workspace_bytes < deepipr_mx4_quantize_workspace_bytes(rows, cols) || !aligned(workspace, 4)))
        return dipr_fail(DEEPIPR_EINVAL, "%s: column sums need the column direction and a workspace", what);
    if (!aligned(x, elem_bytes(dtype)) || !aligned(row_codes, 16) || !aligned(row_scales, 16) || !aligned(col_codes, 16) || !aligned(col_scales, 16))
        return dipr_fail(DEEPIPR_EINVAL, "%s: misaligned pointer", what);
    if (!quantise_fits(rows, cols)) return dipr_fail(DEEPIPR_EINVAL, "%s: matrix too large", what);
    const Matrix m = matrix_of(x, dtype, rows, cols, row_stride, row_codes, row_scales, col_codes, col_scales,
                               col_sums ? static_cast<float *>(workspace) : nullptr);
    quantise(dtype, m, nullptr, static_cast<hipStream_t>(stream));
    if (col_sums) column_sums(m, col_sums, static_cast<hipStream_t>(stream));
    return dipr_check_launch(what);
}

int deepipr_mx4_dequantize(const void *codes, const void *scales, long long rows, long long cols, int transposed, void *out, int dtype,
                           void *stream) {
    const char *what = "mx4_dequantize";
    if (!codes || !scales || !out || !good_dtype(dtype) || rows <= 0 || cols <= 0 || rows > kMaxSide || cols > kMaxSide)
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(out, elem_bytes(dtype))) return dipr_fail(DEEPIPR_EINVAL, "%s: misaligned pointer", what);
    const long long tiles = ((rows + 63) / 64) * ((cols + 127) / 128);
    if (tiles > kMaxGrid) return dipr_fail(DEEPIPR_EINVAL, "%s: matrix too large", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    DiprProf prof(DEEPIPR_K_MX4_DEQUANTIZE);
    prof.bytes = static_cast<double>(rows) * static_cast<double>(cols) * (elem_bytes(dtype) + 0.53125);
    const unsigned char *c = static_cast<const unsigned char *>(codes);
    const unsigned *s = static_cast<const unsigned *>(scales);
#define MX4_DEQUANTISE(T)                                                                                                            \
    do {                                                                                                                             \
        if (transposed) {                                                                                                            \
            DIPR_LAUNCH(prof, (k_mx4_dequantise_t<T>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), st, c, s, rows, cols, out); \
        } else {                                                                                                                     \
            DIPR_LAUNCH(prof, (k_mx4_dequantise<T>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), st, c, s, rows, cols, out);  \
        }                                                                                                                            \
    } while (0)
    switch (dtype) {
        case F32: MX4_DEQUANTISE(F32); break;
        case BF16: MX4_DEQUANTISE(BF16); break;
        default: MX4_DEQUANTISE(F16); break;
    }
#undef MX4_DEQUANTISE
    return dipr_check_launch(what);
}

size_t deepipr_mx4_matmul_workspace_bytes(long long M, long long N, long long K) {
    return M <= 0 || N <= 0 || K <= 0 || !product_fits(M, N, K) ? 0 : product_bytes(M, N, K);
}

int deepipr_mx4_matmul(const void *a_codes, const void *a_scales, const void *b_codes, const void *b_scales, const void *bias, int bias_dtype,
                       long long M, long long N, long long K, void *out, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "mx4_matmul";
    if (!a_codes || !a_scales || !b_codes || !b_scales || !out || !good_dtype(dtype) || (bias && !good_dtype(bias_dtype)) || M <= 0 || N <= 0 || K <= 0)
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!aligned(a_codes, 16) || !aligned(a_scales, 16) || !aligned(b_codes, 16) || !aligned(b_scales, 16) || !aligned(out, elem_bytes(dtype)) ||
        (bias && !aligned(bias, elem_bytes(bias_dtype))))
        return dipr_fail(DEEPIPR_EINVAL, "%s: misaligned pointer", what);
    if (!product_fits(M, N, K)) return dipr_fail(DEEPIPR_EINVAL, "%s: matrix too large", what);
    const size_t need = product_bytes(M, N, K);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return dipr_fail(DEEPIPR_EINVAL, "%s: workspace too small or misaligned", what);
    run(product_of(a_codes, a_scales, b_codes, b_scales, bias, bias_dtype, M, N, K, out), nullptr, dtype, workspace,
        static_cast<hipStream_t>(stream));
    return dipr_check_launch(what);
}

size_t deepipr_mx4_linear_saved_bytes(long long M, long long N, long long K, int need_dx, int need_dw) {
    return M <= 0 || N <= 0 || K <= 0 ? 0 : Saved(nullptr, M, N, K, need_dx != 0, need_dw != 0).bytes;
}
size_t deepipr_mx4_linear_scratch_bytes(long long M, long long N, long long K, int backward) {
    if (!linear_fits(M, N, K)) return 0;
    return backward ? BackwardScratch(nullptr, M, N, K).bytes : ForwardScratch(nullptr, M, N, K, false).bytes;
}
size_t deepipr_mx4_linear_kept_scratch_bytes(int x_dtype, long long M, long long N, long long K) {
    return !good_dtype(x_dtype) || !linear_fits(M, N, K) || is_fused(M, K, x_dtype) ? 0 : ForwardScratch(nullptr, M, N, K, true).bytes;
}

int deepipr_mx4_linear_fwd(const void *x, int x_dtype, long long x_stride, const void *w, int w_dtype, long long w_stride, const void *w_codes,
                           const void *w_scales, const void *bias, int bias_dtype, long long M, long long N, long long K, int need_dx, int need_dw,
                           void *saved, size_t saved_bytes, void *out, void *scratch, size_t scratch_bytes, void *stream) {
    const char *what = "mx4_linear_fwd";
    if (!linear_fits(M, N, K)) return dipr_fail(DEEPIPR_EINVAL, "%s: bad or too large sizes", what);
    const bool kept = !w;
    if (!good_matrix(x, x_dtype, M, K, x_stride) || (!kept && !good_matrix(w, w_dtype, N, K, w_stride)) || !out || !aligned(out, elem_bytes(x_dtype)) ||
        (kept && (!w_codes || !w_scales || !aligned(w_codes, 16) || !aligned(w_scales, 16) || need_dx || need_dw)) ||
        (bias && (!good_dtype(bias_dtype) || !aligned(bias, elem_bytes(bias_dtype)))))
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    const Saved s(saved, M, N, K, need_dx != 0, need_dw != 0);
    const bool fused = kept && is_fused(M, K, x_dtype);
    const ForwardScratch f(scratch, M, N, K, kept);
    if ((!fused && (!scratch || !aligned(scratch, 16) || scratch_bytes < f.bytes)) || (s.bytes && (!saved || !aligned(saved, 16) || saved_bytes < s.bytes)))
        return dipr_fail(DEEPIPR_EINVAL, "%s: scratch or saved memory too small or misaligned", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (fused) {
        product_of_rows(x, x_dtype, x_stride, w_codes, w_scales, bias, bias_dtype, M, N, K, out, st);
        return dipr_check_launch(what);
    }
    const Matrix mx = matrix_of(x, x_dtype, M, K, x_stride, f.x.codes, f.x.scales, s.x_t.codes, s.x_t.scales, nullptr);
    if (kept) {
        quantise(x_dtype, mx, nullptr, st);
    } else {
        const Matrix mw = matrix_of(w, w_dtype, N, K, w_stride, f.w.codes, f.w.scales, s.w_t.codes, s.w_t.scales, nullptr);
        const bool together = x_dtype == w_dtype && !mx.col_codes == !mw.col_codes && quantise_tiles(mx) + quantise_tiles(mw) <= kMaxGrid;
        quantise(x_dtype, mx, together ? &mw : nullptr, st);
        if (!together) quantise(w_dtype, mw, nullptr, st);
    }
    run(product_of(f.x.codes, f.x.scales, kept ? w_codes : f.w.codes, kept ? w_scales : f.w.scales, bias, bias_dtype, M, N, K, out), nullptr, x_dtype,
        f.work, st);
    return dipr_check_launch(what);
}

int deepipr_mx4_linear_bwd(const void *dy, int dy_dtype, long long dy_stride, long long M, long long N, long long K, int need_dx, int need_dw,
                           const void *saved, size_t saved_bytes, void *dx, int dx_dtype, void *dw, int dw_dtype, float *dbias, void *scratch,
                           size_t scratch_bytes, void *stream) {
    const char *what = "mx4_linear_bwd";
    if (!linear_fits(M, N, K)) return dipr_fail(DEEPIPR_EINVAL, "%s: bad or too large sizes", what);
    if (!good_matrix(dy, dy_dtype, M, N, dy_stride) || (dx && (!need_dx || !good_dtype(dx_dtype) || !aligned(dx, elem_bytes(dx_dtype)))) ||
        (dw && (!need_dw || !good_dtype(dw_dtype) || !aligned(dw, elem_bytes(dw_dtype)))) || !aligned(dbias, 4) || (!dx && !dw && !dbias))
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    const Saved s(saved, M, N, K, need_dx != 0, need_dw != 0);
    const BackwardScratch b(scratch, M, N, K);
    if (!scratch || !aligned(scratch, 16) || scratch_bytes < b.bytes || (s.bytes && (!saved || !aligned(saved, 16) || saved_bytes < s.bytes)))
        return dipr_fail(DEEPIPR_EINVAL, "%s: scratch or saved memory too small or misaligned", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool down = dw || dbias;
    const Matrix my = matrix_of(dy, dy_dtype, M, N, dy_stride, dx ? b.y.codes : nullptr, dx ? b.y.scales : nullptr, down ? b.y_t.codes : nullptr,
                                down ? b.y_t.scales : nullptr, dbias ? static_cast<float *>(b.sums) : nullptr);
    quantise(dy_dtype, my, nullptr, st);
    if (dbias) column_sums(my, dbias, st);
    const Product px = product_of(b.y.codes, b.y.scales, s.w_t.codes, s.w_t.scales, nullptr, 0, M, K, N, dx);
    const Product pw = product_of(b.y_t.codes, b.y_t.scales, s.x_t.codes, s.x_t.scales, nullptr, 0, N, K, M, dw);
    if (dx && dw && dx_dtype == dw_dtype && alike(px, pw)) {
        run(pw, &px, dw_dtype, b.work, st);
    } else {
        if (dx) run(px, nullptr, dx_dtype, b.work, st);
        if (dw) run(pw, nullptr, dw_dtype, b.work, st);
    }
    return dipr_check_launch(what);
}

#ifdef DEEPIPR_TEST_HOOKS
int deepipr_debug_mx4_plan(long long M, long long N, long long K, long long *plan_out) {
    if (!plan_out || M <= 0 || N <= 0 || K <= 0 || !product_fits(M, N, K)) return dipr_fail(DEEPIPR_EINVAL, "debug_mx4_plan: bad argument");
    const Plan p = plan(M, N, round_up(K, 128) / 128);
    plan_out[0] = p.form;
    plan_out[1] = p.splits;
    plan_out[2] = p.tail;
    return DEEPIPR_OK;
}
#endif

}  // extern "C"
