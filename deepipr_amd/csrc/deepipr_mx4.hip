// deepipr_mx4.hip -- translation unit of libdeepipr_hip.so: matrices in microscaled 4-bit floating point ("MX4") and their products.
//
// The format (the open MX specification's MXFP4): 32 neighbouring values of a row share a power of two X = 2^(code - 127), held in one
// byte (E8M0; 255 = not a number); each value is a 4-bit float E2M1 -- sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- times X.
// Quantising: code = max(0, biased exponent of max|block| - 2), so max|block| / X lies in [4, 8); values are rounded to the nearest code,
// ties to the even one, and saturate at 6.  Division by X is exact, so every value's code is a function of its block alone.
// A block that holds a NaN or an infinity gets code 255: all of it reads as NaN.
//
// In memory a quantised matrix of R rows and K columns, Kp = K rounded up to 128:
//   codes   [R][Kp / 2] bytes, the value with the lower index in the low half; the columns behind K are zero;
//   scales  [Kp / 128][ceil(R / 64)][64] words of 4 bytes: word l = 16 * b + r of a 64-row group holds the scale of block b (of the
//           four of these 128 columns) for the rows r, 16 + r, 32 + r, 48 + r -- the order in which the lanes of
//           v_mfma_scale_f32_16x16x128_f8f6f4 take them: one coalesced 256-byte load serves four matrix instructions' rows.
#include <cmath>

#include "deepipr_host.h"

namespace {

enum { F32 = DEEPIPR_F32, BF16 = DEEPIPR_BF16, F16 = DEEPIPR_F16 };
constexpr int kThreads = 256;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
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
// four neighbours at once (the caller checked the alignment)
template <int T> __device__ __forceinline__ void store4(void *p, long long i, f32x4 v) {
    if (T == F32) {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p) + i) = v;
    } else {
        u32x2 o;
        if (T == BF16) {
            o.x = f32_to_bf16(v.x) | f32_to_bf16(v.y) << 16;
            o.y = f32_to_bf16(v.z) | f32_to_bf16(v.w) << 16;
        } else {
            o.x = f32_to_f16(v.x) | f32_to_f16(v.y) << 16;
            o.y = f32_to_f16(v.z) | f32_to_f16(v.w) << 16;
        }
        *reinterpret_cast<u32x2 *>(static_cast<unsigned short *>(p) + i) = o;
    }
}

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

template <int T, bool ROW, bool COL, bool SUM>
__global__ __launch_bounds__(kThreads) void k_mx4_quantise(const void *__restrict__ x, long long R, long long C, long long stride, int vec,
                                                           unsigned char *__restrict__ row_codes, unsigned *__restrict__ row_scales,
                                                           unsigned char *__restrict__ col_codes, unsigned *__restrict__ col_scales,
                                                           float *__restrict__ sums) {
    __shared__ float s[kQR * kQP];
    __shared__ unsigned char sc[2][256];
    const long long tiles_c = (C + kQC - 1) / kQC;
    const long long r0 = static_cast<long long>(blockIdx.x) / tiles_c * kQR, c0 = static_cast<long long>(blockIdx.x) % tiles_c * kQC;
    const int tid = threadIdx.x;
    if (vec && c0 + kQC <= C) {                          // whole 16-byte pieces
        constexpr int V = T == F32 ? 4 : 8, PER = kQC / V;
        u32x4 q[kQR * PER / kThreads];
#pragma unroll
        for (int j = 0; j < kQR * PER / kThreads; ++j) {
            const int i = j * kThreads + tid, r = i / PER, c = i % PER * V;
            const long long at = (r0 + r) * stride + c0 + c;
            q[j] = r0 + r < R ? *reinterpret_cast<const u32x4 *>(static_cast<const char *>(x) + at * (T == F32 ? 4 : 2)) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int j = 0; j < kQR * PER / kThreads; ++j) {
            const int i = j * kThreads + tid, r = i / PER, c = i % PER * V;
            float *d = s + r * kQP + c;
            if (T == F32) {
                *reinterpret_cast<u32x4 *>(d) = q[j];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    d[2 * k] = T == BF16 ? __uint_as_float(q[j][k] << 16) : f16_to_f32(q[j][k] & 0xffffu);
                    d[2 * k + 1] = T == BF16 ? __uint_as_float(q[j][k] & 0xffff0000u) : f16_to_f32(q[j][k] >> 16);
                }
            }
        }
    } else {
        for (int i = tid; i < kQR * kQC; i += kThreads) {
            const int r = i / kQC, c = i % kQC;
            s[r * kQP + c] = r0 + r < R && c0 + c < C ? load1<T>(x, (r0 + r) * stride + c0 + c) : 0.0f;
        }
    }
    __syncthreads();
    float v[32];
    if (ROW) {
        const int r = tid >> 2, b = tid & 3;
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<f32x4 *>(v + 4 * k) = *reinterpret_cast<const f32x4 *>(s + r * kQP + b * 32 + 4 * k);
        unsigned code;
        const u32x4 q = quantise32(v, code);
        if (r0 + r < R) *reinterpret_cast<u32x4 *>(row_codes + (r0 + r) * (tiles_c * (kQC / 2)) + c0 / 2 + b * 16) = q;
        sc[0][(b * 16 + (r & 15)) * 4 + (r >> 4)] = static_cast<unsigned char>(code);
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
        const long long pitch = round_up(R, 128) / 2;
        if (c0 + c < C) *reinterpret_cast<u32x4 *>(col_codes + (c0 + c) * pitch + r0 / 2 + h * 16) = q;
        sc[1][(c >> 6) * 128 + (h * 16 + (c & 15)) * 4 + ((c & 63) >> 4)] = static_cast<unsigned char>(code);
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
    if (COL && tid < 64) {
        const int g = tid >> 5;                          // of the tile's two 64-column groups
        const long long rg = c0 / 64 + g;
        if (rg < row_groups(C))
            col_scales[(r0 / 128 * row_groups(C) + rg) * 64 + (r0 / 64 & 1) * 32 + (tid & 31)] = reinterpret_cast<const unsigned *>(sc[1])[tid];
    }
}

// sums [tiles][C] -> out [C], in tile order
__global__ __launch_bounds__(kThreads) void k_mx4_colsum(const float *__restrict__ sums, long long tiles, long long C, float *__restrict__ out) {
    const long long c = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= C) return;
    double v = 0.0;
    for (long long t = 0; t < tiles; ++t) v += static_cast<double>(sums[t * C + c]);
    out[c] = static_cast<float>(v);
}

// ----------------------------------------------------------------------------------------------------------------- dequantise
// The matrix [R][K] of values, or its transpose [K][R].  A thread decodes 8 codes; the transposed form goes through LDS.
__device__ __forceinline__ unsigned scale_at(const unsigned *scales, long long rows, long long r, long long b) {
    const unsigned w = scales[((b >> 2) * row_groups(rows) + (r >> 6)) * 64 + (b & 3) * 16 + (r & 15)];
    return w >> ((r >> 4 & 3) * 8) & 0xffu;
}
__device__ __forceinline__ void decode8(unsigned w, float x, float *v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = a.x * x; v[1] = a.y * x; v[2] = b.x * x; v[3] = b.y * x;
    v[4] = c.x * x; v[5] = c.y * x; v[6] = d.x * x; v[7] = d.y * x;
}

template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_dequantise(const unsigned char *__restrict__ codes, const unsigned *__restrict__ scales,
                                                             long long R, long long K, int vec, void *__restrict__ out) {
    const long long per = (K + 7) / 8, n = R * per, pitch = round_up(K, 128) / 2;
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long r = i / per, k = i % per * 8;
        float v[8];
        decode8(*reinterpret_cast<const unsigned *>(codes + r * pitch + k / 2), scale_value(scale_at(scales, R, r, k / 32)), v);
        if (vec && k + 8 <= K) {
            store4<T>(out, r * K + k, f32x4{v[0], v[1], v[2], v[3]});
            store4<T>(out, r * K + k + 4, f32x4{v[4], v[5], v[6], v[7]});
        } else {
            for (int j = 0; j < 8 && k + j < K; ++j) store1<T>(out, r * K + k + j, v[j]);
        }
    }
}

// out [K][R]: a workgroup takes 64 rows x 64 columns of the matrix
template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_dequantise_t(const unsigned char *__restrict__ codes, const unsigned *__restrict__ scales,
                                                               long long R, long long K, void *__restrict__ out) {
    __shared__ float s[64 * 65];
    const long long tiles_r = (R + 63) / 64;
    const long long r0 = static_cast<long long>(blockIdx.x) % tiles_r * 64, k0 = static_cast<long long>(blockIdx.x) / tiles_r * 64;
    const long long pitch = round_up(K, 128) / 2;
    for (int i = threadIdx.x; i < 64 * 8; i += kThreads) {
        const int r = i >> 3, k = (i & 7) * 8;
        float v[8] = {};
        if (r0 + r < R)                                  // columns behind K lie in the padding: zero codes
            decode8(*reinterpret_cast<const unsigned *>(codes + (r0 + r) * pitch + (k0 + k) / 2),
                    scale_value(scale_at(scales, R, r0 + r, (k0 + k) / 32)), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[(k + j) * 65 + r] = v[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kThreads) {
        const int k = i >> 6, r = i & 63;
        if (k0 + k < K && r0 + r < R) store1<T>(out, (k0 + k) * R + r0 + r, s[k * 65 + r]);
    }
}

// -------------------------------------------------------------------------------------------------------------------- product
// out[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]), A [M][K] and B [N][K] quantised.  v_mfma_scale_f32_16x16x128_f8f6f4: lane l gives 32
// codes of row l % 16 (block l / 16 of the 128 columns) and that block's scale; B is the instruction's first operand, so that a lane
// holds four neighbouring n of one m.  Products and sums in 32 bits.
__device__ __forceinline__ float bias_at(const void *bias, int type, long long n) {
    return type == F32 ? load1<F32>(bias, n) : type == BF16 ? load1<BF16>(bias, n) : load1<F16>(bias, n);
}

template <int SA, int SB>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, unsigned sa, unsigned sb) {
    const i32x8 av = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w), 0, 0, 0, 0};
    const i32x8 bv = {static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, SA, static_cast<int>(sa), SB, static_cast<int>(sb));
}

template <int T>
__global__ __launch_bounds__(kThreads) void k_mx4_gemm(const unsigned char *__restrict__ a, const unsigned *__restrict__ sa,
                                                       const unsigned char *__restrict__ b, const unsigned *__restrict__ sb,
                                                       const void *__restrict__ bias, int bias_type, long long M, long long N, long long kt,
                                                       int vec, void *__restrict__ out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long tiles_n = (N + 127) / 128;
    const long long m0 = static_cast<long long>(blockIdx.x) / tiles_n * 128 + (wave >> 1) * 64;
    const long long n0 = static_cast<long long>(blockIdx.x) % tiles_n * 128 + (wave & 1) * 64;
    if (m0 >= M || n0 >= N) return;
    const long long pitch = kt * 64;
    const unsigned char *pa[4], *pb[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {                        // rows behind the end read the last one; what they give is not stored
        pa[t] = a + min(m0 + t * 16 + (lane & 15), M - 1) * pitch + (lane >> 4) * 16;
        pb[t] = b + min(n0 + t * 16 + (lane & 15), N - 1) * pitch + (lane >> 4) * 16;
    }
    const unsigned *qa = sa + m0 / 64 * 64 + lane, *qb = sb + n0 / 64 * 64 + lane;
    f32x4 acc[4][4] = {};
    for (long long k = 0; k < kt; ++k) {
        u32x4 fa[4], fb[4];
        const unsigned wa = qa[k * row_groups(M) * 64], wb = qb[k * row_groups(N) * 64];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            fa[t] = *reinterpret_cast<const u32x4 *>(pa[t] + k * 64);
            fb[t] = *reinterpret_cast<const u32x4 *>(pb[t] + k * 64);
        }
#define MX4_ROW(J)                                                                      \
        acc[0][J] = mfma<0, J>(fb[0], fa[J], acc[0][J], wb, wa);                        \
        acc[1][J] = mfma<1, J>(fb[1], fa[J], acc[1][J], wb, wa);                        \
        acc[2][J] = mfma<2, J>(fb[2], fa[J], acc[2][J], wb, wa);                        \
        acc[3][J] = mfma<3, J>(fb[3], fa[J], acc[3][J], wb, wa);
        MX4_ROW(0) MX4_ROW(1) MX4_ROW(2) MX4_ROW(3)
#undef MX4_ROW
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long n = n0 + i * 16 + (lane >> 4) * 4;
        f32x4 add = {};
        if (bias)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < N) add[j] = bias_at(bias, bias_type, n + j);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const long long m = m0 + t * 16 + (lane & 15);
            if (m >= M) continue;
            const f32x4 v = acc[i][t] + add;
            if (vec && n + 4 <= N) {
                store4<T>(out, m * N + n, v);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (n + j < N) store1<T>(out, m * N + n + j, v[j]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------- host side
inline bool good_dtype(int d) { return d == F32 || d == BF16 || d == F16; }
inline bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int elem_bytes(int d) { return d == F32 ? 4 : 2; }
constexpr long long kMaxSide = 1ll << 40, kMaxGrid = 1ll << 30;

template <int T>
void launch_quantise(DiprProf &prof, const void *x, long long R, long long C, long long stride, int vec, void *rc, void *rs, void *cc, void *cs,
                     float *sums, hipStream_t st) {
    // blocks down the columns need the padding rows' zeros too
    const long long tiles_r = cc ? round_up(R, 128) / kQR : (R + kQR - 1) / kQR, tiles_c = (C + kQC - 1) / kQC;
    const dim3 grid(static_cast<unsigned>(tiles_r * tiles_c)), block(kThreads);
#define MX4_QUANTISE(ROW, COL, SUM)                                                                                                  \
    DIPR_LAUNCH(prof, (k_mx4_quantise<T, ROW, COL, SUM>), grid, block, st, x, R, C, stride, vec, static_cast<unsigned char *>(rc),   \
                static_cast<unsigned *>(rs), static_cast<unsigned char *>(cc), static_cast<unsigned *>(cs), sums)
    if (rc && cc && sums) MX4_QUANTISE(true, true, true);
    else if (rc && cc) MX4_QUANTISE(true, true, false);
    else if (cc && sums) MX4_QUANTISE(false, true, true);
    else if (cc) MX4_QUANTISE(false, true, false);
    else MX4_QUANTISE(true, false, false);
#undef MX4_QUANTISE
}

}  // namespace

extern "C" {

size_t deepipr_mx4_code_bytes(long long rows, long long cols) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<size_t>(rows) * static_cast<size_t>(round_up(cols, 128) / 2);
}
size_t deepipr_mx4_scale_bytes(long long rows, long long cols) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<size_t>(round_up(cols, 128) / 128) * static_cast<size_t>(row_groups(rows)) * 256;
}
size_t deepipr_mx4_quantize_workspace_bytes(long long rows, long long cols) {
    return rows <= 0 || cols <= 0 ? 0 : static_cast<size_t>(round_up(rows, 128) / kQR) * static_cast<size_t>(cols) * sizeof(float);
}

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
    const long long tiles = round_up(rows, 128) / kQR * ((cols + kQC - 1) / kQC);
    if (tiles > kMaxGrid) return dipr_fail(DEEPIPR_EINVAL, "%s: matrix too large", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int vec = aligned(x, 16) && (rows == 1 || row_stride * elem_bytes(dtype) % 16 == 0);
    float *sums = col_sums ? static_cast<float *>(workspace) : nullptr;
    DiprProf prof(DEEPIPR_K_MX4_QUANTIZE);
    prof.bytes = static_cast<double>(rows) * static_cast<double>(cols) * (elem_bytes(dtype) + 0.53125 * ((row_codes ? 1 : 0) + (col_codes ? 1 : 0)));
    switch (dtype) {
        case F32: launch_quantise<F32>(prof, x, rows, cols, row_stride, vec, row_codes, row_scales, col_codes, col_scales, sums, st); break;
        case BF16: launch_quantise<BF16>(prof, x, rows, cols, row_stride, vec, row_codes, row_scales, col_codes, col_scales, sums, st); break;
        default: launch_quantise<F16>(prof, x, rows, cols, row_stride, vec, row_codes, row_scales, col_codes, col_scales, sums, st); break;
    }
    if (col_sums)
        hipLaunchKernelGGL(k_mx4_colsum, dim3(static_cast<unsigned>((cols + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, sums,
                           round_up(rows, 128) / kQR, cols, col_sums);
    return dipr_check_launch(what);
}

int deepipr_mx4_dequantize(const void *codes, const void *scales, long long rows, long long cols, int transposed, void *out, int dtype,
                           void *stream) {
    const char *what = "mx4_dequantize";
    if (!codes || !scales || !out || !good_dtype(dtype) || rows <= 0 || cols <= 0 || rows > kMaxSide || cols > kMaxSide)
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!aligned(codes, 16) || !aligned(scales, 16) || !aligned(out, elem_bytes(dtype))) return dipr_fail(DEEPIPR_EINVAL, "%s: misaligned pointer", what);
    const long long tiles = ((rows + 63) / 64) * ((cols + 63) / 64);
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
            const long long want = (rows * ((cols + 7) / 8) + kThreads - 1) / kThreads;                                              \
            const int vec = cols % 4 == 0 && aligned(out, 16);                                                                       \
            DIPR_LAUNCH(prof, (k_mx4_dequantise<T>), dim3(static_cast<unsigned>(want < 16384 ? want : 16384)), dim3(kThreads), st, c, s, rows, \
                        cols, vec, out);                                                                                             \
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

size_t deepipr_mx4_matmul_workspace_bytes(long long, long long, long long) { return 0; }

int deepipr_mx4_matmul(const void *a_codes, const void *a_scales, const void *b_codes, const void *b_scales, const void *bias, int bias_dtype,
                       long long M, long long N, long long K, void *out, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "mx4_matmul";
    if (!a_codes || !a_scales || !b_codes || !b_scales || !out || !good_dtype(dtype) || (bias && !good_dtype(bias_dtype)) || M <= 0 || N <= 0 ||
        K <= 0 || M > kMaxSide || N > kMaxSide || K > kMaxSide)
        return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!aligned(a_codes, 16) || !aligned(a_scales, 16) || !aligned(b_codes, 16) || !aligned(b_scales, 16) || !aligned(out, elem_bytes(dtype)) ||
        (bias && !aligned(bias, elem_bytes(bias_dtype))))
        return dipr_fail(DEEPIPR_EINVAL, "%s: misaligned pointer", what);
    if (workspace_bytes < deepipr_mx4_matmul_workspace_bytes(M, N, K) || (!workspace && deepipr_mx4_matmul_workspace_bytes(M, N, K)))
        return dipr_fail(DEEPIPR_EINVAL, "%s: workspace too small", what);
    const long long tiles = ((M + 127) / 128) * ((N + 127) / 128);
    if (tiles > kMaxGrid) return dipr_fail(DEEPIPR_EINVAL, "%s: matrix too large", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int vec = N % 4 == 0 && aligned(out, 4 * elem_bytes(dtype));
    DiprProf prof(DEEPIPR_K_MX4_MATMUL);
    prof.bytes = 2.0 * static_cast<double>(M) * static_cast<double>(N) * static_cast<double>(K);
#define MX4_GEMM(T)                                                                                                                  \
    DIPR_LAUNCH(prof, (k_mx4_gemm<T>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), st, static_cast<const unsigned char *>(a_codes), \
                static_cast<const unsigned *>(a_scales), static_cast<const unsigned char *>(b_codes), static_cast<const unsigned *>(b_scales), \
                bias, bias_dtype, M, N, round_up(K, 128) / 128, vec, out)
    switch (dtype) {
        case F32: MX4_GEMM(F32); break;
        case BF16: MX4_GEMM(BF16); break;
        default: MX4_GEMM(F16); break;
    }
#undef MX4_GEMM
    return dipr_check_launch(what);
}

}  // extern "C"
