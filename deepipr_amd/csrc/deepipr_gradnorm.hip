// deepipr_gradnorm.hip -- translation unit of libdeepipr_hip.so: the global norm of a list of tensors, the list scaled down to a
// largest norm, and the SGD step behind that clipping.
//
// Mathematics: n = (sum over all elements of all tensors of |g|^p)^(1/p), p = 1, 2 or infinity; f = min(1, max_norm / (n + 1e-6)).
// Squares and sums are held in 64 bits (1e30 and 1e-30 square without leaving the range), summed in a fixed order.
//
// What bounds it: bytes.  The norm reads every gradient once; clipping reads and writes them once more; the step reads gradient,
// parameter and momentum and writes the last two.  The list travels in the launch arguments (240 tensors a launch): no table in
// device memory, no copy in front of the launch, and a captured launch keeps its own list.
//
// Work split: the tensors are laid end to end in units of 64 elements (a tensor's last unit may be short) and cut into runs of up to 256
// units, across tensor borders where they fall: tensors of any sizes load all workgroups alike.  At most 1024 workgroups a launch take
// the runs in turn.  Each leaves one partial sum; the next launch's workgroups each add all of them up (8 KB from L2) instead of a launch
// in between.  The step's run space is the flat parameter buffer itself (parameters start on multiples of 64 floats there).
// Measured: norm + clip of 391 odd bf16 tensors (0.54 GB, just written by a copy) 446 us, the copy included 4.7 TB/s; the clipped step of
// 61 M parameters 292 us = 5.0 TB/s; a large copy reaches 4.7 to 5.0 on this card.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "deepipr_host.h"

namespace {

constexpr int kThreads = 256;
constexpr int kEntries = 240;                 // entries per launch: 240 * 16 bytes of the 4 KB of launch arguments
constexpr int kMaxGroups = 1024;              // workgroups per launch: 4 of 4 waves per CU
// A run is 1024 to 16384 elements: a workgroup takes about 0.1 us (clip 0.2) for every tensor in its run (measured: 20 000 elements in 239
// tensors 14 us with runs of 1024 at least, 40 with 4096; a million in 100 11 / 9).
constexpr unsigned kMinUnits = 16, kMaxUnits = 256;
constexpr int kMaxPartials = 4096;            // workgroups of all launches of one list
constexpr int kOneThreads = 1024;
constexpr unsigned long long kOneUnits = 128; // up to 8192 elements in up to 4 tensors: one workgroup, one launch (5130 in two 5.4 us,
constexpr int kOneEntries = 4;                // 7.0 in two launches, and one launch less on the host; 16384 in two 6.6 / 5.8)
constexpr long long kEntryMax = 1ll << 29;    // elements per entry; longer tensors take several entries
constexpr double kClipEps = 1e-6;

enum { F32 = DEEPIPR_F32, BF16 = DEEPIPR_BF16, F16 = DEEPIPR_F16 };

struct List {
    const void *ptr[kEntries];
    unsigned count[kEntries];                 // elements | dtype << 30
    unsigned start[kEntries];                 // first unit of the entry in this launch's run space
    unsigned long long base;                  // step only: the place of unit 0 in param / momentum, in units of 64 floats
    int n;
    unsigned units;                           // of the whole launch
    unsigned per;                             // units per run
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_to_f32(unsigned short h) { return __uint_as_float(static_cast<unsigned>(h) << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float f) {          // nearest, ties to even; NaN stays NaN
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<unsigned short>((u >> 16) | 0x40u);
    return static_cast<unsigned short>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float f16_to_f32(unsigned short h) {
    _Float16 v;
    __builtin_memcpy(&v, &h, 2);
    return static_cast<float>(v);
}
__device__ __forceinline__ unsigned short f32_to_f16(float f) {
    const _Float16 v = static_cast<_Float16>(f);
    unsigned short h;
    __builtin_memcpy(&h, &v, 2);
    return h;
}

template <int T> struct Elem;
template <> struct Elem<F32> {
    typedef float type;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<BF16> {
    typedef unsigned short type;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(unsigned short v) { return bf16_to_f32(v); }
    static __device__ __forceinline__ unsigned short put(float v) { return f32_to_bf16(v); }
};
template <> struct Elem<F16> {
    typedef unsigned short type;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(unsigned short v) { return f16_to_f32(v); }
    static __device__ __forceinline__ unsigned short put(float v) { return f32_to_f16(v); }
};

template <int T> union Pack {
    u32x4 q;
    typename Elem<T>::type e[Elem<T>::kVec];
};

// P = 2: sum of squares, 1: sum of magnitudes, 0: largest magnitude (a NaN wins and stays)
template <int P> __device__ __forceinline__ void take(double &acc, float v) {
    if (P == 2) {
        const double d = v;
        acc = fma(d, d, acc);
    } else if (P == 1) {
        acc += static_cast<double>(fabsf(v));
    } else {
        const double d = fabsf(v);
        if (d > acc || d != d) acc = d;
    }
}
template <int P> __device__ __forceinline__ double join(double a, double b) {
    if (P) return a + b;
    return (b > a || b != b) ? b : a;
}

template <int P> __device__ __forceinline__ double wave_join(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = join<P>(v, __shfl_xor(v, off, 64));
    return v;
}
// The same value in every thread; `red`: a double of LDS for each of the TH / 64 waves
template <int P, int TH> __device__ __forceinline__ double block_join(double v, double *red) {
    v = wave_join<P>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = join<P>(join<P>(red[0], red[1]), join<P>(red[2], red[3]));
#pragma unroll
    for (int i = 4; i < TH / 64; ++i) r = join<P>(r, red[i]);
    __syncthreads();
    return r;
}

// The entry that holds unit u: the last one whose start is <= u
__device__ __forceinline__ int entry_of(const List &L, unsigned u) {
    int lo = 0, hi = L.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (L.start[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Calls f(entry, first element, end element) for the pieces of this workgroup's runs, in order
template <class F> __device__ __forceinline__ void walk(const List &L, F f) {
    for (unsigned lo = blockIdx.x * L.per; lo < L.units; lo += gridDim.x * L.per) {
        const unsigned hi = min(lo + L.per, L.units);
        for (int i = entry_of(L, lo); i < L.n && L.start[i] < hi; ++i) {
            const unsigned n = L.count[i] & 0x3fffffffu;
            const unsigned s = L.start[i];
            const unsigned long long a = lo > s ? (lo - s) * 64ull : 0ull;
            const unsigned b = min((hi - s) * 64ull, static_cast<unsigned long long>(n));
            if (a < b) f(i, static_cast<unsigned>(a), b);              // (a >= b: a gap in front of the next entry)
        }
    }
}

template <int T, int P, int TH>
__device__ __forceinline__ void norm_piece(const void *base, unsigned a, unsigned b, double *acc) {
    typedef typename Elem<T>::type E;
    constexpr int V = Elem<T>::kVec;
    const E *p = static_cast<const E *>(base) + a;
    unsigned n = b - a;
    // up to the first 16-byte boundary by single elements (torch aligns storages, but a tensor may start anywhere in one)
    const unsigned head = min(n, static_cast<unsigned>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(E)));
    if (threadIdx.x < head) take<P>(acc[0], Elem<T>::get(p[threadIdx.x]));
    p += head;
    n -= head;
    const u32x4 *q = reinterpret_cast<const u32x4 *>(p);
    const unsigned nv = n / V;
    unsigned i = threadIdx.x;
    for (; i + 3 * TH < nv; i += 4 * TH) {
        Pack<T> v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j].q = q[i + j * TH];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) take<P>(acc[k & 3], Elem<T>::get(v[j].e[k]));
    }
    for (; i < nv; i += TH) {
        Pack<T> v;
        v.q = q[i];
#pragma unroll
        for (int k = 0; k < V; ++k) take<P>(acc[k & 3], Elem<T>::get(v.e[k]));
    }
    const unsigned rest = n - nv * V;
    if (threadIdx.x < rest) take<P>(acc[0], Elem<T>::get(p[nv * V + threadIdx.x]));
}

// This workgroup's part of the sum, in every thread
template <int P, int TH> __device__ __forceinline__ double norm_runs(const List &L, double *red) {
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    walk(L, [&](int i, unsigned a, unsigned b) {
        const void *p = L.ptr[i];
        switch (L.count[i] >> 30) {
            case F32: norm_piece<F32, P, TH>(p, a, b, acc); break;
            case BF16: norm_piece<BF16, P, TH>(p, a, b, acc); break;
            default: norm_piece<F16, P, TH>(p, a, b, acc); break;
        }
    });
    return block_join<P, TH>(join<P>(join<P>(acc[0], acc[1]), join<P>(acc[2], acc[3])), red);
}
template <int P>
__global__ __launch_bounds__(kThreads) void k_norm_partials(const List L, double *__restrict__ part) {
    __shared__ double red[4];
    const double s = norm_runs<P, kThreads>(L, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm out of the partial sums, the same in every thread
template <int P> __device__ __forceinline__ double norm_of(const double *__restrict__ part, int n, double *red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) v = join<P>(v, part[i]);
    v = block_join<P, kThreads>(v, red);
    return P == 2 ? sqrt(v) : v;
}

// min(1, max / (n + eps)); NaN and infinity go the way of the arithmetic: a NaN norm gives NaN, an infinite one 0.  The factor and its
// product with a gradient are held in 64 bits: a norm near the end of float's range would leave a float factor with few digits.  The
// product is rounded to 32 bits, and for 16-bit tensors again to their type: next to a border that can be the other neighbour (an
// error of half a step and 2^-24 of the value).
__device__ __forceinline__ double factor_of(double norm, float max_norm) {
    const double f = static_cast<double>(max_norm) / (norm + kClipEps);
    return f >= 1.0 ? 1.0 : f;
}
__device__ __forceinline__ float times(double f, float g) { return static_cast<float>(f * static_cast<double>(g)); }

template <int P>
__global__ __launch_bounds__(kThreads) void k_norm_finish(const double *__restrict__ part, int n, float *__restrict__ norm) {
    __shared__ double red[4];
    const double v = norm_of<P>(part, n, red);
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
}

template <int T, int TH>
__device__ __forceinline__ void scale_piece(void *base, unsigned a, unsigned b, double f) {
    typedef typename Elem<T>::type E;
    constexpr int V = Elem<T>::kVec;
    E *p = static_cast<E *>(base) + a;
    unsigned n = b - a;
    const unsigned head = min(n, static_cast<unsigned>(((16u - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(E)));
    if (threadIdx.x < head) p[threadIdx.x] = Elem<T>::put(times(f, Elem<T>::get(p[threadIdx.x])));
    p += head;
    n -= head;
    u32x4 *q = reinterpret_cast<u32x4 *>(p);
    const unsigned nv = n / V;
    unsigned i = threadIdx.x;
    for (; i + 3 * TH < nv; i += 4 * TH) {
        Pack<T> v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j].q = q[i + j * TH];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int k = 0; k < V; ++k) v[j].e[k] = Elem<T>::put(times(f, Elem<T>::get(v[j].e[k])));
            q[i + j * TH] = v[j].q;
        }
    }
    for (; i < nv; i += TH) {
        Pack<T> v;
        v.q = q[i];
#pragma unroll
        for (int k = 0; k < V; ++k) v.e[k] = Elem<T>::put(times(f, Elem<T>::get(v.e[k])));
        q[i] = v.q;
    }
    const unsigned rest = n - nv * V;
    if (threadIdx.x < rest) p[nv * V + threadIdx.x] = Elem<T>::put(times(f, Elem<T>::get(p[nv * V + threadIdx.x])));
}

template <int TH> __device__ __forceinline__ void scale_runs(const List &L, double f) {
    walk(L, [&](int i, unsigned a, unsigned b) {
        void *p = const_cast<void *>(L.ptr[i]);
        switch (L.count[i] >> 30) {
            case F32: scale_piece<F32, TH>(p, a, b, f); break;
            case BF16: scale_piece<BF16, TH>(p, a, b, f); break;
            default: scale_piece<F16, TH>(p, a, b, f); break;
        }
    });
}
// A factor of exactly 1 leaves every value as it is (1 * x = x in every type): nothing is read or written then.
template <int P>
__global__ __launch_bounds__(kThreads) void k_clip(const List L, const double *__restrict__ part, int n, float max_norm,
                                                   float *__restrict__ norm) {
    __shared__ double red[4];
    const double v = norm_of<P>(part, n, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(v);
    const double f = factor_of(v, max_norm);
    if (f != 1.0) scale_runs<kThreads>(L, f);
}

// A short list in one launch of one workgroup: the norm and, if CLIP, the scaling
template <int P, bool CLIP>
__global__ __launch_bounds__(kOneThreads) void k_one(const List L, float max_norm, float *__restrict__ norm) {
    __shared__ double red[kOneThreads / 64];
    double v = norm_runs<P, kOneThreads>(L, red);
    if (P == 2) v = sqrt(v);
    if (threadIdx.x == 0) *norm = static_cast<float>(v);
    if (!CLIP) return;
    const double f = factor_of(v, max_norm);
    if (f != 1.0) scale_runs<kOneThreads>(L, f);
}

__device__ __forceinline__ void sgd1(float &p, float g, float &buf, float lr, float mu, float wd, double gs) {
    const float d = fmaf(wd, p, times(gs, g));
    buf = fmaf(mu, buf, d);
    p = fmaf(-lr, buf, p);
}

// hp = {lr, momentum, weight decay, grad scale, max norm}; the norm is that of the scaled gradients.  Unclipped (factor 1) the
// arithmetic is the plain step's, bit for bit.
__global__ __launch_bounds__(kThreads) void k_sgd_clipped(const List L, const double *__restrict__ part, int n,
                                                          float *__restrict__ param, float *__restrict__ buf,
                                                          const float *__restrict__ hp, float *__restrict__ norm) {
    __shared__ double red[4];
    const float lr = hp[0], mu = hp[1], wd = hp[2];
    const double v = norm_of<2>(part, n, red) * fabs(static_cast<double>(hp[3]));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = static_cast<float>(v);
    const double gs = factor_of(v, hp[4]) * static_cast<double>(hp[3]);
    walk(L, [&](int i, unsigned a, unsigned b) {
        const float *g = static_cast<const float *>(L.ptr[i]) + a;
        const size_t off = static_cast<size_t>(L.base + L.start[i]) * 64 + a;
        float *p = param + off, *m = buf + off;
        const unsigned len = b - a;
        unsigned done = 0;
        if ((reinterpret_cast<uintptr_t>(g) & 15u) == 0) {       // param / buf pieces start on 256-byte boundaries (host check)
            const unsigned nv = len / 4;
            const float4 *g4 = reinterpret_cast<const float4 *>(g);
            float4 *p4 = reinterpret_cast<float4 *>(p), *m4 = reinterpret_cast<float4 *>(m);
            unsigned j = threadIdx.x;
            for (; j + kThreads < nv; j += 2 * kThreads) {
                float4 gv[2], pv[2], mv[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    gv[k] = g4[j + k * kThreads];
                    pv[k] = p4[j + k * kThreads];
                    mv[k] = m4[j + k * kThreads];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    sgd1(pv[k].x, gv[k].x, mv[k].x, lr, mu, wd, gs);
                    sgd1(pv[k].y, gv[k].y, mv[k].y, lr, mu, wd, gs);
                    sgd1(pv[k].z, gv[k].z, mv[k].z, lr, mu, wd, gs);
                    sgd1(pv[k].w, gv[k].w, mv[k].w, lr, mu, wd, gs);
                    p4[j + k * kThreads] = pv[k];
                    m4[j + k * kThreads] = mv[k];
                }
            }
            for (; j < nv; j += kThreads) {
                const float4 gv = g4[j];
                float4 pv = p4[j], mv = m4[j];
                sgd1(pv.x, gv.x, mv.x, lr, mu, wd, gs);
                sgd1(pv.y, gv.y, mv.y, lr, mu, wd, gs);
                sgd1(pv.z, gv.z, mv.z, lr, mu, wd, gs);
                sgd1(pv.w, gv.w, mv.w, lr, mu, wd, gs);
                p4[j] = pv;
                m4[j] = mv;
            }
            done = nv * 4;
        }
        for (unsigned j = done + threadIdx.x; j < len; j += kThreads) sgd1(p[j], g[j], m[j], lr, mu, wd, gs);
    });
}

// ------------------------------------------------------------------------------------------------------------------- host side
inline size_t elem_bytes(long long dtype) { return dtype == F32 ? 4 : 2; }
inline bool good_dtype(long long d) { return d == F32 || d == BF16 || d == F16; }

// Checks the caller's arrays; -> units of the whole list and the number of entries, or a negative code.
int survey(const char *what, const DeepiprTensor *t, int n, size_t *elements, unsigned long long *units, size_t *bytes) {
    if (n < 0 || (n && !t)) return dipr_fail(DEEPIPR_EINVAL, "%s: bad list", what);
    *elements = *bytes = 0;
    *units = 0;
    for (int i = 0; i < n; ++i) {
        if (t[i].count < 0 || !good_dtype(t[i].dtype) || (t[i].count && !t[i].data))
            return dipr_fail(DEEPIPR_EINVAL, "%s: bad tensor %d", what, i);
        if (reinterpret_cast<uintptr_t>(t[i].data) % elem_bytes(t[i].dtype))
            return dipr_fail(DEEPIPR_EINVAL, "%s: tensor %d is not aligned to its type", what, i);
        *elements += static_cast<size_t>(t[i].count);
        *units += (static_cast<unsigned long long>(t[i].count) + 63) / 64;
        *bytes += static_cast<size_t>(t[i].count) * elem_bytes(t[i].dtype);
    }
    // a launch's units are counted in 32 bits: 240 entries of 2^29 elements stay below
    if (*elements >= (1ull << 42)) return dipr_fail(DEEPIPR_EINVAL, "%s: more than 2^42 elements", what);
    return DEEPIPR_OK;
}

// Two entries of a list that is WRITTEN must not share memory (two workgroups would read and write the same element): -> the code of
// the refusal.  span(t): the first and the end address of an entry, in any unit.
template <class F> int disjoint(const char *what, const DeepiprTensor *t, int n, F span) {
    typedef std::pair<unsigned long long, unsigned long long> Span;
    Span few[64], *all = n <= 64 ? few : new (std::nothrow) Span[n];
    if (!all) return dipr_fail(DEEPIPR_EINVAL, "%s: out of host memory", what);
    int m = 0;
    for (int i = 0; i < n; ++i)
        if (t[i].count) all[m++] = span(t[i]);
    std::sort(all, all + m);
    bool ok = true;
    for (int i = 1; i < m; ++i) ok = ok && all[i].first >= all[i - 1].second;
    if (all != few) delete[] all;
    return ok ? DEEPIPR_OK : dipr_fail(DEEPIPR_EINVAL, "%s: two tensors of the list share memory", what);
}

inline long long entries_of(const DeepiprTensor *t, int n) {
    long long entries = 0;
    for (int i = 0; i < n; ++i) entries += (t[i].count + kEntryMax - 1) / kEntryMax;
    return entries;
}
// How a list is cut: units per run, workgroups per launch (0: more launches than kMaxPartials partial sums allow)
struct Cut {
    unsigned per, groups;
};
inline Cut cut(const DeepiprTensor *t, int n, unsigned long long units) {
    const unsigned long long launches = static_cast<unsigned long long>((entries_of(t, n) + kEntries - 1) / kEntries);
    if (launches > kMaxPartials) return Cut{1, 0};
    const unsigned long long most = launches ? kMaxPartials / launches : 1;
    Cut c;
    c.groups = static_cast<unsigned>(most < kMaxGroups ? most : kMaxGroups);
    unsigned long long per = units / c.groups / (launches ? launches : 1);
    if (per > kMaxUnits) per = kMaxUnits;
    if (per < kMinUnits) per = kMinUnits;
    c.per = static_cast<unsigned>((per + 3) / 4 * 4);
    return c;
}

// Cuts the list into launches and calls f(list, workgroups) for each; f returns false to stop.  PLACED: units are those of the entries'
// offsets (in ascending order) instead of end to end.
template <bool PLACED, class F> bool launches(const DeepiprTensor *t, int n, const Cut &c, F f) {
    const unsigned per = c.per, groups = c.groups;
    List L;
    L.n = 0;
    L.units = 0;
    L.per = per;
    L.base = 0;
    auto flush = [&]() {
        if (!L.n) return true;
        const unsigned runs = (L.units + per - 1) / per;
        const bool ok = f(L, static_cast<int>(runs < groups ? runs : groups));
        L.n = 0;
        L.units = 0;
        return ok;
    };
    for (int i = 0; i < n; ++i) {
        long long at = 0;
        while (at < t[i].count) {
            const long long len = t[i].count - at < kEntryMax ? t[i].count - at : kEntryMax;
            if (PLACED) {
                const unsigned long long place = static_cast<unsigned long long>(t[i].offset + at) / 64;
                if (L.n && place - L.base > (1u << 30) && !flush()) return false;          // start stays within 32 bits
                if (!L.n) L.base = place;
                L.units = static_cast<unsigned>(place - L.base);
            }
            L.ptr[L.n] = static_cast<const char *>(t[i].data) + at * elem_bytes(t[i].dtype);
            L.count[L.n] = static_cast<unsigned>(len) | static_cast<unsigned>(t[i].dtype) << 30;
            L.start[L.n] = L.units;
            L.units += static_cast<unsigned>((len + 63) / 64);
            at += len;
            if (++L.n == kEntries && !flush()) return false;
        }
    }
    return flush();
}

// Every launch is timed by itself, with its own bytes.
inline double bytes_of(const List &L) {
    double bytes = 0.0;
    for (int i = 0; i < L.n; ++i) bytes += static_cast<double>(L.count[i] & 0x3fffffffu) * static_cast<double>(elem_bytes(L.count[i] >> 30));
    return bytes;
}

template <int P> int partials(const char *what, const DeepiprTensor *t, int n, const Cut &per, double *part, int *used, hipStream_t st) {
    int at = 0;
    const bool ok = launches<false>(t, n, per, [&](const List &L, int runs) {
        if (at + runs > kMaxPartials) return false;
        DiprProf prof(DEEPIPR_K_GRAD_NORM);
        if (prof.a) prof.bytes = bytes_of(L);
        DIPR_LAUNCH(prof, (k_norm_partials<P>), dim3(runs), dim3(kThreads), st, L, part + at);
        at += runs;
        return true;
    });
    *used = at;
    if (!ok) return dipr_fail(DEEPIPR_EINVAL, "%s: more tensors than %d partial sums cover", what, kMaxPartials);
    return dipr_check_launch(what);
}

// A list that one workgroup takes
inline bool is_short(const DeepiprTensor *t, int n, unsigned long long units) { return units <= kOneUnits && entries_of(t, n) <= kOneEntries; }
template <bool CLIP> int one(const char *what, const DeepiprTensor *t, int n, unsigned long long units, int norm_type, size_t bytes, float max_norm,
                             float *norm, hipStream_t st) {
    DiprProf prof(CLIP ? DEEPIPR_K_GRAD_CLIP : DEEPIPR_K_GRAD_NORM);
    prof.bytes = (CLIP ? 3.0 : 1.0) * static_cast<double>(bytes);
    launches<false>(t, n, Cut{static_cast<unsigned>(units), 1}, [&](const List &L, int) {
        const dim3 grid(1), block(kOneThreads);
        switch (norm_type) {
            case 2: DIPR_LAUNCH(prof, (k_one<2, CLIP>), grid, block, st, L, max_norm, norm); break;
            case 1: DIPR_LAUNCH(prof, (k_one<1, CLIP>), grid, block, st, L, max_norm, norm); break;
            default: DIPR_LAUNCH(prof, (k_one<0, CLIP>), grid, block, st, L, max_norm, norm); break;
        }
        return true;
    });
    return dipr_check_launch(what);
}

int check_common(const char *what, int norm_type, const void *workspace, size_t workspace_bytes) {
    if (norm_type != 0 && norm_type != 1 && norm_type != 2) return dipr_fail(DEEPIPR_EINVAL, "%s: norm_type 0 (infinity), 1 or 2", what);
    if (!workspace || workspace_bytes < kMaxPartials * sizeof(double))
        return dipr_fail(DEEPIPR_EINVAL, "%s: workspace too small", what);
    if (reinterpret_cast<uintptr_t>(workspace) & 7u) return dipr_fail(DEEPIPR_EINVAL, "%s: workspace not aligned to 8 bytes", what);
    return DEEPIPR_OK;
}

int list_partials(const char *what, const DeepiprTensor *t, int n, int norm_type, const Cut &per, double *part, int *used, hipStream_t st) {
    switch (norm_type) {
        case 2: return partials<2>(what, t, n, per, part, used, st);
        case 1: return partials<1>(what, t, n, per, part, used, st);
        default: return partials<0>(what, t, n, per, part, used, st);
    }
}

}  // namespace

extern "C" {

size_t deepipr_grad_norm_workspace_bytes(void) { return kMaxPartials * sizeof(double); }

int deepipr_grad_norm(const DeepiprTensor *tensors, int n, int norm_type, float *norm, void *workspace, size_t workspace_bytes,
                      void *stream) {
    const char *what = "grad_norm";
    size_t elements, bytes;
    unsigned long long units;
    if (!norm) return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    int rc = check_common(what, norm_type, workspace, workspace_bytes);
    if (rc == DEEPIPR_OK) rc = survey(what, tensors, n, &elements, &units, &bytes);
    if (rc != DEEPIPR_OK) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    double *part = static_cast<double *>(workspace);
    const Cut per = cut(tensors, n, units);
    if (!per.groups) return dipr_fail(DEEPIPR_EINVAL, "%s: too many tensors", what);
    if (elements && is_short(tensors, n, units)) return one<false>(what, tensors, n, units, norm_type, bytes, 0.0f, norm, st);
    int used = 0;
    if (elements) {
        rc = list_partials(what, tensors, n, norm_type, per, part, &used, st);
        if (rc != DEEPIPR_OK) return rc;
    }
    DiprProf prof(DEEPIPR_K_GRAD_NORM);
    prof.bytes = used * 8.0;
    switch (norm_type) {
        case 2: DIPR_LAUNCH(prof, k_norm_finish<2>, dim3(1), dim3(kThreads), st, part, used, norm); break;
        case 1: DIPR_LAUNCH(prof, k_norm_finish<1>, dim3(1), dim3(kThreads), st, part, used, norm); break;
        default: DIPR_LAUNCH(prof, k_norm_finish<0>, dim3(1), dim3(kThreads), st, part, used, norm); break;
    }
    return dipr_check_launch(what);
}

int deepipr_grad_clip(const DeepiprTensor *tensors, int n, int norm_type, float max_norm, float *norm, void *workspace,
                      size_t workspace_bytes, void *stream) {
    const char *what = "grad_clip";
    size_t elements, bytes;
    unsigned long long units;
    if (!norm) return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if (!(max_norm >= 0.0f)) return dipr_fail(DEEPIPR_EINVAL, "%s: max_norm must not be negative or NaN", what);
    int rc = check_common(what, norm_type, workspace, workspace_bytes);
    if (rc == DEEPIPR_OK) rc = survey(what, tensors, n, &elements, &units, &bytes);
    if (rc != DEEPIPR_OK) return rc;
    if (!elements) return deepipr_grad_norm(tensors, n, norm_type, norm, workspace, workspace_bytes, stream);
    rc = disjoint(what, tensors, n, [](const DeepiprTensor &t) {
        const unsigned long long a = reinterpret_cast<uintptr_t>(t.data);
        return std::make_pair(a, a + static_cast<unsigned long long>(t.count) * elem_bytes(t.dtype));
    });
    if (rc != DEEPIPR_OK) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    double *part = static_cast<double *>(workspace);
    const Cut per = cut(tensors, n, units);
    if (!per.groups) return dipr_fail(DEEPIPR_EINVAL, "%s: too many tensors", what);
    if (is_short(tensors, n, units)) return one<true>(what, tensors, n, units, norm_type, bytes, max_norm, norm, st);
    int used = 0;
    rc = list_partials(what, tensors, n, norm_type, per, part, &used, st);
    if (rc != DEEPIPR_OK) return rc;
    launches<false>(tensors, n, per, [&](const List &L, int runs) {
        DiprProf prof(DEEPIPR_K_GRAD_CLIP);
        if (prof.a) prof.bytes = 2.0 * bytes_of(L);
        switch (norm_type) {
            case 2: DIPR_LAUNCH(prof, (k_clip<2>), dim3(runs), dim3(kThreads), st, L, part, used, max_norm, norm); break;
            case 1: DIPR_LAUNCH(prof, (k_clip<1>), dim3(runs), dim3(kThreads), st, L, part, used, max_norm, norm); break;
            default: DIPR_LAUNCH(prof, (k_clip<0>), dim3(runs), dim3(kThreads), st, L, part, used, max_norm, norm); break;
        }
        return true;
    });
    return dipr_check_launch(what);
}

int deepipr_sgd_momentum_step_clipped(float *param, float *momentum_buf, const DeepiprTensor *grads, int n, const float *hyper,
                                      float *norm, void *workspace, size_t workspace_bytes, void *stream) {
    const char *what = "sgd_momentum_step_clipped";
    size_t elements, bytes;
    unsigned long long units;
    if (!param || !momentum_buf || !hyper || !norm || n <= 0) return dipr_fail(DEEPIPR_EINVAL, "%s: bad argument", what);
    if ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(momentum_buf)) & 15u)
        return dipr_fail(DEEPIPR_EINVAL, "%s: param and momentum_buf must be 16-byte aligned", what);
    int rc = check_common(what, 2, workspace, workspace_bytes);
    if (rc == DEEPIPR_OK) rc = survey(what, grads, n, &elements, &units, &bytes);
    if (rc != DEEPIPR_OK) return rc;
    long long end = 0;
    for (int i = 0; i < n; ++i) {
        if (grads[i].dtype != F32 || grads[i].offset % 64 || grads[i].offset < end || grads[i].offset >= (1ll << 42))
            return dipr_fail(DEEPIPR_EINVAL, "%s: gradient %d: float32, its place a multiple of 64 floats behind the one before", what, i);
        end = grads[i].offset + grads[i].count;
    }
    if (!elements) return dipr_fail(DEEPIPR_EINVAL, "%s: nothing to update", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    double *part = static_cast<double *>(workspace);
    const Cut per = cut(grads, n, units);
    if (!per.groups) return dipr_fail(DEEPIPR_EINVAL, "%s: too many tensors", what);
    int used = 0;
    rc = list_partials(what, grads, n, 2, per, part, &used, st);
    if (rc != DEEPIPR_OK) return rc;
    launches<true>(grads, n, per, [&](const List &L, int runs) {
        DiprProf prof(DEEPIPR_K_SGD);
        if (prof.a) prof.bytes = 5.0 * bytes_of(L);
        DIPR_LAUNCH(prof, k_sgd_clipped, dim3(runs), dim3(kThreads), st, L, part, used, param, momentum_buf, hyper, norm);
        return true;
    });
    return dipr_check_launch(what);
}

}  // extern "C"
