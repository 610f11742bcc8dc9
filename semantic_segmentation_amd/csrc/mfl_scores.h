// Shared by the kernels that read rows of scores (mfl_top_labels.hip, mfl_distillation.hip, mfl_sample_labels.hip).
//
// A row is one distribution over C labels.  Scores are reached as element (n, c, s) of [N][C][S] with any three strides,
// so that a pixel of a label map (class planes, pixel stride 1), a line of a score matrix (S = 1, class stride 1) and a
// channels-last map (class stride 1, pixel stride C) are all read where they lie.  Row r = n * S + s.
#ifndef MFL_SCORES_H
#define MFL_SCORES_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mfl.h"

namespace mfl_scores {

struct Rows {
    const void *p;
    long long sn, sc, ss;       // strides in elements
    unsigned rows, S;           // N * S rows, S of them per n
    int C;
};

// 16-bit scores travel as their bit patterns
struct bf16_t { uint16_t u; };
struct f16_t { _Float16 h; };

__device__ inline float to_float(float v) { return v; }
__device__ inline float to_float(bf16_t v) { return __builtin_bit_cast(float, (uint32_t)v.u << 16); }
__device__ inline float to_float(f16_t v) { return (float)v.h; }

// one rounding, to nearest even; a NaN stays one
__device__ inline void from_float(float v, float &o) { o = v; }
__device__ inline void from_float(float v, f16_t &o) { o.h = (_Float16)v; }
__device__ inline void from_float(float v, bf16_t &o) { o.u = __builtin_bit_cast(uint16_t, (__bf16)v); }

// 16 bytes of scores at any address of their type (the hardware takes unaligned vector accesses)
typedef uint32_t words4 __attribute__((ext_vector_type(4)));
typedef words4 words4_at2 __attribute__((aligned(2)));
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
template <typename T> __device__ inline words4 load_words(const T *p) { return *(const words4_at2 *)p; }
// ... of data that is not read again soon
template <typename T> __device__ inline words4 load_words_once(const T *p) { return __builtin_nontemporal_load((const words4_at2 *)p); }
template <typename T> __device__ inline void unpack(words4 w, float (&x)[kVec<T>])
{
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) {
        // (a copy: a bit cast of a vector's element takes its first one)
        const uint32_t u = w[sizeof(T) == 4 ? i : i / 2];
        if constexpr (sizeof(T) == 4) x[i] = __builtin_bit_cast(float, u);
        else x[i] = to_float(__builtin_bit_cast(T, (uint16_t)(u >> (16 * (i & 1)))));
    }
}
template <typename T> __device__ inline void load_vec(const T *p, float (&x)[kVec<T>]) { unpack<T>(load_words(p), x); }
// (streamed past the caches: a gradient of many labels does not stay in them)
template <typename T> __device__ inline void store_vec(T *p, const float (&x)[kVec<T>])
{
    words4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __builtin_bit_cast(uint32_t, x[i]);
        } else {
            T lo, hi;
            from_float(x[2 * i], lo);
            from_float(x[2 * i + 1], hi);
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | (uint32_t)__builtin_bit_cast(uint16_t, hi) << 16;
        }
    }
    __builtin_nontemporal_store(w, (words4_at2 *)p);
}

// Values of a tensor whose type is known at run time only (the teacher's side): all bits first, so that the loads of a
// block are in flight together, then the conversion
template <int N, typename At> __device__ inline void load_any(float (&v)[N], const void *p, int dtype, At at)
{
    uint32_t raw[N];
    if (dtype == MFL_F32) {
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j] = ((const uint32_t *)p)[at(j)];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j] = ((const uint16_t *)p)[at(j)];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float h = (float)__builtin_bit_cast(_Float16, (uint16_t)raw[j]);
        const float b = __builtin_bit_cast(float, dtype == MFL_BF16 ? raw[j] << 16 : raw[j]);
        v[j] = dtype == MFL_F16 ? h : b;
    }
}

// one score, streamed past the caches
template <typename T> __device__ inline void store_once(float v, T *p)
{
    T o;
    from_float(v, o);
    if constexpr (sizeof(T) == 4) __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, o), (uint32_t *)p);
    else __builtin_nontemporal_store(__builtin_bit_cast(uint16_t, o), (uint16_t *)p);
}

// Order of scores as signed integers: -inf < ... < -0 = +0 < ... < +inf < NaN
__device__ inline int score_key(float v)
{
    int u = __builtin_bit_cast(int, v);
    u = u == (int)0x80000000 ? 0 : u;
    u = (u & 0x7fffffff) > 0x7f800000 ? 0x7fffffff : u;
    return u ^ ((u >> 31) & 0x7fffffff);
}
__device__ inline float key_score(int k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }

// Order of a row's labels: larger score first, the lower label first among equals; no two labels share a rank key
__device__ inline uint64_t rank_key(int key, int c) { return (uint64_t)((uint32_t)key ^ 0x80000000u) << 32 | (uint32_t)~c; }
__device__ inline int rank_label(uint64_t k) { return (int)~(uint32_t)k; }
__device__ inline float rank_score(uint64_t k) { return key_score((int)((uint32_t)(k >> 32) ^ 0x80000000u)); }

// larger of two, NaN if one is
__device__ inline float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// The K best labels of a row in one lane's registers, best first.  A label and its score are one 64-bit number, the score's
// order above 20 bits of the label's complement, kept as a double in [1, 2) (0: none): the double-precision maximum and
// minimum, which run at the vector unit's full rate, then do with two instructions a place what a compare, a median and two
// selects do on separate words (45 against 23 per score at K = 8).
constexpr int kBestLabels = 1 << 20;            // labels a place can name
__device__ inline double larger(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ inline double smaller(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ inline double place_of(float x, int c)
{
    x += 0.f;                                   // -0 becomes +0
    uint32_t u = x == x ? __builtin_bit_cast(uint32_t, x) : 0x7fffffffu;
    u ^= (uint32_t)((int)u >> 31) | 0x80000000u;
    const uint32_t hi = __builtin_amdgcn_alignbit(0x3ffu, u, 12), lo = u << 20 | (uint32_t)(kBestLabels - 1 - c);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ inline float place_score(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t u = __builtin_amdgcn_alignbit((uint32_t)(b >> 32), (uint32_t)b, 20);
    return __builtin_bit_cast(float, u ^ ((uint32_t)((int)~u >> 31) | 0x80000000u));
}
__device__ inline int place_label(double v) { return kBestLabels - 1 - (int)((uint32_t)__builtin_bit_cast(uint64_t, v) & (kBestLabels - 1)); }
template <int K> struct Best {
    double v[K];
    __device__ Best()
    {
#pragma unroll
        for (int j = 0; j < K; ++j) v[j] = 0.0;
    }
    // returns what falls off: the smallest of the K + 1
    __device__ double insert(double x)
    {
        const double off = smaller(x, v[K - 1]);
#pragma unroll
        for (int j = K - 1; j > 0; --j) v[j] = larger(smaller(v[j - 1], x), v[j]);      // the middle one of the three
        v[0] = larger(v[0], x);
        return off;
    }
};

// (m, s) stands for s * exp(m): running maximum and sum.  m = -inf: nothing yet; m = NaN: a NaN was among them (an infinite
// score makes s NaN as well, so s alone cannot tell).
struct LogSum {
    float m, s;
};
__device__ inline float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
// both in units of scores; c = log2(e) / temperature
__device__ inline LogSum join(LogSum a, LogSum b, float c)
{
    const float m = max_or_nan(a.m, b.m), r = finite_or_zero(m);
    return {m, a.s * __builtin_amdgcn_exp2f((a.m - r) * c) + b.s * __builtin_amdgcn_exp2f((b.m - r) * c)};
}
__device__ inline void add_score(LogSum &a, float v, float c)
{
    const float m = max_or_nan(a.m, v), r = finite_or_zero(m);
    a.s = a.s * __builtin_amdgcn_exp2f((a.m - r) * c) + __builtin_amdgcn_exp2f((v - r) * c);
    a.m = m;
}
__device__ inline LogSum wave_join(LogSum a, float c)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const LogSum b = {__shfl_xor(a.m, o), __shfl_xor(a.s, o)};
        a = join(a, b, c);
    }
    return a;
}

// (m, s) stands for (1 + s) * exp(m), m the largest term: where one term outweighs all others, 1 + s would keep nothing of
// them in fp32, and -log of that term's share, log1p(s), is just what a confident row's loss consists of.  m = -inf, s = -1:
// nothing yet.
struct Excess {
    float m, s;
};
constexpr Excess kNoExcess = {-INFINITY, -1.f};
__device__ inline Excess join(Excess a, Excess b, float c)
{
    const bool first = a.m >= b.m;
    const float ref = finite_or_zero(first ? a.m : b.m);
    const Excess hi = first ? a : b, lo = first ? b : a;
    return {hi.m, fmaf(1.f + lo.s, __builtin_amdgcn_exp2f((lo.m - ref) * c), hi.s)};
}
__device__ inline Excess wave_join(Excess a, float c)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, Excess{__shfl_xor(a.m, o), __shfl_xor(a.s, o)}, c);
    return a;
}

// -inf where bit i of the mask is set, by its bits: two instructions
__device__ inline float minus_inf_where(uint32_t mask, int i, float x)
{
    const int m = (int)(mask << (31 - i)) >> 31;
    return __builtin_bit_cast(float, (m & (int)0xff800000) | (~m & __builtin_bit_cast(int, x)));
}

// log(1 + s) for s >= -1 to a few steps: log(u) of the rounded u = 1 + s, scaled by the part of s that u keeps (Kahan).  From
// 2^24 on u is s to half a step, and the part is not looked at: the reciprocal of a number above 2^126 is flushed to zero.
__device__ inline float log_1p(float s)
{
    const float u = 1.f + s, kept = u - 1.f;
    if (kept == 0.f) return s;
    return s < 0x1p24f ? logf(u) * (s * __builtin_amdgcn_rcpf(kept)) : logf(u);
}

// log(s * exp(m / temperature)); -inf for nothing, an infinite score stays infinite and a NaN a NaN
__device__ inline float log_of(LogSum a, float inv_t)
{
    if (a.m == INFINITY) return INFINITY;
    return a.s == 0.f ? -INFINITY : fmaf(a.m, inv_t, logf(a.s));
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr double kLog2eD = 1.44269504088896340736;

// (log2(e) / temperature and its inverse have to be ordinary fp32 numbers)
inline bool temperature_ok(double t) { return t >= 1e-30 && t <= 1e30; }

// exp((score - m) / temperature) in 64 bits, for scores up to m: 2^y = 2^n 2^f with n = rint(y), f in [-1/2, 1/2], and the
// Taylor polynomial of 2^f to f^11 (the next term is 2^-47).  The largest score weighs exactly 1.
struct Weight {
    double m, a;                // a = log2(e) / temperature
    __device__ double operator()(float x) const { return scaled(x, 0); }
    // ... times 2^by
    __device__ double scaled(float x, int by) const
    {
        const double y = fmax(((double)x - m) * a, -1100.0);     // (2^-1100 is 0; -inf would leave f undefined)
        const double n = __builtin_rint(y), f = y - n;
        double p = 4.4455382718708117e-10;                       // ln(2)^n / n!
        p = fma(p, f, 7.0549116208011233e-09);
        p = fma(p, f, 1.0178086009239699e-07);
        p = fma(p, f, 1.3215486790144309e-06);
        p = fma(p, f, 1.5252733804059840e-05);
        p = fma(p, f, 1.5403530393381610e-04);
        p = fma(p, f, 1.3333558146428443e-03);
        p = fma(p, f, 9.6181291076284772e-03);
        p = fma(p, f, 5.5504108664821580e-02);
        p = fma(p, f, 2.4022650695910071e-01);
        p = fma(p, f, 6.9314718055994531e-01);
        p = fma(p, f, 1.0);
        return __builtin_ldexp(p, (int)n + by);
    }
};

// Host: a launch's threads are counted in 32 bits
inline bool launchable(unsigned long long blocks, unsigned threads) { return blocks * threads < (1ull << 32); }

// Host: the arguments every call shares.  0 or an error code; fills the view.
inline int make_rows(Rows &r, const void *p, int dtype, int N, int C, int S, long long sn, long long sc, long long ss)
{
    if (!p || N <= 0 || C <= 0 || S <= 0 || sn < 0 || sc < 0 || ss < 0) return MFL_ERR_INVALID_ARGUMENT;
    if (dtype != MFL_F32 && dtype != MFL_BF16 && dtype != MFL_F16) return MFL_ERR_INVALID_ARGUMENT;
    if ((long long)N * S > 0x7fffffffll || C > (1 << 30)) return MFL_ERR_TOO_LARGE;
    r = {p, sn, sc, ss, (unsigned)((long long)N * S), (unsigned)S, C};
    return MFL_OK;
}

}  // namespace mfl_scores

#endif
