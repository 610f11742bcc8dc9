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
__device__ inline void from_float(float v, bf16_t &o)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    o.u = (u & 0x7fffffffu) > 0x7f800000u ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

// a value of a tensor whose type is known at run time only (uniform branch; the teacher's k values of a row)
__device__ inline float load_any(const void *p, int dtype, size_t i)
{
    if (dtype == MFL_F32) return ((const float *)p)[i];
    if (dtype == MFL_BF16) return to_float(((const bf16_t *)p)[i]);
    return to_float(((const f16_t *)p)[i]);
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

// (m, s) stands for s * exp(m): running maximum and sum.  m = -inf: nothing yet.
struct LogSum {
    float m, s;
};
__device__ inline float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
// both in units of scores; c = log2(e) / temperature
__device__ inline LogSum join(LogSum a, LogSum b, float c)
{
    const float m = fmaxf(a.m, b.m), r = finite_or_zero(m);
    return {m, a.s * __builtin_amdgcn_exp2f((a.m - r) * c) + b.s * __builtin_amdgcn_exp2f((b.m - r) * c)};
}
__device__ inline void add_score(LogSum &a, float v, float c)
{
    const float m = fmaxf(a.m, v), r = finite_or_zero(m);
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

// log(s * exp(m / temperature)); -inf for nothing, and an infinite score stays infinite
__device__ inline float log_of(LogSum a, float inv_t)
{
    if (a.m == INFINITY) return INFINITY;
    return a.s == 0.f ? -INFINITY : fmaf(a.m, inv_t, logf(a.s));
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2eD = 1.44269504088896340736;

// (log2(e) / temperature and its inverse have to be ordinary fp32 numbers)
inline bool temperature_ok(double t) { return t >= 1e-30 && t <= 1e30; }

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
