// Distillation loss against a teacher's top labels, and its gradient.  Beside the class-weighted NLL of the reference's
// training step (AdvancedModel.py:295-299), whose target is one label; here it is the teacher's distribution, kept as its
// k largest scores t_j with their labels and, optionally, rest = log of what all other labels hold at this temperature.
//
// With b = score / T, Z = log sum exp(b), O = the labels outside the record, Z_O the same sum over O:
//   p_j = exp(t_j / T - A), p_rest = exp(rest - A), A = log(sum_j exp(t_j / T) + exp(rest))
//   q_i = exp(b_i - Z), q_rest = exp(Z_O - Z)
//   loss = T^2 (sum_j p_j (log p_j - log q_j) + p_rest (log p_rest - log q_rest))
//   d loss / d score_i = T (q_i - sum of the p_j with label i)                        i in the record
//                      = T (q_rest - p_rest) exp(b_i - Z_O)   with rest               otherwise
//                      = T q_i                                without
// Entries whose label is outside [0, C) belong to no class and are passed over; a term with p = 0 is 0; a row that is not
// valid, has no entry left or whose scores are all -inf has loss 0 and gradient 0.
//
// Z_O is summed directly over O, never as a difference: where the record holds nearly all the mass, Z - (record) would
// leave nothing but rounding.  Softmax statistics are fp32 as (m, log s) with m the row's largest score, which is exact:
// differences b_i - Z then lose nothing to the size of the scores.
//   stats[0] = m,  stats[1] = Z - m / T,  stats[2] = Z_O - Z (0 without rest)
#include "mfl_scores.h"

namespace {

using namespace mfl_scores;

struct Teacher {
    const void *values;
    int dtype;
    const int *labels;
    const float *rest;
    const unsigned char *valid;
    int k;
    float c2, inv_t, t;         // log2(e) / T, 1 / T, T
};

constexpr int kLaneThreads = 256;
constexpr int kChunkWords = 8;          // labels marked at a time by a lane: 32 * 8 bits

// The teacher's side of one row, by one lane: running sum over the entries (units of scores) and the rest.
struct Target {
    LogSum sum;
    float log_a;                // A - sum.m / T
    float log_p_rest, p_rest;
    bool any;                   // the teacher's distribution holds something
};
__device__ inline Target target_of(const Teacher &t, int C, size_t base, size_t step, unsigned r)
{
    Target g;
    g.sum = {-INFINITY, 0.f};
    g.any = false;
    for (int j = 0; j < t.k; ++j) {
        const int i = t.labels[base + j * step];
        if ((unsigned)i >= (unsigned)C) continue;
        g.any = true;
        add_score(g.sum, load_any(t.values, t.dtype, base + j * step), t.c2);
    }
    const float rest = t.rest ? t.rest[r] : -INFINITY;
    // the rest joins in units of the scores: exp(rest) = exp((rest * T) / T)
    if (rest != -INFINITY) {
        const float m = fmaxf(g.sum.m, rest * t.t), ref = finite_or_zero(m);
        g.sum.s = g.sum.s * __builtin_amdgcn_exp2f((g.sum.m - ref) * t.c2) + __builtin_amdgcn_exp2f((rest - ref * t.inv_t) * kLog2e);
        g.sum.m = m;
    }
    g.any = g.any && !(g.sum.s == 0.f);
    g.log_a = logf(g.sum.s);
    g.log_p_rest = rest == -INFINITY ? -INFINITY : (rest - g.sum.m * t.inv_t) - g.log_a;
    g.p_rest = __builtin_amdgcn_exp2f(g.log_p_rest * kLog2e);
    return g;
}

// p (log p - log q); nothing where p is 0
__device__ inline float share_term(float p, float log_p, float log_q) { return p == 0.f ? 0.f : p * (log_p - log_q); }

struct Stats {
    float m, z, mo, zo;         // as above
};
constexpr Stats kNoStats = {-INFINITY, 0.f, -INFINITY, 0.f};
__device__ inline Stats stats_of(LogSum all, LogSum out, bool rest)
{
    if (all.m == -INFINITY && all.s == 0.f) return kNoStats;
    const bool some = rest && !(out.m == -INFINITY && out.s == 0.f);
    return {all.m, logf(all.s), some ? out.m : -INFINITY, some ? logf(out.s) : 0.f};
}
__device__ inline float log_q_rest(const Stats &a, float inv_t)
{
    return a.mo == -INFINITY ? -INFINITY : (a.mo - a.m) * inv_t + (a.zo - a.z);
}
__device__ inline void put(float *loss, float *stats, size_t rows, unsigned r, float l, const Stats &a)
{
    loss[r] = l;
    stats[r] = a.m;
    stats[rows + r] = a.z;
    stats[2 * rows + r] = a.mo;
    stats[3 * rows + r] = a.zo;
}
__device__ inline Stats load_stats(const float *stats, size_t rows, unsigned r)
{
    return {stats[r], stats[rows + r], stats[2 * rows + r], stats[3 * rows + r]};
}

// What a label's gradient is made of:  up * (exp(..top) - taken)  in the record,  f_out * exp(..out)  outside
struct Slope {
    float up, f_out, m_top, o_top, m_out, o_out;
};
__device__ inline Slope slope_of(const Stats &a, const Teacher &t, const Target &g, float grad_loss)
{
    Slope s;
    s.up = s.f_out = grad_loss * t.t;
    s.m_top = s.m_out = a.m;
    s.o_top = s.o_out = -a.z * kLog2e;
    if (t.rest) {
        s.f_out = 0.f;
        if (a.mo != -INFINITY) {
            s.f_out = s.up * (__builtin_amdgcn_exp2f(log_q_rest(a, t.inv_t) * kLog2e) - g.p_rest);
            s.m_out = a.mo;
            s.o_out = -a.zo * kLog2e;
        }
    }
    return s;
}
// taken: the record's share of the label, -1 where it is not named
__device__ inline float slope(const Slope &s, float x, float taken, float c2)
{
    const bool named = taken >= 0.f;
    const float e = __builtin_amdgcn_exp2f((x - (named ? s.m_top : s.m_out)) * c2 + (named ? s.o_top : s.o_out));
    return named ? s.up * (e - taken) : s.f_out * e;
}

// One lane per row: see mfl_top_labels.hip for the shapes of work.
template <typename T, bool REST>
__global__ void __launch_bounds__(kLaneThreads)
forward_lanes_kernel(Rows in, Teacher t, float *__restrict__ loss, float *__restrict__ stats)
{
    __shared__ uint32_t marks[kChunkWords][kLaneThreads];
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const size_t base = (size_t)n * t.k * in.S + s;
    if (t.valid && !t.valid[r]) return put(loss, stats, in.rows, r, 0.f, kNoStats);
    const Target g = target_of(t, in.C, base, in.S, r);
    if (!g.any) return put(loss, stats, in.rows, r, 0.f, kNoStats);
    LogSum out = {-INFINITY, 0.f}, top = {-INFINITY, 0.f};
    for (int c0 = 0; c0 < in.C; c0 += 32 * kChunkWords) {
        const int c1 = min(in.C, c0 + 32 * kChunkWords);
        if (REST) {
            for (int w = 0; w < kChunkWords; ++w) marks[w][threadIdx.x] = 0;
            for (int j = 0; j < t.k; ++j) {
                const int i = t.labels[base + (size_t)j * in.S];
                if (i < c0 || i >= c1) continue;
                const uint32_t bit = 1u << ((i - c0) & 31), old = marks[(i - c0) >> 5][threadIdx.x];
                if (!(old & bit)) {     // a label named twice counts once on the student's side
                    marks[(i - c0) >> 5][threadIdx.x] = old | bit;
                    add_score(top, to_float(p[i * in.sc]), t.c2);
                }
            }
        }
        for (int c = c0; c < c1; c += 32) {
            const uint32_t word = REST ? marks[(c - c0) >> 5][threadIdx.x] : 0;
            const int end = min(32, c1 - c);
            constexpr int U = 8;
            const T *q = p + c * in.sc;
            int i = 0;
            for (; i + U <= end; i += U) {
                float x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = to_float(q[(i + u) * in.sc]);
                float m = out.m;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (REST && (word >> (i + u) & 1)) x[u] = -INFINITY;
                    m = fmaxf(m, x[u]);
                }
                const float ref = finite_or_zero(m);
                float sum = out.s * __builtin_amdgcn_exp2f((out.m - ref) * t.c2);
#pragma unroll
                for (int u = 0; u < U; ++u) sum += __builtin_amdgcn_exp2f((x[u] - ref) * t.c2);
                out = {m, sum};
            }
            for (; i < end; ++i)
                if (!(REST && (word >> i & 1))) add_score(out, to_float(q[i * in.sc]), t.c2);
        }
    }
    const LogSum all = REST ? join(out, top, t.c2) : out;
    const Stats a = stats_of(all, out, REST);
    if (a.m == -INFINITY) return put(loss, stats, in.rows, r, 0.f, a);
    float sum = REST ? share_term(g.p_rest, g.log_p_rest, log_q_rest(a, t.inv_t)) : 0.f;
    for (int j = 0; j < t.k; ++j) {
        const int i = t.labels[base + (size_t)j * in.S];
        if ((unsigned)i >= (unsigned)in.C) continue;
        const float lp = (load_any(t.values, t.dtype, base + (size_t)j * in.S) - g.sum.m) * t.inv_t - g.log_a;
        const float lq = (to_float(p[i * in.sc]) - a.m) * t.inv_t - a.z;
        sum += share_term(__builtin_amdgcn_exp2f(lp * kLog2e), lp, lq);
    }
    put(loss, stats, in.rows, r, t.t * t.t * sum, a);
}

// Gradient of the scores.  What the record takes from a label lies in LDS, one column of 32 labels per lane (-1: not named).
template <typename T>
__global__ void __launch_bounds__(kLaneThreads)
backward_lanes_kernel(Rows in, Teacher t, const float *__restrict__ stats, const float *__restrict__ grad_loss, T *__restrict__ grad,
                      long long gn, long long gc, long long gs)
{
    __shared__ float taken[32][kLaneThreads];
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    T *out = grad + (long long)n * gn + (long long)s * gs;
    const size_t base = (size_t)n * t.k * in.S + s;
    const Stats a = load_stats(stats, in.rows, r);
    Target g;
    g.any = false;
    if (!(t.valid && !t.valid[r]) && a.m != -INFINITY) g = target_of(t, in.C, base, in.S, r);
    if (!g.any) {
        for (int c = 0; c < in.C; ++c) from_float(0.f, out[c * gc]);
        return;
    }
    const Slope sl = slope_of(a, t, g, grad_loss[r]);
    for (int i = 0; i < 32; ++i) taken[i][threadIdx.x] = -1.f;
    for (int c0 = 0; c0 < in.C; c0 += 32) {
        const int end = min(32, in.C - c0);
        for (int j = 0; j < t.k; ++j) {
            const int i = t.labels[base + (size_t)j * in.S] - c0;
            if (i < 0 || i >= end) continue;
            const float lp = (load_any(t.values, t.dtype, base + (size_t)j * in.S) - g.sum.m) * t.inv_t - g.log_a;
            taken[i][threadIdx.x] = fmaxf(taken[i][threadIdx.x], 0.f) + __builtin_amdgcn_exp2f(lp * kLog2e);
        }
        const T *q = p + c0 * in.sc;
        T *w = out + c0 * gc;
        for (int i = 0; i < end; ++i) {
            const float share = taken[i][threadIdx.x];
            from_float(slope(sl, to_float(q[i * in.sc]), share, t.c2), w[i * gc]);
            if (share >= 0.f) taken[i][threadIdx.x] = -1.f;
        }
    }
}

constexpr int kRowThreads = 256;
constexpr int kSegment = 1 << 16;       // labels marked at a time by a workgroup: 8 KB of bits

__device__ inline LogSum block_join(LogSum a, LogSum (*part)[2], int which, float c)
{
    a = wave_join(a, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][which] = a;
    __syncthreads();
    a = part[0][which];
    for (int w = 1; w < kRowThreads / 64; ++w) a = join(a, part[w][which], c);
    return a;
}

template <typename T, bool REST>
__global__ void __launch_bounds__(kRowThreads)
forward_rows_kernel(Rows in, Teacher t, float *__restrict__ loss, float *__restrict__ stats)
{
    extern __shared__ uint32_t bits[];
    __shared__ LogSum part[kRowThreads / 64][2];
    const unsigned r = blockIdx.x;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const size_t base = (size_t)n * t.k * in.S + s;
    float l = 0.f;
    Stats a = kNoStats;
    bool live = !(t.valid && !t.valid[r]);
    Target g;
    if (live) {
        g = target_of(t, in.C, base, in.S, r);      // (every lane the same; k entries)
        live = g.any;
    }
    if (live) {
        LogSum out = {-INFINITY, 0.f}, top = {-INFINITY, 0.f};
        for (int c0 = 0; c0 < in.C; c0 += kSegment) {
            const int c1 = min(in.C, c0 + kSegment);
            if (REST) {
                __syncthreads();
                for (int w = threadIdx.x; w < (c1 - c0 + 31) / 32; w += kRowThreads) bits[w] = 0;
                __syncthreads();
                for (int j = threadIdx.x; j < t.k; j += kRowThreads) {
                    const int i = t.labels[base + (size_t)j * in.S];
                    if (i < c0 || i >= c1) continue;
                    const uint32_t bit = 1u << ((i - c0) & 31);
                    // (a label named twice counts once on the student's side)
                    if (!(atomicOr(&bits[(i - c0) >> 5], bit) & bit)) add_score(top, to_float(p[i * in.sc]), t.c2);
                }
                __syncthreads();
            }
            for (int c = c0 + threadIdx.x; c < c1; c += kRowThreads)
                if (!(REST && (bits[(c - c0) >> 5] >> ((c - c0) & 31) & 1))) add_score(out, to_float(p[c * in.sc]), t.c2);
        }
        out = block_join(out, part, 0, t.c2);
        LogSum all = out;
        if (REST) {
            top = block_join(top, part, 1, t.c2);
            all = join(out, top, t.c2);
        }
        a = stats_of(all, out, REST);
        if (a.m != -INFINITY && threadIdx.x == 0) {
            float sum = REST ? share_term(g.p_rest, g.log_p_rest, log_q_rest(a, t.inv_t)) : 0.f;
            for (int j = 0; j < t.k; ++j) {
                const int i = t.labels[base + (size_t)j * in.S];
                if ((unsigned)i >= (unsigned)in.C) continue;
                const float lp = (load_any(t.values, t.dtype, base + (size_t)j * in.S) - g.sum.m) * t.inv_t - g.log_a;
                const float lq = (to_float(p[i * in.sc]) - a.m) * t.inv_t - a.z;
                sum += share_term(__builtin_amdgcn_exp2f(lp * kLog2e), lp, lq);
            }
            l = t.t * t.t * sum;
        }
    }
    if (threadIdx.x == 0) put(loss, stats, in.rows, r, l, a);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
backward_rows_kernel(Rows in, Teacher t, const float *__restrict__ stats, const float *__restrict__ grad_loss, T *__restrict__ grad,
                     long long gn, long long gc, long long gs)
{
    __shared__ int label[MFL_MAX_TOP_LABELS];
    __shared__ float share[MFL_MAX_TOP_LABELS];
    const unsigned r = blockIdx.x;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    T *out = grad + (long long)n * gn + (long long)s * gs;
    const size_t base = (size_t)n * t.k * in.S + s;
    const Stats a = load_stats(stats, in.rows, r);
    Target g;
    g.any = false;
    if (!(t.valid && !t.valid[r]) && a.m != -INFINITY) g = target_of(t, in.C, base, in.S, r);
    if (!g.any) {
        for (int c = threadIdx.x; c < in.C; c += kRowThreads) from_float(0.f, out[c * gc]);
        return;
    }
    for (int j = threadIdx.x; j < t.k; j += kRowThreads) {
        label[j] = t.labels[base + (size_t)j * in.S];
        share[j] = __builtin_amdgcn_exp2f(((load_any(t.values, t.dtype, base + (size_t)j * in.S) - g.sum.m) * t.inv_t - g.log_a) * kLog2e);
    }
    __syncthreads();
    const Slope sl = slope_of(a, t, g, grad_loss[r]);
    for (int c = threadIdx.x; c < in.C; c += kRowThreads) {
        float taken = -1.f;
        for (int j = 0; j < t.k; ++j)
            if (label[j] == c) taken = fmaxf(taken, 0.f) + share[j];
        from_float(slope(sl, to_float(p[c * in.sc]), taken, t.c2), out[c * gc]);
    }
}

bool by_rows(const Rows &in) { return in.sc == 1 && in.C >= 512; }

template <typename T>
int run_forward(const Rows &in, const Teacher &t, float *loss, float *stats, hipStream_t st)
{
    if (by_rows(in)) {
        const size_t lds = t.rest ? (size_t)((in.C < kSegment ? in.C : kSegment) + 31) / 32 * 4 : 0;
        if (t.rest) hipLaunchKernelGGL((forward_rows_kernel<T, true>), dim3(in.rows), dim3(kRowThreads), lds, st, in, t, loss, stats);
        else hipLaunchKernelGGL((forward_rows_kernel<T, false>), dim3(in.rows), dim3(kRowThreads), lds, st, in, t, loss, stats);
    } else {
        const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
        if (t.rest) hipLaunchKernelGGL((forward_lanes_kernel<T, true>), grid, block, 0, st, in, t, loss, stats);
        else hipLaunchKernelGGL((forward_lanes_kernel<T, false>), grid, block, 0, st, in, t, loss, stats);
    }
    return (int)hipGetLastError();
}

template <typename T>
int run_backward(const Rows &in, const Teacher &t, const float *stats, const float *grad_loss, void *grad, long long gn, long long gc,
                 long long gs, hipStream_t st)
{
    if (by_rows(in)) {
        hipLaunchKernelGGL(backward_rows_kernel<T>, dim3(in.rows), dim3(kRowThreads), 0, st, in, t, stats, grad_loss, (T *)grad, gn, gc, gs);
    } else {
        const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
        hipLaunchKernelGGL(backward_lanes_kernel<T>, grid, block, 0, st, in, t, stats, grad_loss, (T *)grad, gn, gc, gs);
    }
    return (int)hipGetLastError();
}

int make_teacher(Teacher &t, const void *values, int dtype, const int *labels, const float *rest, const unsigned char *valid, int k,
                 double temperature)
{
    if (!values || !labels || k < 1 || k > MFL_MAX_TOP_LABELS || !temperature_ok(temperature)) return MFL_ERR_INVALID_ARGUMENT;
    if (dtype != MFL_F32 && dtype != MFL_BF16 && dtype != MFL_F16) return MFL_ERR_INVALID_ARGUMENT;
    t = {values, dtype, labels, rest, valid, k, (float)(kLog2eD / temperature), (float)(1.0 / temperature), (float)temperature};
    return MFL_OK;
}

}  // namespace

extern "C" {

size_t mfl_distillation_workspace_bytes(int N, int C, int S, int dtype, int k)
{
    (void)N, (void)C, (void)S, (void)dtype, (void)k;
    return 0;
}

int mfl_distillation_forward(const void *scores, int dtype, int N, int C, int S, long long stride_n, long long stride_c,
                             long long stride_s, const void *values, int values_dtype, const int *labels, const float *rest,
                             const unsigned char *valid, int k, double temperature, float *loss, float *stats, void *workspace,
                             size_t workspace_bytes, mfl_stream_t stream)
{
    Rows in;
    Teacher t;
    int rc = make_rows(in, scores, dtype, N, C, S, stride_n, stride_c, stride_s);
    if (!rc) rc = make_teacher(t, values, values_dtype, labels, rest, valid, k, temperature);
    if (rc) return rc;
    if (!loss || !stats) return MFL_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < mfl_distillation_workspace_bytes(N, C, S, dtype, k)) return MFL_ERR_WORKSPACE;
    (void)workspace;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run_forward<float>(in, t, loss, stats, st);
    case MFL_BF16: return run_forward<bf16_t>(in, t, loss, stats, st);
    default: return run_forward<f16_t>(in, t, loss, stats, st);
    }
}

int mfl_distillation_backward(const void *scores, int dtype, int N, int C, int S, long long stride_n, long long stride_c,
                              long long stride_s, const void *values, int values_dtype, const int *labels, const float *rest,
                              const unsigned char *valid, int k, double temperature, const float *stats, const float *grad_loss,
                              void *d_scores, long long d_stride_n, long long d_stride_c, long long d_stride_s, mfl_stream_t stream)
{
    Rows in, out;
    Teacher t;
    int rc = make_rows(in, scores, dtype, N, C, S, stride_n, stride_c, stride_s);
    if (!rc) rc = make_rows(out, d_scores, dtype, N, C, S, d_stride_n, d_stride_c, d_stride_s);
    if (!rc) rc = make_teacher(t, values, values_dtype, labels, rest, valid, k, temperature);
    if (rc) return rc;
    if (!stats || !grad_loss) return MFL_ERR_INVALID_ARGUMENT;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run_backward<float>(in, t, stats, grad_loss, d_scores, out.sn, out.sc, out.ss, st);
    case MFL_BF16: return run_backward<bf16_t>(in, t, stats, grad_loss, d_scores, out.sn, out.sc, out.ss, st);
    default: return run_backward<f16_t>(in, t, stats, grad_loss, d_scores, out.sn, out.sc, out.ss, st);
    }
}

}  // extern "C"
