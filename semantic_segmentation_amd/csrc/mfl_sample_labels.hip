// One label per row drawn from given random numbers: next to argmax_labels (AdvancedModel.py:420-421), which answers with
// the largest marginal, an answer that follows the marginals.  The reference has no counterpart.
//
// With w_c = exp((score_c - largest) / T) and the row's labels ordered by score (the lower label first among equals):
//   keep the first top_k;  S = their sum;  of those the ones in front of which less than top_p * S has been summed;
//   of those the ones with w_c >= min_p.  (The first label always stays.)
//   label = the first kept one, in label order, whose running sum exceeds u * (sum of the kept), and
//   logprob = log(w_label / sum of the kept).
// The order of label numbers, not of scores, is what the running sum follows: without filters nothing has to be sorted.
//
// All weights and sums are 64-bit floats: a label's border in a row of 10^5 labels is 10^-5 of the mass wide, so fp32
// sums (10^-7) would misplace about one draw in a hundred, and a batch of maps has millions of draws.
//
// Settings may differ from n to n (arrays of N).  T <= 0 takes the largest; top_k <= 0, top_p >= 1 and min_p <= 0 keep all.
// A row without a finite largest score (all -inf, or a NaN or +inf among them) has no distribution: label -1, logprob -inf.
#include "mfl_scores.h"

namespace {

using namespace mfl_scores;

struct Settings {
    double t, top_p, min_p;
    int top_k;
    const float *t_n, *top_p_n, *min_p_n;
    const int *top_k_n;
};
struct Filter {
    double inv_t, top_p, min_p;
    int top_k;                  // INT_MAX: no limit
    bool ranked;                // the order of the labels matters
};
__device__ inline Filter filter_of(const Settings &f, unsigned n, int C)
{
    Filter r;
    const double t = f.t_n ? (double)f.t_n[n] : f.t;
    r.top_p = f.top_p_n ? (double)f.top_p_n[n] : f.top_p;
    r.min_p = f.min_p_n ? (double)f.min_p_n[n] : f.min_p;
    r.top_k = f.top_k_n ? f.top_k_n[n] : f.top_k;
    if (r.top_k <= 0 || r.top_k >= C) r.top_k = 0x7fffffff;
    if (!(t > 0)) r.top_k = 1;
    r.inv_t = t > 0 ? fmax(1.0 / t, 1e-30) : 1.0;       // (never 0: -inf * 0)
    if (!(r.top_p < 1)) r.top_p = 1;
    r.ranked = r.top_k < C || r.top_p < 1;
    return r;
}

struct Out {
    void *labels;
    int bytes;                  // of a label: 1, 4 or 8
    float *logprob;
};
__device__ inline void put(const Out &o, unsigned r, int label, double logprob)
{
    if (o.bytes == 8) ((long long *)o.labels)[r] = label;
    else if (o.bytes == 4) ((int *)o.labels)[r] = label;
    else ((unsigned char *)o.labels)[r] = (unsigned char)label;       // none: 255, the void label
    if (o.logprob) o.logprob[r] = (float)logprob;
}

// The draw u in [0, 1): anything below counts as 0
__device__ inline double draw_of(float u) { return u > 0 ? (double)u : 0.0; }

// One lane per row.
constexpr int kLaneThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kLaneThreads)
sample_lanes_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const Filter f = filter_of(set, n, in.C);
    int mk = (int)0x80000000;
    for (int c = 0; c < in.C; ++c) mk = max(mk, score_key(to_float(p[c * in.sc])));
    const float m = key_score(mk);
    if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    auto weight = [&](float x) { return exp(((double)x - (double)m) * f.inv_t); };
    uint64_t cut = 0;                               // kept by rank: rank_key >= cut
    if (f.ranked) {
        // binary search over the rank keys, from the top bit down
        auto search = [&](auto reached) {
            uint64_t k = 0;
            for (int b = 63; b >= 0; --b)
                if (reached(k | 1ull << b)) k |= 1ull << b;
            return k;
        };
        double total = 0;
        if (f.top_k < in.C)
            cut = search([&](uint64_t k) {
                int count = 0;
                for (int c = 0; c < in.C; ++c) count += rank_key(score_key(to_float(p[c * in.sc])), c) >= k;
                return count >= f.top_k;
            });
        if (f.top_p < 1) {
            for (int c = 0; c < in.C; ++c) {
                const float x = to_float(p[c * in.sc]);
                if (rank_key(score_key(x), c) >= cut) total += weight(x);
            }
            const uint64_t top = rank_key(mk, 0);
            const uint64_t nucleus = search([&](uint64_t k) {
                if (k > top) return false;
                double sum = 0;
                for (int c = 0; c < in.C; ++c) {
                    const float x = to_float(p[c * in.sc]);
                    const uint64_t key = rank_key(score_key(x), c);
                    if (key >= cut && key >= k) sum += weight(x);
                }
                return sum > 0 && sum >= f.top_p * total;
            });
            cut = nucleus > cut ? nucleus : cut;
        }
    }
    auto kept_weight = [&](float x, int c) {
        const double w = weight(x);
        const bool keep = (w >= f.min_p || score_key(x) == mk) && rank_key(score_key(x), c) >= cut;
        return keep ? w : 0.0;
    };
    double total = 0;
    for (int c = 0; c < in.C; ++c) total += kept_weight(to_float(p[c * in.sc]), c);
    const double target = draw_of(uniform[r]) * total;
    double run = 0, got = 0;
    int label = -1;
    for (int c = 0; c < in.C; ++c) {
        const double w = kept_weight(to_float(p[c * in.sc]), c);
        if (w == 0) continue;
        run += w;
        label = c;
        got = w;
        if (run > target) break;
    }
    put(out, r, label, log(got / total));
}

// One workgroup per row.
constexpr int kRowThreads = 256;
template <typename V> __device__ inline V block_sum(V v, V *part)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < kRowThreads / 64; ++w) v += part[w];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
sample_rows_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    __shared__ double part[kRowThreads / 64], sums[kRowThreads];
    __shared__ int ipart[kRowThreads / 64];
    const unsigned r = blockIdx.x;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const Filter f = filter_of(set, n, in.C);
    int mk = (int)0x80000000;
    for (int c = threadIdx.x; c < in.C; c += kRowThreads) mk = max(mk, score_key(to_float(p[c * in.sc])));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mk = max(mk, __shfl_xor(mk, o));
    if ((threadIdx.x & 63) == 0) ipart[threadIdx.x >> 6] = mk;
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; ++w) mk = max(mk, ipart[w]);
    const float m = key_score(mk);
    if (!(fabsf(m) < INFINITY)) {
        if (threadIdx.x == 0) put(out, r, -1, -INFINITY);
        return;
    }
    auto weight = [&](float x) { return exp(((double)x - (double)m) * f.inv_t); };
    uint64_t cut = 0;
    if (f.ranked) {
        auto search = [&](auto reached) {
            uint64_t k = 0;
            for (int b = 63; b >= 0; --b)
                if (reached(k | 1ull << b)) k |= 1ull << b;
            return k;
        };
        if (f.top_k < in.C)
            cut = search([&](uint64_t k) {
                int count = 0;
                for (int c = threadIdx.x; c < in.C; c += kRowThreads) count += rank_key(score_key(to_float(p[c * in.sc])), c) >= k;
                return block_sum(count, ipart) >= f.top_k;
            });
        if (f.top_p < 1) {
            auto mass = [&](uint64_t k) {
                double sum = 0;
                for (int c = threadIdx.x; c < in.C; c += kRowThreads) {
                    const float x = to_float(p[c * in.sc]);
                    const uint64_t key = rank_key(score_key(x), c);
                    if (key >= cut && key >= k) sum += weight(x);
                }
                return block_sum(sum, part);
            };
            const double goal = f.top_p * mass(0);
            const uint64_t nucleus = search([&](uint64_t k) {
                const double sum = mass(k);
                return sum > 0 && sum >= goal;
            });
            cut = nucleus > cut ? nucleus : cut;
        }
    }
    auto kept_weight = [&](float x, int c) {
        const double w = weight(x);
        const bool keep = (w >= f.min_p || score_key(x) == mk) && rank_key(score_key(x), c) >= cut;
        return keep ? w : 0.0;
    };
    // every thread a run of neighbouring labels
    const int chunk = (in.C + kRowThreads - 1) / kRowThreads;
    const int c0 = threadIdx.x * chunk, c1 = min(in.C, c0 + chunk);
    double mine = 0;
    for (int c = c0; c < c1; ++c) mine += kept_weight(to_float(p[c * in.sc]), c);
    sums[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0;
        int last = 0;
        for (int i = 0; i < kRowThreads; ++i) {
            total += sums[i];
            if (sums[i] > 0) last = i;
        }
        const double target = draw_of(uniform[r]) * total;
        double run = 0, got = 0;
        int label = -1;
        for (int i = 0; i < kRowThreads; ++i) {
            const double next = run + sums[i];
            if (next > target || i == last) {
                // (rounding may leave the target just past a run's last label: the search then goes on in the next run)
                for (int c = i * chunk; c < in.C; ++c) {
                    const double w = kept_weight(to_float(p[c * in.sc]), c);
                    if (w == 0) continue;
                    run += w;
                    label = c;
                    got = w;
                    if (run > target) break;
                }
                break;
            }
            run = next;
        }
        put(out, r, label, log(got / total));
    }
}

template <typename T>
int run(const Rows &in, const Settings &set, const float *uniform, const Out &out, hipStream_t st)
{
    if (in.sc == 1 && in.C >= 512)
        hipLaunchKernelGGL(sample_rows_kernel<T>, dim3(in.rows), dim3(kRowThreads), 0, st, in, set, uniform, out);
    else
        hipLaunchKernelGGL(sample_lanes_kernel<T>, dim3((in.rows + kLaneThreads - 1) / kLaneThreads), dim3(kLaneThreads), 0, st, in, set,
                           uniform, out);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t mfl_sample_labels_workspace_bytes(int N, int C, int S, int dtype)
{
    (void)N, (void)C, (void)S, (void)dtype;
    return 0;
}

int mfl_sample_labels(const void *scores, int dtype, int N, int C, int S, long long stride_n, long long stride_c, long long stride_s,
                      const float *uniform, double temperature, const float *temperature_n, int top_k, const int *top_k_n, double top_p,
                      const float *top_p_n, double min_p, const float *min_p_n, void *labels, int label_bytes, float *logprob,
                      void *workspace, size_t workspace_bytes, mfl_stream_t stream)
{
    Rows in;
    const int rc = make_rows(in, scores, dtype, N, C, S, stride_n, stride_c, stride_s);
    if (rc) return rc;
    if (!uniform || !labels || (label_bytes != 1 && label_bytes != 4 && label_bytes != 8) || (label_bytes == 1 && C > 255))
        return MFL_ERR_INVALID_ARGUMENT;
    // (a setting that comes as an array is not looked at here)
    if ((!temperature_n && temperature != 0 && !temperature_ok(temperature)) || (!top_k_n && top_k < 0) ||
        (!top_p_n && !(top_p > 0 && top_p <= 1)) || (!min_p_n && !(min_p >= 0 && min_p <= 1)))
        return MFL_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < mfl_sample_labels_workspace_bytes(N, C, S, dtype)) return MFL_ERR_WORKSPACE;
    (void)workspace;
    const Settings set = {temperature, top_p, min_p, top_k, temperature_n, top_p_n, min_p_n, top_k_n};
    const Out out = {labels, label_bytes, logprob};
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run<float>(in, set, uniform, out, st);
    case MFL_BF16: return run<bf16_t>(in, set, uniform, out, st);
    default: return run<f16_t>(in, set, uniform, out, st);
    }
}

}  // extern "C"
