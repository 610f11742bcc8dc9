// The k largest scores of every row with their labels, and rest = log sum exp(score / temperature) over all other labels:
// what a teacher leaves behind for a student.  Beside argmax_labels (AdvancedModel.py:420-421), which is k = 1 without
// the rest; the reference has no counterpart.
//
// Order: larger score first, lower label first among equals, NaN above everything.
//
// Two shapes of work.
//   lanes   one lane per row, the k best in the lane's registers, labels streamed once.  Neighbouring pixels of a label
//           map are neighbouring lanes, so every load of a class plane is coalesced.  A new score is sorted in
//           (a compare, a median and two selects per place); what falls off the list's end can no longer be among the k best
//           and goes into the rest's running sum, so one pass gives both and the rest is never a difference of two sums.
//   rows    one workgroup per row, for rows of many labels.
#include "mfl_scores.h"

namespace {

using namespace mfl_scores;

constexpr int kLaneThreads = 256;

template <typename T, int K>
__global__ void __launch_bounds__(kLaneThreads)
top_lanes_kernel(Rows in, float c2, float inv_t, int k, T *__restrict__ values, int *__restrict__ labels, float *__restrict__ rest)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    constexpr int kNone = (int)0x80000000;          // below every score's key
    int v[K], id[K];
#pragma unroll
    for (int j = 0; j < K; ++j) { v[j] = kNone; id[j] = -1; }
    LogSum sum = {-INFINITY, 0.f};
    // From the last place up: a place whose holder is smaller takes the new score or, where that goes further up, the holder
    // above (strictly smaller: an earlier label stays in front of its equals).  Returns what falls off, the smallest of the
    // K + 1.
    auto insert = [&](float x, int c) {
        const int xv = score_key(x);
        const int off = min(xv, v[K - 1]);
        bool up = xv > v[K - 1];
#pragma unroll
        for (int j = K - 1; j > 0; --j) {
            const bool above = xv > v[j - 1];
            id[j] = up ? (above ? id[j - 1] : c) : id[j];
            v[j] = max(min(v[j - 1], xv), v[j]);    // the middle one of the three
            up = above;
        }
        id[0] = up ? c : id[0];
        v[0] = max(v[0], xv);
        return off;
    };
    const int head = in.C < K ? in.C : K;           // nothing real falls off before the list is full
    int c = 0;
    for (; c < head; ++c, p += in.sc) insert(to_float(*p), c);
    constexpr int U = 8;
    for (; c + U <= in.C; c += U, p += U * in.sc) {
        float x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = to_float(p[i * in.sc]);
        float m = sum.m;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x[i] = key_score(insert(x[i], c + i));
            m = fmaxf(m, x[i]);
        }
        const float ref = finite_or_zero(m);
        float t = sum.s * __builtin_amdgcn_exp2f((sum.m - ref) * c2);
#pragma unroll
        for (int i = 0; i < U; ++i) t += __builtin_amdgcn_exp2f((x[i] - ref) * c2);
        sum = {m, t};
    }
    for (; c < in.C; ++c, p += in.sc) add_score(sum, key_score(insert(to_float(*p), c)), c2);
    const size_t base = ((size_t)n * k) * in.S + s;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (j < k) {
            from_float(key_score(v[j]), values[base + (size_t)j * in.S]);
            labels[base + (size_t)j * in.S] = id[j];
        } else if (v[j] != kNone) {
            add_score(sum, key_score(v[j]), c2);
        }
    }
    rest[r] = log_of(sum, inv_t);
}

// One workgroup per row: k times the best label below the one before, then the rest in one pass.
template <typename T>
__global__ void __launch_bounds__(256)
top_rows_kernel(Rows in, float c2, float inv_t, int k, T *__restrict__ values, int *__restrict__ labels, float *__restrict__ rest)
{
    __shared__ uint64_t best[4];
    __shared__ LogSum part[4];
    const unsigned r = blockIdx.x;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const size_t base = ((size_t)n * k) * in.S + s;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    uint64_t last = ~0ull;
    for (int j = 0; j < k; ++j) {
        uint64_t b = 0;
        for (int c = threadIdx.x; c < in.C; c += 256) {
            const uint64_t key = rank_key(score_key(to_float(p[c * in.sc])), c);
            if ((j == 0 || key < last) && key > b) b = key;     // (the key of a NaN on label 0 is ~0)
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)b, o);
            b = other > b ? other : b;
        }
        if (lane == 0) best[wave] = b;
        __syncthreads();
        for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
        __syncthreads();
        last = b;
        if (threadIdx.x == 0) {
            from_float(rank_score(b), values[base + (size_t)j * in.S]);
            labels[base + (size_t)j * in.S] = rank_label(b);
        }
    }
    LogSum sum = {-INFINITY, 0.f};
    for (int c = threadIdx.x; c < in.C; c += 256) {
        const float x = to_float(p[c * in.sc]);
        if (rank_key(score_key(x), c) < last) add_score(sum, x, c2);
    }
    sum = wave_join(sum, c2);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) sum = join(sum, part[w], c2);
        rest[r] = log_of(sum, inv_t);
    }
}

template <typename T>
int run(const Rows &in, double temperature, int k, void *values, int *labels, float *rest, hipStream_t st)
{
    const float c2 = (float)(kLog2eD / temperature), inv_t = (float)(1.0 / temperature);
    if (k > 32 || (in.sc == 1 && in.C >= 512) || in.rows < 64) {
        hipLaunchKernelGGL(top_rows_kernel<T>, dim3(in.rows), dim3(256), 0, st, in, c2, inv_t, k, (T *)values, labels, rest);
        return (int)hipGetLastError();
    }
    const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
#define MFL_TOP(K) hipLaunchKernelGGL((top_lanes_kernel<T, K>), grid, block, 0, st, in, c2, inv_t, k, (T *)values, labels, rest)
    if (k <= 1) MFL_TOP(1);
    else if (k <= 2) MFL_TOP(2);
    else if (k <= 4) MFL_TOP(4);
    else if (k <= 8) MFL_TOP(8);
    else if (k <= 16) MFL_TOP(16);
    else MFL_TOP(32);
#undef MFL_TOP
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t mfl_top_labels_workspace_bytes(int N, int C, int S, int dtype, int k)
{
    (void)N, (void)C, (void)S, (void)dtype, (void)k;
    return 0;
}

int mfl_top_labels(const void *scores, int dtype, int N, int C, int S, long long stride_n, long long stride_c, long long stride_s,
                   double temperature, int k, void *values, int *labels, float *rest, void *workspace, size_t workspace_bytes,
                   mfl_stream_t stream)
{
    Rows in;
    const int rc = make_rows(in, scores, dtype, N, C, S, stride_n, stride_c, stride_s);
    if (rc) return rc;
    if (!values || !labels || !rest || k < 1 || k > MFL_MAX_TOP_LABELS || k > C || !temperature_ok(temperature))
        return MFL_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < mfl_top_labels_workspace_bytes(N, C, S, dtype, k)) return MFL_ERR_WORKSPACE;
    (void)workspace;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run<float>(in, temperature, k, values, labels, rest, st);
    case MFL_BF16: return run<bf16_t>(in, temperature, k, values, labels, rest, st);
    default: return run<f16_t>(in, temperature, k, values, labels, rest, st);
    }
}

}  // extern "C"
