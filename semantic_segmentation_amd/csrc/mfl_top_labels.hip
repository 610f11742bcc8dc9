// The k largest scores of every row with their labels, and rest = log sum exp(score / temperature) over all other labels:
// what a teacher leaves behind for a student.  Beside argmax_labels (AdvancedModel.py:420-421), which is k = 1 without
// the rest; the reference has no counterpart.
//
// Order: larger score first, lower label first among equals, NaN above everything.
//
// Two shapes of work, here and in the other operators on rows.
//   lanes   one lane per row, the k best in the lane's registers, labels streamed once.  Neighbouring pixels of a label
//           map are neighbouring lanes, so every load of a class plane is coalesced (where few labels lie side by side, in
//           channels-last maps and matrices, lanes are C scores apart and a line is read in C loads).  A new score is sorted
//           in; what falls off the list's end can no longer be among the k best and goes into the rest's running sum, so one
//           pass gives both and the rest is never a difference of two sums.
//   rows    one or more waves per row, for rows of many labels (mfl_wave_top.h).
//
// Measured on MI355X.  Lanes, 8 x 21 x 512 x 512 fp32, k = 4: 51 us, 4.9 TB/s, the rate of a large copy (channels-last 114 us;
// bf16 44 and 59); 4 x 150 x 512 x 512, k = 8: 161 us, 4.3 TB/s (the list as separate words for score and label: 198 us, bound
// by the vector unit).  Rows, 1024 x 32001 bf16, k = 64: 36 us, 1.8 TB/s, bound by the vector unit (about 20 instructions a
// score, 9 of them the rest's exponential and sum); where a mask leaves ten labels of each row 81 us, since every -inf then
// reaches the list's bound.  Maps with k > 32, a wave a pixel: 2 x 150 x 512 x 512, k = 40, 1017 us.
#include "mfl_wave_top.h"

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
    Best<K> best;
    LogSum sum = {-INFINITY, 0.f};
    const int head = in.C < K ? in.C : K;           // nothing real falls off before the list is full
    int c = 0;
    for (; c < head; ++c, p += in.sc) best.insert(place_of(to_float(*p), c));
    constexpr int U = 8;
    for (; c + U <= in.C; c += U) {
        T raw[U];
#pragma unroll
        for (int i = 0; i < U; ++i, p += in.sc) raw[i] = *p;
        float x[U], m = sum.m;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x[i] = place_score(best.insert(place_of(to_float(raw[i]), c + i)));
            m = max_or_nan(m, x[i]);
        }
        const float ref = finite_or_zero(m);
        float t = sum.s * __builtin_amdgcn_exp2f((sum.m - ref) * c2);
#pragma unroll
        for (int i = 0; i < U; ++i) t += __builtin_amdgcn_exp2f((x[i] - ref) * c2);
        sum = {m, t};
    }
    for (; c < in.C; ++c, p += in.sc) add_score(sum, place_score(best.insert(place_of(to_float(*p), c))), c2);
    const size_t base = ((size_t)n * k) * in.S + s;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (j < k) {
            from_float(place_score(best.v[j]), values[base + (size_t)j * in.S]);
            labels[base + (size_t)j * in.S] = place_label(best.v[j]);
        } else if (best.v[j] != 0.0) {
            add_score(sum, place_score(best.v[j]), c2);
        }
    }
    rest[r] = log_of(sum, inv_t);
}

template <typename T>
__device__ inline void put_row(WaveTop<true> &top, const Rows &in, unsigned r, int k, float inv_t, T *values, int *labels, float *rest)
{
    const unsigned n = r / in.S, s = r - n * in.S;
    const size_t base = (size_t)n * k * in.S + s;
    top.ranked([&](int rank, uint64_t key) {
        from_float(rank_score(key), values[base + (size_t)rank * in.S]);
        labels[base + (size_t)rank * in.S] = rank_label(key);
    });
    const LogSum sum = wave_join(top.rest, top.c2);
    if ((threadIdx.x & 63) == 0) rest[r] = log_of(sum, inv_t);
}

// One wave per row
template <typename T>
__global__ void __launch_bounds__(kWaveTopThreads)
top_waves_kernel(Rows in, float c2, float inv_t, int k, T *__restrict__ values, int *__restrict__ labels, float *__restrict__ rest)
{
    __shared__ uint64_t lists[kWaveTopThreads / 64][kListKeys];
    const int wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x * (kWaveTopThreads / 64) + wave;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    WaveTop<true> top(lists[wave], k, c2);
    if (in.sc == 1 && in.C >= 8 * 64 * kVec<T>) {
        float m[4];
        top.look(p, 0, 4, m);
        top.foresee(m);
    }
    top.stream(p, in.sc, 0, in.C);
    top.cut();
    put_row(top, in, r, k, inv_t, values, labels, rest);
}

// One workgroup per part of a row.  With one part the row is finished here, else the part's best go to the workspace.
template <typename T>
__global__ void __launch_bounds__(kWaveTopThreads)
top_parts_kernel(Rows in, float c2, float inv_t, int k, int parts, uint64_t *__restrict__ keys, LogSum *__restrict__ sums,
                 T *__restrict__ values, int *__restrict__ labels, float *__restrict__ rest)
{
    __shared__ TopShared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    WaveTop<true> top(sh.lists[wave], k, c2);
    const int size = top_part_labels(in.C, parts);
    const int begin = min(in.C, (int)part * size), end = min(in.C, begin + size);
    if (!top_of_part(top, sh, p, in.sc, begin, end)) return;
    if (parts == 1) {
        top.cut();
        put_row(top, in, r, k, inv_t, values, labels, rest);
        return;
    }
    const int slots = part_keys(k);
    for (int j = lane; j < slots; j += 64) keys[(size_t)blockIdx.x * slots + j] = j < top.count ? top.list[j] : 0;
    const LogSum sum = wave_join(top.rest, c2);
    if (lane == 0) sums[blockIdx.x] = sum;
}

// One workgroup per row: the best of its parts' best
template <typename T>
__global__ void __launch_bounds__(kWaveTopThreads)
top_join_kernel(Rows in, float c2, float inv_t, int k, int parts, const uint64_t *__restrict__ keys, const LogSum *__restrict__ sums,
                T *__restrict__ values, int *__restrict__ labels, float *__restrict__ rest)
{
    __shared__ TopShared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x;
    const int n = parts * part_keys(k);
    WaveTop<true> top(sh.lists[wave], k, c2);
    if (!top_of_keys(top, sh, keys + (size_t)r * n, n)) return;
    top.cut();
    if (lane < parts) top.rest = join(top.rest, sums[(size_t)r * parts + lane], c2);
    put_row(top, in, r, k, inv_t, values, labels, rest);
}

// Rows of many neighbouring labels, long lists, and few rows go to waves.  Lanes / waves, fp32, k = 4, us: 4096 x 64 14 / 13,
// 16384 x 64 13 / 23, 4096 x 256 32 / 14, 16384 x 256 32 / 37, 16384 x 512 60 / 38, 131072 x 1024 356 / 335.  (Many rows of
// 256 to 1000 labels would do better with lanes: 131072 x 256 80 / 236.)
bool by_waves(const Rows &in, int k)
{
    return k > 32 || in.C > kBestLabels || (in.sc == 1 && (in.C >= 256 || (in.C >= 64 && in.rows <= 4096))) || (in.C >= 1024 && in.rows <= 4096);
}

template <typename T>
int run(const Rows &in, double temperature, int k, void *values, int *labels, float *rest, void *workspace, hipStream_t st)
{
    const float c2 = (float)(kLog2eD / temperature), inv_t = (float)(1.0 / temperature);
    if (by_waves(in, k)) {
        if (!launchable((unsigned long long)in.rows * (row_per_wave(in.rows, in.C) ? 1 : top_parts(in.rows, in.C)), kWaveTopThreads))
            return MFL_ERR_TOO_LARGE;
        if (row_per_wave(in.rows, in.C)) {
            const unsigned per = kWaveTopThreads / 64;
            hipLaunchKernelGGL(top_waves_kernel<T>, dim3((in.rows + per - 1) / per), dim3(kWaveTopThreads), 0, st, in, c2, inv_t, k,
                               (T *)values, labels, rest);
            return (int)hipGetLastError();
        }
        const int parts = top_parts(in.rows, in.C);
        uint64_t *keys = (uint64_t *)workspace;
        LogSum *sums = (LogSum *)(keys + (size_t)in.rows * parts * part_keys(k));
        hipLaunchKernelGGL(top_parts_kernel<T>, dim3(in.rows * parts), dim3(kWaveTopThreads), 0, st, in, c2, inv_t, k, parts, keys, sums,
                           (T *)values, labels, rest);
        if (parts > 1)
            hipLaunchKernelGGL(top_join_kernel<T>, dim3(in.rows), dim3(kWaveTopThreads), 0, st, in, c2, inv_t, k, parts, keys, sums, (T *)values, labels,
                               rest);
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
    Rows in;
    if (make_rows(in, "", dtype, N, C, S, 0, 1, 0) || k < 1 || k > MFL_MAX_TOP_LABELS) return 0;
    const int parts = top_parts(in.rows, in.C);
    return parts > 1 ? (size_t)in.rows * parts * (part_keys(k) * sizeof(uint64_t) + sizeof(LogSum)) : 0;
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
    const size_t need = by_waves(in, k) ? mfl_top_labels_workspace_bytes(N, C, S, dtype, k) : 0;
    if (need && (!workspace || workspace_bytes < need)) return MFL_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run<float>(in, temperature, k, values, labels, rest, workspace, st);
    case MFL_BF16: return run<bf16_t>(in, temperature, k, values, labels, rest, workspace, st);
    default: return run<f16_t>(in, temperature, k, values, labels, rest, workspace, st);
    }
}

}  // extern "C"
