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
// Shapes of work: one lane per row (label maps), one wave or workgroup per row where top_k cuts the row to a short list
// (mfl_wave_top.h), and one workgroup per row otherwise, which finds the cut by a histogram of the weights.
//
// A row without a finite largest score (all -inf, or a NaN or +inf among them) has no distribution: label -1, logprob -inf.
#include "mfl_wave_top.h"

namespace {

using namespace mfl_scores;

typedef __attribute__((address_space(3))) double lds_double;

struct Settings {
    double t, top_p, min_p;
    int top_k;
    const float *t_n, *top_p_n, *min_p_n;
    const int *top_k_n;
};
struct Filter {
    double inv_t, top_p, min_p;
    int top_k;                  // INT_MAX: no limit
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
    if (!(r.min_p > 0)) r.min_p = 0;
    if (r.min_p > 1) r.top_k = 1, r.min_p = 0;
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

template <typename T> struct RowOf {
    const T *p;
    unsigned n;
    __device__ RowOf(const Rows &in, unsigned r)
    {
        n = r / in.S;
        p = (const T *)in.p + (long long)n * in.sn + (long long)(r - n * in.S) * in.ss;
    }
};

// ---- one lane per row
//
// Without top_k and top_p the labels are streamed once, in blocks: a block's weights next to its own largest score, summed;
// at the end the block sums are put on one scale, the draw names a block, and that block is read again for the label.  With
// top_k or top_p the lane keeps its best labels (Best), and looks for the draw among them; where top_p needs more labels than
// the list holds, a binary search over the rank keys finds the cut.

constexpr int kLaneThreads = 256;
constexpr int kLoneBlock = 24;          // up to this many labels a lane's scores stay in registers
constexpr int kBlocks = 8;              // block sums a lane keeps
constexpr int kBlock = 32;              // labels in flight

template <typename T, int CB> __device__ inline void load_block(float (&x)[CB], const T *p, long long sc, int c0, int C)
{
    T raw[CB];
    const T *q = p + c0 * sc;
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        raw[i] = *q;
        q += c0 + i + 1 < C ? sc : 0;           // (the last one again)
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) x[i] = i == 0 || c0 + i < C ? to_float(raw[i]) : -INFINITY;
}
template <int CB> __device__ inline float largest_of(const float (&x)[CB], float m)
{
#pragma unroll
    for (int i = 0; i < CB; ++i) m = max_or_nan(m, x[i]);
    return m;
}
// Weights that min_p keeps.  (No score above -inf: all 0.)
template <int CB> __device__ inline void weights_of(double (&w)[CB], const float (&x)[CB], const Weight &weight, double min_p)
{
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const double v = weight(x[i]);
        w[i] = v >= min_p ? v : 0.0;
    }
}
// The first of a block's labels whose running sum, from `run` on, exceeds the target, else the last that weighs something
template <int CB> __device__ inline void pick(const double (&w)[CB], double run, double target, int &label, double &got)
{
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const bool open = w[i] > 0 && !(label >= 0 && run > target);
        run += open ? w[i] : 0.0;
        label = open ? i : label;
        got = open ? w[i] : got;
    }
}

// All labels in registers
template <typename T, int CB>
__global__ void __launch_bounds__(kLaneThreads)
plain_lone_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    float x[CB];
    load_block(x, row.p, in.sc, 0, in.C);
    const float u = uniform[r];
    const Filter f = filter_of(set, row.n, in.C);
    const float m = largest_of(x, -INFINITY);
    if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    const Weight weight = {m, f.inv_t * kLog2eD};
    double w[CB], total = 0;
    weights_of(w, x, weight, f.min_p);
#pragma unroll
    for (int i = 0; i < CB; ++i) total += w[i];
    int label = -1;
    double got = 0;
    pick(w, 0.0, draw_of(u) * total, label, got);
    put(out, r, label, log(got / total));
}

struct LaneSums {
    double sum[kBlocks][kLaneThreads];
    float top[kBlocks][kLaneThreads];
};
template <typename T>
__device__ inline void plain_lane(const Rows &in, const T *p, const Filter &f, float u, unsigned r, const Out &out, LaneSums &sh)
{
    const int per = (in.C + kBlocks * kBlock - 1) / (kBlocks * kBlock) * kBlock, blocks = (in.C + per - 1) / per;
    const double a = f.inv_t * kLog2eD;
    float m = -INFINITY, x[kBlock];
    if (f.min_p > 0) {          // the threshold needs the largest score first
        for (int c = 0; c < in.C; c += kBlock) {
            load_block(x, p, in.sc, c, in.C);
            m = largest_of(x, m);
        }
        if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    }
    double w[kBlock];
    for (int b = 0; b < blocks; ++b) {
        double sum = 0;
        float top = m;
        for (int c = b * per; c < min(in.C, (b + 1) * per); c += kBlock) {
            load_block(x, p, in.sc, c, in.C);
            if (!(f.min_p > 0)) {
                const float next = largest_of(x, top);
                if (c > b * per && next != top) sum *= Weight{next, a}(top);
                top = next;
            }
            // (labels of the next block, where the block's size is not a multiple of what is in flight: there are none)
            weights_of(w, x, Weight{top == -INFINITY ? 0.0 : (double)top, a}, f.min_p);
#pragma unroll
            for (int i = 0; i < kBlock; ++i) sum += w[i];
        }
        sh.sum[b][threadIdx.x] = sum;
        sh.top[b][threadIdx.x] = top;
    }
    if (!(f.min_p > 0)) {
        for (int b = 0; b < blocks; ++b) m = max_or_nan(m, sh.top[b][threadIdx.x]);
        if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    }
    const Weight weight = {m, a};
    double total = 0;
    for (int b = 0; b < blocks; ++b) {
        const double s = sh.sum[b][threadIdx.x] * weight(sh.top[b][threadIdx.x]);
        sh.sum[b][threadIdx.x] = s;
        total += s;
    }
    const double target = draw_of(u) * total;
    double front = 0, run = 0;
    int block = 0;
    bool past = false;
    for (int b = 0; b < blocks; ++b) {
        const double s = sh.sum[b][threadIdx.x];
        if (s > 0 && !past) {
            block = b;
            front = run;
        }
        run += s;
        past = past || (s > 0 && run > target);
    }
    int label = -1;
    double got = 0;
    for (int c = block * per; c < min(in.C, (block + 1) * per); c += kBlock) {
        load_block(x, p, in.sc, c, in.C);
        weights_of(w, x, weight, f.min_p);
        int here = -1;
        double v = 0;
        pick(w, front, target, here, v);
#pragma unroll
        for (int i = 0; i < kBlock; ++i) front += w[i];
        if (here >= 0) {
            label = c + here;
            got = v;
        }
        if (here >= 0 && front > target) break;
    }
    put(out, r, label, log(got / total));
}

template <typename T>
__global__ void __launch_bounds__(kLaneThreads)
plain_lanes_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    __shared__ LaneSums sh;
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    plain_lane(in, row.p, filter_of(set, row.n, in.C), uniform[r], r, out, sh);
}

// The cut by a binary search over the rank keys, then the draw: for any settings
template <typename T>
__device__ inline void search_lane(const Rows &in, const T *p, const Filter &f, float u, unsigned r, const Out &out)
{
    int mk = (int)0x80000000;
    for (int c = 0; c < in.C; ++c) mk = max(mk, score_key(to_float(p[c * in.sc])));
    const float m = key_score(mk);
    if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    const Weight weight = {m, f.inv_t * kLog2eD};
    auto search = [&](auto reached) {
        uint64_t k = 0;
        for (int b = 63; b >= 0; --b)
            if (reached(k | 1ull << b)) k |= 1ull << b;
        return k;
    };
    uint64_t cut = 0;                               // kept by rank: rank_key >= cut
    if (f.top_k < in.C)
        cut = search([&](uint64_t k) {
            int count = 0;
            for (int c = 0; c < in.C; ++c) count += rank_key(score_key(to_float(p[c * in.sc])), c) >= k;
            return count >= f.top_k;
        });
    if (f.top_p < 1) {
        auto mass = [&](uint64_t from) {
            double sum = 0;
            for (int c = 0; c < in.C; ++c) {
                const float x = to_float(p[c * in.sc]);
                if (rank_key(score_key(x), c) >= from) sum += weight(x);
            }
            return sum;
        };
        const double goal = f.top_p * mass(cut);
        const uint64_t nucleus = search([&](uint64_t k) {
            const double sum = mass(k > cut ? k : cut);
            return sum > 0 && sum >= goal;
        });
        cut = nucleus > cut ? nucleus : cut;
    }
    auto kept_weight = [&](float x, int c) {
        const double w = weight(x);
        return w >= f.min_p && rank_key(score_key(x), c) >= cut ? w : 0.0;
    };
    double total = 0;
    for (int c = 0; c < in.C; ++c) total += kept_weight(to_float(p[c * in.sc]), c);
    const double target = draw_of(u) * total;
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

// The K best of the row; MASS: also what all labels weigh, for a top_p of more than the list.  Returns false where the list
// does not reach.
template <typename T, int K, bool MASS>
__device__ inline bool list_lane(const Rows &in, const T *p, const Filter &f, float u, unsigned r, const Out &out)
{
    Best<K> best;
    constexpr int U = 8;
    const double a = f.inv_t * kLog2eD;
    double mass = 0;
    float m = -INFINITY;
    for (int c = 0; c < in.C; c += U) {
        float x[U];
        load_block(x, p, in.sc, c, in.C);
        if (MASS) {
            const float next = largest_of(x, m);
            if (next != m) mass = m == -INFINITY ? 0.0 : mass * Weight{next, a}(m);
            m = next;
            if (m > -INFINITY) {
                const Weight weight = {m, a};
#pragma unroll
                for (int i = 0; i < U; ++i) mass += weight(x[i]);
            }
        }
        // (behind the last label: the lowest place of all, below every label's)
#pragma unroll
        for (int i = 0; i < U; ++i) best.insert(c + i < in.C ? place_of(x[i], c + i) : 0.0);
    }
    m = place_score(best.v[0]);
    if (!(fabsf(m) < INFINITY)) {
        put(out, r, -1, -INFINITY);
        return true;
    }
    const Weight weight = {m, a};
    double w[K], total = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        w[j] = j < f.top_k && best.v[j] != 0.0 ? weight(place_score(best.v[j])) : 0.0;
        total += w[j];
    }
    if (MASS && f.top_k > K) total = mass;
    const double goal = f.top_p * total;
    double front = 0, sum = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const bool keep = j == 0 || ((f.top_p >= 1 || front < goal) && w[j] >= f.min_p);
        front += w[j];
        w[j] = keep ? w[j] : 0.0;
        sum += w[j];
    }
    if (MASS && f.top_k > K && in.C > K && (f.top_p >= 1 || front < goal)) return false;
    // label by label, in label order, until the running sum is past the target
    const double target = draw_of(u) * sum;
    double run = 0, got = 0;
    int label = -1;
    for (;;) {
        int next = 0x7fffffff;
        double v = 0;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int l = place_label(best.v[j]);
            const bool here = w[j] > 0 && l > label && l < next;
            next = here ? l : next;
            v = here ? w[j] : v;
        }
        if (next == 0x7fffffff) break;
        run += v;
        label = next;
        got = v;
        if (run > target) break;
    }
    put(out, r, label, log(got / sum));
    return true;
}

template <typename T, int K>
__global__ void __launch_bounds__(kLaneThreads)
list_lanes_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    list_lane<T, K, false>(in, row.p, filter_of(set, row.n, in.C), uniform[r], r, out);
}

// Any settings, of each n its own
constexpr int kAnyList = 16;
template <typename T>
__global__ void __launch_bounds__(kLaneThreads)
any_lanes_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    __shared__ LaneSums sh;
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    const float u = uniform[r];
    if (f.top_k >= in.C && f.top_p >= 1) return plain_lane(in, row.p, f, u, r, out, sh);
    if (in.C <= kBestLabels && (f.top_k <= kAnyList || f.top_k >= in.C) && list_lane<T, kAnyList, true>(in, row.p, f, u, r, out)) return;
    search_lane(in, row.p, f, u, r, out);
}

// ---- rows that top_k cuts to a short list

// One wave: draws from the list (at most 128 keys, in any order) of the row's best labels
template <bool REST>
__device__ inline void draw_from_list(const WaveTop<REST> &top, const Filter &f, float u, unsigned r, const Out &out, lds_double *share)
{
    const int lane = threadIdx.x & 63;
    uint64_t key[2], best = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        key[h] = lane + 64 * h < top.count ? top.list[lane + 64 * h] : 0;
        best = key[h] > best ? key[h] : best;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)best, o);
        best = other > best ? other : best;
    }
    const float m = rank_score(best);
    if (!(fabsf(m) < INFINITY)) {
        if (lane == 0) put(out, r, -1, -INFINITY);
        return;
    }
    const Weight weight = {m, f.inv_t * kLog2eD};
    double w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w[h] = key[h] ? weight(rank_score(key[h])) : 0.0;
        share[lane + 64 * h] = w[h];
    }
    __builtin_amdgcn_wave_barrier();
    if (f.top_p < 1 || f.min_p > 0 || f.top_k < top.count) {
        double front[2] = {0, 0}, total = 0;
        int above[2] = {0, 0};
        for (int j = 0; j < top.count; ++j) {
            const uint64_t other = top.list[j];
            const double v = share[j];
            total += v;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                front[h] += other > key[h] ? v : 0.0;
                above[h] += other > key[h];
            }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool keep = key[h] == best || (above[h] < f.top_k && (front[h] < f.top_p * total || f.top_p >= 1) && w[h] >= f.min_p);
            w[h] = keep ? w[h] : 0.0;
            share[lane + 64 * h] = w[h];
        }
        __builtin_amdgcn_wave_barrier();
    }
    // running sums in label order
    double upto[2] = {0, 0}, total = 0;
    for (int j = 0; j < top.count; ++j) {
        const int other = rank_label(top.list[j]);
        const double v = share[j];
        total += v;
#pragma unroll
        for (int h = 0; h < 2; ++h) upto[h] += other <= rank_label(key[h]) ? v : 0.0;
    }
    const double target = draw_of(u) * total;
    int hit = 0x7fffffff, last = -1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (w[h] > 0) {
            if (upto[h] > target) hit = min(hit, rank_label(key[h]));
            last = max(last, rank_label(key[h]));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        hit = min(hit, __shfl_xor(hit, o));
        last = max(last, __shfl_xor(last, o));
    }
    const int label = hit == 0x7fffffff ? last : hit;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (key[h] && rank_label(key[h]) == label) put(out, r, label, log(w[h] / total));
}

template <typename T>
__global__ void __launch_bounds__(kWaveTopThreads)
list_waves_kernel(Rows in, Settings set, int k, const float *__restrict__ uniform, Out out)
{
    __shared__ uint64_t lists[kWaveTopThreads / 64][kListKeys];
    __shared__ double share[kWaveTopThreads / 64][MFL_MAX_TOP_LABELS];
    const int wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x * (kWaveTopThreads / 64) + wave;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    WaveTop<false> top(lists[wave], k, 0.f);
    if (in.sc == 1 && in.C >= 8 * 64 * kVec<T>) {
        float m[4];
        top.look(row.p, 0, 4, m);
        top.foresee(m);
    }
    top.stream(row.p, in.sc, 0, in.C);
    top.cut();
    draw_from_list(top, filter_of(set, row.n, in.C), uniform[r], r, out, (lds_double *)share[wave]);
}

template <typename T>
__global__ void __launch_bounds__(kWaveTopThreads)
list_parts_kernel(Rows in, Settings set, int k, int parts, const float *__restrict__ uniform, uint64_t *__restrict__ keys, Out out)
{
    __shared__ TopShared sh;
    __shared__ double share[MFL_MAX_TOP_LABELS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const RowOf<T> row(in, r);
    WaveTop<false> top(sh.lists[wave], k, 0.f);
    const int size = top_part_labels(in.C, parts);
    const int begin = min(in.C, (int)part * size), end = min(in.C, begin + size);
    if (!top_of_part(top, sh, row.p, in.sc, begin, end)) return;
    if (parts == 1) return draw_from_list(top, filter_of(set, row.n, in.C), uniform[r], r, out, (lds_double *)share);
    for (int j = lane; j < k; j += 64) keys[(size_t)blockIdx.x * k + j] = j < top.count ? top.list[j] : 0;
}

template <typename T>
__global__ void __launch_bounds__(64)
list_join_kernel(Rows in, Settings set, int k, int parts, const float *__restrict__ uniform, const uint64_t *__restrict__ keys, Out out)
{
    __shared__ uint64_t list[kListKeys];
    __shared__ double share[MFL_MAX_TOP_LABELS];
    const unsigned r = blockIdx.x;
    WaveTop<false> top(list, k, 0.f);
    top.join(keys + (size_t)r * parts * k, parts * k);
    top.cut();
    draw_from_list(top, filter_of(set, r / in.S, in.C), uniform[r], r, out, (lds_double *)share);
}

// ---- rows of many labels, any settings: one workgroup per row
//
//   1  the largest score
//   2  where top_k or top_p cut: a histogram over 2048 bins of (largest - score) / T, 32 a unit: counts, and masses as
//      64-bit fixed point (2^51 or less for the largest weight, so that C of them fit), whose sums do not depend on the
//      order of the atomics; running sums over the bins name the bin that the cut falls into
//   3  that bin's labels, a list in LDS; every one counts what lies above it in the list, and the lowest that stays is the
//      cut.  (A bin of more labels than the list holds, all of nearly one score: a binary search over the rank keys.)
//   4  the kept weights summed in runs of neighbouring labels, the run that the draw falls into, the label in it
//
// Steps 2 to 4 read the row again, from the caches if it fits.  Weights below the cut cost a compare in step 4.

constexpr int kBins = 2048;
constexpr float kBinsPerUnit = 32.f;
constexpr int kRuns = 1024;
constexpr int kBinList = 2048;

template <typename V, int NT> __device__ inline V block_sum(V v, V *part)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < NT / 64; ++w) v += part[w];
    return v;
}
// Sum over the threads in front, and over all
template <typename V, int NT> __device__ inline V block_front(V v, V *part, V &all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V other = __shfl_up(upto, o);
        if (lane >= o) upto += other;
    }
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    V before = 0;
    all = 0;
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) before = all;
        all += part[w];
    }
    const V ahead = __shfl_up(upto, 1);
    return before + (lane ? ahead : V(0));
}

template <typename T, int NT> struct BlockRow {
    struct Shared {
        uint32_t counts[kBins];
        unsigned long long masses[kBins];
        unsigned long long key[kBinList], key_mass[kBinList];
        double runs[kRuns];
        unsigned long long upart[NT / 64];
        double dpart[NT / 64];
        float fpart[NT / 64];
        unsigned listed, bin;
        unsigned long long bin_front, low_key;
    };
    Shared &sh;
    const T *p;
    long long sc;
    int C;
    float m, scale;
    Weight weight;
    int bits;                   // of the fixed-point masses

    __device__ int bin_of(float x) const { return min((int)((m - x) * scale), kBins - 1); }
    __device__ uint64_t mass(float x) const
    {
        // 2^52 + an integer below 2^52: the low bits of the sum are that integer
        const double v = __builtin_ldexp(weight(x), bits) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xfffffffffffffull;
    }
    // f(score, label) over the row
    template <typename F> __device__ void each(F f) const
    {
        if (sc == 1) {
            constexpr int V = kVec<T>, U = 2;
            int c = threadIdx.x * V;
            for (; c + (U - 1) * NT * V + V <= C; c += U * NT * V) {
                float x[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u) load_vec(p + c + u * NT * V, x[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < V; ++i) f(x[u][i], c + u * NT * V + i);
            }
            for (; c < C; c += NT * V) {
                if (c + V <= C) {
                    float x[V];
                    load_vec(p + c, x);
#pragma unroll
                    for (int i = 0; i < V; ++i) f(x[i], c + i);
                } else {
                    for (int i = c; i < C; ++i) f(to_float(p[i]), i);
                }
            }
        } else {
            for (int c = threadIdx.x; c < C; c += NT) f(to_float(p[c * sc]), c);
        }
    }

    __device__ void largest()
    {
        float v = -INFINITY;
        each([&](float x, int) { v = max_or_nan(v, x); });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = max_or_nan(v, __shfl_xor(v, o));
        if ((threadIdx.x & 63) == 0) sh.fpart[threadIdx.x >> 6] = v;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) v = max_or_nan(v, sh.fpart[w]);
        m = v;
    }

    // The lowest rank key that stays, where labels of at least `low` stay while front < goal, front = what the labels above
    // hold: their number (COUNT) or mass.  The sum over everything is at least goal.
    template <bool COUNT> __device__ uint64_t cut_at(double goal, uint64_t low)
    {
        // the bin it falls into, and what the bins in front of it hold
        constexpr int per = kBins / NT;
        unsigned long long mine = 0, all;
        for (int i = 0; i < per; ++i) mine += COUNT ? sh.counts[threadIdx.x * per + i] : sh.masses[threadIdx.x * per + i];
        unsigned long long front = block_front<unsigned long long, NT>(mine, sh.upart, all);
        if (threadIdx.x == 0) sh.listed = 0, sh.low_key = ~0ull;
        if ((double)front < goal && (double)(front + mine) >= goal) {
            int b = threadIdx.x * per;
            for (;; ++b) {
                const unsigned long long here = COUNT ? sh.counts[b] : sh.masses[b];
                if ((double)(front + here) >= goal) break;
                front += here;
            }
            sh.bin = b;
            sh.bin_front = front;
        }
        __syncthreads();
        const int bin = sh.bin;
        front = sh.bin_front;
        each([&](float x, int c) {
            if (bin_of(x) != bin) return;
            const uint64_t key = rank_key(score_key(x), c);
            if (key < low) return;
            const unsigned at = atomicAdd(&sh.listed, 1u);
            if (at >= (unsigned)kBinList) return;
            sh.key[at] = key;
            sh.key_mass[at] = COUNT ? 1 : mass(x);
        });
        __syncthreads();
        const int n = sh.listed;
        if (n <= kBinList) {
            for (int i = threadIdx.x; i < n; i += NT) {
                const uint64_t key = sh.key[i];
                unsigned long long above = 0;
                for (int j = 0; j < n; ++j) above += sh.key[j] > key ? sh.key_mass[j] : 0;
                if ((double)(front + above) < goal) atomicMin(&sh.low_key, key);
            }
            __syncthreads();
            return sh.low_key;
        }
        // the largest key from which on at least `goal` is held
        uint64_t best = 0;
        for (int b = 63; b >= 0; --b) {
            const uint64_t at = best | 1ull << b, from = at > low ? at : low;
            unsigned long long held = 0;
            each([&](float x, int c) {
                if (bin_of(x) == bin && rank_key(score_key(x), c) >= from) held += COUNT ? 1 : mass(x);
            });
            held = block_sum<unsigned long long, NT>(held, sh.upart);
            if ((double)(front + held) >= goal) best = at;
        }
        return best > low ? best : low;
    }

    // The lowest rank key that top_k and top_p keep
    __device__ uint64_t cut(const Filter &f)
    {
        for (int i = threadIdx.x; i < kBins; i += NT) sh.counts[i] = 0, sh.masses[i] = 0;
        __syncthreads();
        const bool count = f.top_k < C, masses = f.top_p < 1;
        each([&](float x, int) {
            const int b = bin_of(x);
            if (count) atomicAdd(&sh.counts[b], 1u);
            if (masses) {
                const uint64_t v = mass(x);
                if (v) atomicAdd(&sh.masses[b], (unsigned long long)v);
            }
        });
        __syncthreads();
        uint64_t low = 0;
        if (count) {
            low = cut_at<true>((double)f.top_k, 0);
            if (masses) {
                // what is left of the bin, and nothing behind it
                const int bin = bin_of(rank_score(low));
                unsigned long long left = 0;
                each([&](float x, int c) {
                    if (bin_of(x) == bin && rank_key(score_key(x), c) >= low) left += mass(x);
                });
                left = block_sum<unsigned long long, NT>(left, sh.upart);
                for (int i = threadIdx.x; i < kBins; i += NT)
                    if (i >= bin) sh.masses[i] = i == bin ? left : 0;
                __syncthreads();
            }
        }
        if (masses) {
            unsigned long long mine = 0;
            for (int i = threadIdx.x; i < kBins; i += NT) mine += sh.masses[i];
            const double total = (double)block_sum<unsigned long long, NT>(mine, sh.upart);
            const double goal = f.top_p * total;
            // (nothing to reach: the first label stays alone)
            low = goal > 0 ? cut_at<false>(goal, low) : cut_at<true>(1.0, 0);
        }
        return low;
    }

    // Step 4.  cut: lowest rank key that stays
    __device__ void draw(uint64_t cut, double min_p, float u, unsigned r, const Out &out)
    {
        constexpr int V = kVec<T>, step = 64 * V;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int tiles = (C + step - 1) / step, per = (tiles + kRuns - 1) / kRuns, runs = (tiles + per - 1) / per;
        const float cut_score = cut ? rank_score(cut) : -INFINITY;
        // a tile's kept weights
        auto tile = [&](int t, double (&w)[V]) {
            const int c = t * step + lane * V;
            float x[V];
            if (sc == 1 && c + V <= C) {
                load_vec(p + c, x);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = c + i < C ? to_float(p[(c + i) * sc]) : -INFINITY;
            }
            float best = x[0];
#pragma unroll
            for (int i = 1; i < V; ++i) best = fmaxf(best, x[i]);
            const bool some = __any(best >= cut_score && best > -INFINITY);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                w[i] = 0;
                if (some && x[i] >= cut_score && rank_key(score_key(x[i]), c + i) >= cut) {
                    const double v = weight(x[i]);
                    w[i] = v >= min_p ? v : 0.0;
                }
            }
            return some;
        };
        for (int e = wave; e < runs; e += NT / 64) {
            double sum = 0;
            for (int t = e * per; t < min(tiles, (e + 1) * per); ++t) {
                double w[V];
                if (!tile(t, w)) continue;
#pragma unroll
                for (int i = 0; i < V; ++i) sum += w[i];
            }
            if (__any(sum > 0)) {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
            }
            if (lane == 0) sh.runs[e] = sum;
        }
        __syncthreads();
        // the run that the draw falls into, or the last one that holds something
        constexpr int mine = kRuns / NT > 0 ? kRuns / NT : 1;
        double sum = 0, all;
        int last = -1;
        for (int i = 0; i < mine; ++i) {
            const int e = threadIdx.x * mine + i;
            if (e < runs && sh.runs[e] > 0) sum += sh.runs[e], last = e;
        }
        double front = block_front<double, NT>(sum, sh.dpart, all);
        if (threadIdx.x == 0) sh.bin = 0, sh.listed = ~0u;
        __syncthreads();
        if (last >= 0) atomicMax(&sh.bin, (unsigned)last);
        const double target = draw_of(u) * all;
        if (sum > 0 && front + sum > target) {       // (the lowest run wins)
            for (int i = 0; i < mine; ++i) {
                const int e = threadIdx.x * mine + i;
                const double next = front + (e < runs ? sh.runs[e] : 0.0);
                if (next > target) {
                    atomicMin(&sh.listed, (unsigned)e);
                    break;
                }
                front = next;
            }
        }
        __syncthreads();
        const int run = sh.listed != ~0u ? (int)sh.listed : (int)sh.bin;
        if (wave) return;
        front = 0;
        for (int i = lane; i < run; i += 64) front += sh.runs[i];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) front += __shfl_xor(front, o);
        int label = -1;
        double got = 0;
        for (int t = run * per; t < min(tiles, (run + 1) * per); ++t) {
            double w[V];
            if (!tile(t, w)) continue;
            double own = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) own += w[i];
            double upto = own;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double other = __shfl_up(upto, o);
                if (lane >= o) upto += other;
            }
            // the first lane past the target, else the last one that holds something (so far)
            const uint64_t past = __ballot(own > 0 && front + upto > target), holds = __ballot(own > 0);
            if (past || holds) {
                const int who = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)holds);
                double run_sum = front + upto - own;
                int l = -1;
                double g = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const bool open = w[i] > 0 && !(l >= 0 && run_sum > target);
                    run_sum += open ? w[i] : 0.0;
                    l = open ? t * step + lane * V + i : l;
                    g = open ? w[i] : g;
                }
                label = __shfl(l, who);
                got = __shfl(g, who);
            }
            if (past) break;
            front += __shfl(upto, 63);
        }
        if (lane == 0) put(out, r, label, log(got / all));
    }
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT)
sample_blocks_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    __shared__ typename BlockRow<T, NT>::Shared sh;
    const unsigned r = blockIdx.x;
    const RowOf<T> at(in, r);
    const Filter f = filter_of(set, at.n, in.C);
    const int wide = 32 - __builtin_clz(in.C);      // C < 2^wide
    BlockRow<T, NT> row = {sh, at.p, in.sc, in.C, 0.f, 0.f, {}, min(51, 62 - wide)};
    row.largest();
    if (!(fabsf(row.m) < INFINITY)) {
        if (threadIdx.x == 0) put(out, r, -1, -INFINITY);
        return;
    }
    row.scale = (float)fmin(f.inv_t * kBinsPerUnit, 1e30);
    row.weight = {row.m, f.inv_t * kLog2eD};
    const uint64_t cut = f.top_k < in.C || f.top_p < 1 ? row.cut(f) : 0;
    __syncthreads();
    row.draw(cut, f.min_p, uniform[r], r, out);
}

// top_k for all rows, and short enough for a list (temperature 0: the best one)
int list_length(const Settings &set)
{
    if (set.top_k_n) return 0;
    if (!set.t_n && set.t == 0) return 1;
    return set.top_k >= 1 && set.top_k <= MFL_MAX_TOP_LABELS ? set.top_k : 0;
}
bool by_lanes(const Rows &in) { return !(in.sc == 1 && in.C >= 256); }

template <typename T>
int run(const Rows &in, const Settings &set, const float *uniform, const Out &out, void *workspace, hipStream_t st)
{
    if (by_lanes(in)) {
        const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
#define MFL_LANES(...) hipLaunchKernelGGL(__VA_ARGS__, grid, block, 0, st, in, set, uniform, out)
        // what the list has to hold: top_k, or with top_p alone every label
        const bool no_k = !set.top_k_n && (set.top_k == 0 || set.top_k >= in.C), no_p = !set.top_p_n && set.top_p == 1;
        const bool same_t = !set.t_n && set.t > 0, below_1 = !set.min_p_n;
        const int k = list_length(set) ? list_length(set) : no_k && in.C <= 32 ? in.C : 0;
        if (no_k && no_p && same_t && below_1) {
            if (in.C <= 8) MFL_LANES((plain_lone_kernel<T, 8>));
            else if (in.C <= kLoneBlock) MFL_LANES((plain_lone_kernel<T, kLoneBlock>));
            else MFL_LANES((plain_lanes_kernel<T>));
        } else if (k && k <= 32 && in.C <= kBestLabels) {
            if (k <= 1) MFL_LANES((list_lanes_kernel<T, 1>));
            else if (k <= 4) MFL_LANES((list_lanes_kernel<T, 4>));
            else if (k <= 8) MFL_LANES((list_lanes_kernel<T, 8>));
            else if (k <= 16) MFL_LANES((list_lanes_kernel<T, 16>));
            else if (k <= 24) MFL_LANES((list_lanes_kernel<T, 24>));
            else MFL_LANES((list_lanes_kernel<T, 32>));
        } else {
            MFL_LANES((any_lanes_kernel<T>));
        }
#undef MFL_LANES
        return (int)hipGetLastError();
    }
    const int k = list_length(set) < in.C ? list_length(set) : 0;
    if (k) {
        if (in.C < kBlockLabels) {
            const unsigned per = kWaveTopThreads / 64;
            hipLaunchKernelGGL(list_waves_kernel<T>, dim3((in.rows + per - 1) / per), dim3(kWaveTopThreads), 0, st, in, set, k, uniform, out);
            return (int)hipGetLastError();
        }
        const int parts = top_parts(in.rows, in.C);
        uint64_t *keys = (uint64_t *)workspace;
        hipLaunchKernelGGL(list_parts_kernel<T>, dim3(in.rows * parts), dim3(kWaveTopThreads), 0, st, in, set, k, parts, uniform, keys, out);
        if (parts > 1) hipLaunchKernelGGL(list_join_kernel<T>, dim3(in.rows), dim3(64), 0, st, in, set, k, parts, uniform, keys, out);
        return (int)hipGetLastError();
    }
    if (in.C <= 4096) hipLaunchKernelGGL((sample_blocks_kernel<T, 256>), dim3(in.rows), dim3(256), 0, st, in, set, uniform, out);
    else hipLaunchKernelGGL((sample_blocks_kernel<T, 1024>), dim3(in.rows), dim3(1024), 0, st, in, set, uniform, out);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t mfl_sample_labels_workspace_bytes(int N, int C, int S, int dtype)
{
    Rows in;
    if (make_rows(in, "", dtype, N, C, S, 0, 1, 0) || C < kBlockLabels) return 0;
    const int parts = top_parts(in.rows, in.C);
    return parts > 1 ? (size_t)in.rows * parts * MFL_MAX_TOP_LABELS * sizeof(uint64_t) : 0;
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
    const size_t need = by_lanes(in) ? 0 : mfl_sample_labels_workspace_bytes(N, C, S, dtype);
    if (need && (!workspace || workspace_bytes < need)) return MFL_ERR_WORKSPACE;
    const Settings set = {temperature, top_p, min_p, top_k, temperature_n, top_p_n, min_p_n, top_k_n};
    const Out out = {labels, label_bytes, logprob};
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run<float>(in, set, uniform, out, workspace, st);
    case MFL_BF16: return run<bf16_t>(in, set, uniform, out, workspace, st);
    default: return run<f16_t>(in, set, uniform, out, workspace, st);
    }
}

}  // extern "C"
