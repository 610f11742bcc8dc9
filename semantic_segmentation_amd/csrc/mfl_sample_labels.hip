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
// sums (10^-7) would misplace about one draw in a hundred, and a batch of maps has millions of draws.  The masses of a
// histogram are integers, a label's rounded to a part in 2^min(51, 62 - bits of C) of itself (2^45 at 128 000 labels, 2^31
// at the most that a call takes), however far below the largest weight it lies (Bins).
//
// Settings may differ from n to n (arrays of N).  T <= 0 takes the largest; top_k <= 0, top_p >= 1 and min_p <= 0 keep all.
// Shapes of work: one lane per row (label maps), one wave or workgroup per row where top_k cuts the row to a short list
// (mfl_wave_top.h), and one workgroup per row otherwise, which finds the cut by a histogram of the weights.
//
// Measured on MI355X.  Lanes: 8 x 21 x 512 x 512 fp32 without filters 58 us (3.6 TB/s; a 64-bit exponential is 17
// instructions, so the vector unit is about as busy as the memory), top_p alone 210 (every label is sorted into the list);
// 2 x 150 x 512 x 512 with top_k 5, top_p and min_p 78 us (4.0 TB/s), top_p alone 1007.  Rows: 1 x 128000 bf16, top_k 50, 21 us
// and 64 x 50001 f16 without filters 20 us (two launches; the second is 12 us of one workgroup's work); 256 x 128000 fp32, every
// row its own temperature and top_p, 137 us: 25 the largest score (the rate of a copy), 40 the histogram (64-bit exponentials
// and LDS atomics), 43 the sweep, the rest scans and the pick; a binary search over whole passes instead of the histogram took
// 12.9 ms, a fourth pass for the runs 187 us.  Where the cut's bin holds more than its list of 2048, the row is gone over again:
// 64 x 200000 bf16 at T 1.3 and top_p 0.9 854 us (fp32 153), 4 x 128000 fp32 of standard deviation 0.05 3.5 ms (1: 91 us).
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
// the list holds, it goes on with the next best.

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

// All labels in registers.  The label is the number of running sums up to the target.
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
    double upto[CB], total = 0;
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        if (i == 0 || i + 4 <= CB || i < in.C) {        // (of the last ones, only those that are there)
            const double v = weight(x[i]);
            total += v >= f.min_p ? v : 0.0;
        }
        upto[i] = total;
    }
    const double target = draw_of(u) * total;
    int label = 0;
#pragma unroll
    for (int i = 0; i < CB; ++i) label += upto[i] <= target;
    if (label >= in.C) {                // past all of it: the last one that weighs something
        double before = 0;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            label = upto[i] > before ? i : label;
            before = upto[i];
        }
    }
    put(out, r, label, log(weight(to_float(row.p[label * in.sc])) / total));
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

// Takes one block after another into the list: the best labels of those placed before `last`
template <typename T, int K, typename F> __device__ inline void list_pass(Best<K> &best, const Rows &in, const T *p, double last, F seen)
{
    constexpr int U = 8;
    for (int c = 0; c < in.C; c += U) {
        float x[U];
        load_block(x, p, in.sc, c, in.C);
        seen(x);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const double v = place_of(x[i], c + i);
            best.insert(c + i < in.C && v < last ? v : 0.0);
        }
    }
}
constexpr double kBeforeAll = 2.0;

// The draw among the list's first labels: w holds what each keeps, sum all of it
template <int K> __device__ inline void draw_by_label(const Best<K> &best, const double (&w)[K], double sum, float u, unsigned r, const Out &out)
{
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
}

// The draw among the labels placed from `cut` on, with the scores read again
template <typename T>
__device__ inline void draw_from_cut(const Rows &in, const T *p, double cut, const Weight &weight, double min_p, float u, unsigned r, const Out &out)
{
    double sum = 0;
    auto kept = [&](const float (&x)[8], int c, double (&w)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double v = weight(x[i]);
            w[i] = c + i < in.C && v >= min_p && place_of(x[i], c + i) >= cut ? v : 0.0;
        }
    };
    for (int c = 0; c < in.C; c += 8) {
        float x[8];
        double w[8];
        load_block(x, p, in.sc, c, in.C);
        kept(x, c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += w[i];
    }
    const double target = draw_of(u) * sum;
    double run = 0, got = 0;
    int label = -1;
    for (int c = 0; c < in.C; c += 8) {
        float x[8];
        double w[8];
        load_block(x, p, in.sc, c, in.C);
        kept(x, c, w);
        int here = -1;
        double v = 0;
        pick(w, run, target, here, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) run += w[i];
        if (here >= 0) label = c + here, got = v;
        if (here >= 0 && run > target) break;
    }
    put(out, r, label, log(got / sum));
}
// ... of at most CB labels, in registers
template <int CB, typename T>
__device__ inline void draw_from_cut_lone(const Rows &in, const T *p, double cut, const Weight &weight, double min_p, float u, unsigned r, const Out &out)
{
    float x[CB];
    load_block(x, p, in.sc, 0, in.C);
    double upto[CB], total = 0;
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        const double v = weight(x[i]);
        total += i < in.C && v >= min_p && place_of(x[i], i) >= cut ? v : 0.0;
        upto[i] = total;
    }
    const double target = draw_of(u) * total;
    int label = 0;
#pragma unroll
    for (int i = 0; i < CB; ++i) label += upto[i] <= target;
    if (label >= in.C) {                // past all of it: the last one that weighs something
        double before = 0;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            label = upto[i] > before ? i : label;
            before = upto[i];
        }
    }
    put(out, r, label, log(weight(to_float(p[label * in.sc])) / total));
}

// The list holds all that top_k leaves, or (ALL) all labels: then the draw follows the scores once more instead of looking for
// one list entry after the other
template <typename T, int K, bool ALL>
__global__ void __launch_bounds__(kLaneThreads)
list_lanes_kernel(Rows in, Settings set, const float *__restrict__ uniform, Out out)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    const float u = uniform[r];
    Best<K> best;
    list_pass(best, in, row.p, kBeforeAll, [](const float (&)[8]) {});
    const float m = place_score(best.v[0]);
    if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    const Weight weight = {m, f.inv_t * kLog2eD};
    double w[K], total = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        w[j] = j < f.top_k && best.v[j] != 0.0 ? weight(place_score(best.v[j])) : 0.0;
        total += w[j];
    }
    const double goal = f.top_p * total;
    if constexpr (ALL) {
        double front = 0, cut = best.v[0];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            cut = w[j] > 0 && (f.top_p >= 1 || front < goal) ? best.v[j] : cut;
            front += w[j];
        }
        return draw_from_cut_lone<K>(in, row.p, cut, weight, f.min_p, u, r, out);
    }
    double front = 0, sum = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const bool keep = j == 0 || ((f.top_p >= 1 || front < goal) && w[j] >= f.min_p);
        front += w[j];
        w[j] = keep ? w[j] : 0.0;
        sum += w[j];
    }
    draw_by_label(best, w, sum, u, r, out);
}

// Any settings, of each n its own: the best K labels, then the next K, until the cut is found
template <typename T>
__device__ inline void ranked_lane(const Rows &in, const T *p, const Filter &f, float u, unsigned r, const Out &out)
{
    constexpr int K = 24;
    const double a = f.inv_t * kLog2eD;
    double mass = 0;            // of all labels
    float m = -INFINITY;
    Best<K> best;
    list_pass(best, in, p, kBeforeAll, [&](const float (&x)[8]) {
        const float next = largest_of(x, m);
        if (next != m) mass = m == -INFINITY ? 0.0 : mass * Weight{next, a}(m);
        m = next;
        if (m > -INFINITY && f.top_p < 1 && f.top_k >= in.C) {
            const Weight weight = {m, a};
#pragma unroll
            for (int i = 0; i < 8; ++i) mass += weight(x[i]);
        }
    });
    if (!(fabsf(m) < INFINITY)) return put(out, r, -1, -INFINITY);
    const Weight weight = {m, a};
    // goes on from the list in hand: stop(place, weight, rank) for one label after the other
    auto in_order = [&](auto stop) {
        int rank = 0;
        for (;;) {
            double last = 0;
            bool done = false;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (done || best.v[j] == 0.0) {
                    done = true;
                    continue;
                }
                last = best.v[j];
                done = stop(best.v[j], weight(place_score(best.v[j])), rank);
                ++rank;
            }
            if (done || rank >= in.C) return;
            best = Best<K>();
            list_pass(best, in, p, last, [](const float (&)[8]) {});
        }
    };
    const Best<K> first = best;
    double total = mass;
    if (f.top_p < 1 && f.top_k < in.C) {
        total = 0;
        in_order([&](double, double w, int rank) {
            total += w;
            return rank + 1 >= f.top_k;
        });
        best = first;
    }
    const double goal = f.top_p * total;
    double front = 0, cut = 0;
    in_order([&](double place, double w, int rank) {
        if (rank > 0 && (rank >= f.top_k || (f.top_p < 1 && !(front < goal)))) return true;
        cut = place;
        front += w;
        return false;
    });
    draw_from_cut(in, p, cut, weight, f.min_p, u, r, out);
}

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
    ranked_lane(in, row.p, f, u, r, out);
}

// ---- rows that top_k cuts to a short list: of at most k labels (rows of a longer one are passed over)

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
    if (f.top_k < top.count) {
        int above[2] = {0, 0};
        for (int j = 0; j < top.count; ++j) {
            const uint64_t other = top.list[j];
#pragma unroll
            for (int h = 0; h < 2; ++h) above[h] += other > key[h];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            w[h] = above[h] < f.top_k ? w[h] : 0.0;
            share[lane + 64 * h] = w[h];
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (f.top_p < 1 || f.min_p > 0) {
        double front[2] = {0, 0}, total = 0;
        for (int j = 0; j < top.count; ++j) {
            const uint64_t other = top.list[j];
            const double v = share[j];
            total += v;
#pragma unroll
            for (int h = 0; h < 2; ++h) front[h] += other > key[h] ? v : 0.0;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool keep = key[h] == best || ((front[h] < f.top_p * total || f.top_p >= 1) && w[h] >= f.min_p);
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
    const Filter f = filter_of(set, row.n, in.C);
    if (f.top_k > k) return;
    WaveTop<false> top(lists[wave], f.top_k, 0.f);
    if (in.sc == 1 && in.C >= 8 * 64 * kVec<T>) {
        float m[4];
        top.look(row.p, 0, 4, m);
        top.foresee(m);
    }
    top.stream(row.p, in.sc, 0, in.C);
    top.cut();
    draw_from_list(top, f, uniform[r], r, out, (lds_double *)share[wave]);
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
    const Filter f = filter_of(set, row.n, in.C);
    if (f.top_k > k) return;
    WaveTop<false> top(sh.lists[wave], f.top_k, 0.f);
    const int size = top_part_labels(in.C, parts);
    const int begin = min(in.C, (int)part * size), end = min(in.C, begin + size);
    if (!top_of_part(top, sh, row.p, in.sc, begin, end)) return;
    if (parts == 1) {
        top.cut();
        return draw_from_list(top, f, uniform[r], r, out, (lds_double *)share);
    }
    const int slots = part_keys(k);
    for (int j = lane; j < slots; j += 64) keys[(size_t)blockIdx.x * slots + j] = j < top.count ? top.list[j] : 0;
}

__global__ void __launch_bounds__(kWaveTopThreads)
list_join_kernel(Rows in, Settings set, int k, int parts, const float *__restrict__ uniform, const uint64_t *__restrict__ keys, Out out)
{
    __shared__ TopShared sh;
    __shared__ double share[MFL_MAX_TOP_LABELS];
    const unsigned r = blockIdx.x;
    const int n = parts * part_keys(k);
    const Filter f = filter_of(set, r / in.S, in.C);
    if (f.top_k > k) return;
    WaveTop<false> top(sh.lists[threadIdx.x >> 6], f.top_k, 0.f);
    if (!top_of_keys(top, sh, keys + (size_t)r * n, n)) return;
    top.cut();
    draw_from_list(top, f, uniform[r], r, out, (lds_double *)share);
}

// ---- rows of many labels, any settings: one workgroup per row
//
//   1  the largest score
//   2  where top_k or top_p cut: a histogram over 4096 bins of (largest - score) / T, 128 a unit (a quarter of that for short
//      rows): counts, and masses as 64-bit fixed point (2^51 or less for a bin's own largest weight, so that C of them fit),
//      whose sums do not depend on the order of the atomics; running sums over the bins name the bin that the cut falls into
//   3  that bin's labels, a list in LDS; every one counts what lies above it in the list, and the lowest that stays is the
//      cut.  (A bin of more labels than the list holds: where they share one score, counted along the row, else a binary
//      search over the rank keys.)  On the way the weights above the bin are summed in runs of neighbouring labels
//   4  the run that the draw falls into, and the label in it
//
// Steps 2 and 3 read the row again, from the caches if it fits; scores below the cut cost a compare in step 3.

// (all of it in one function, so that what lies in LDS is known to)
#define MFL_INLINE __device__ __attribute__((always_inline))

constexpr int kRuns = 256;
constexpr int kBinList = 2048;
constexpr float kUnits = 32.f;          // what the bins cover

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

// The bin in which a running sum over all threads' bins reaches the goal, and what is left of the goal there.  A thread has n
// bins, held(0) .. held(n - 1), with `front` in front of them.  (Sums of doubles, each rounded by itself: where they leave a
// gap at the goal, the next bin that holds something, or the last, has it.)  first = ~0 and last = 0 before, with a barrier
// between; some bin holds something.
struct Reach {
    unsigned first, last;
    int bin;
    double left;
};
template <typename F> MFL_INLINE void find_bin(int n, double front, double mine, double goal, F held, Reach &sh)
{
    const uint64_t holds = __ballot(mine > 0), past = __ballot(mine > 0 && front + mine >= goal);
    if ((threadIdx.x & 63) == 0) {
        if (past) atomicMin(&sh.first, threadIdx.x + __ffsll((unsigned long long)past) - 1);
        if (holds) atomicMax(&sh.last, threadIdx.x + 63 - __clzll((long long)holds));
    }
    __syncthreads();
    if (threadIdx.x == (sh.first != ~0u ? sh.first : sh.last)) {
        int at = -1;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const double here = held(i);
            if (here > 0 && (at < 0 || front < goal)) {
                at = i;
                sh.left = goal - front;
            }
            front += here;
        }
        sh.bin = threadIdx.x * n + max(at, 0);
    }
    __syncthreads();
}

// What the listed keys above one hold.  The list ends in zeros up to a multiple of eight, so that eight are on their way at once.
MFL_INLINE unsigned long long held_above(const unsigned long long *keys, const unsigned long long *masses, int n, uint64_t key)
{
    unsigned long long above = 0;
    for (int j = 0; j < n; j += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) above += keys[j + i] > key ? masses[j + i] : 0;
    }
    return above;
}

// Bins of (largest - score) / T and fixed-point masses of a row.  A bin's weights are at most 2^-edge(bin); its masses are
// integers in steps of 2^-(bits + edge(bin)).  (One step for all bins, next to the row's largest weight, would leave nothing of
// a tail that may hold 10^-7 of the mass at 10^6 labels, where draws are 2^-24 apart.)
template <int BINS> struct Bins {
    static constexpr int kBins = BINS;
    float m, scale;
    Weight weight;
    int bits;                   // of the largest mass

    // (a bin's log2(e) units in 2^-19, rounded down by 5 10^-6 of itself or more: bin_of is off by 2 10^-7 at most)
    static constexpr uint32_t kBinEdge = (uint32_t)(kUnits / BINS * kLog2eD * (1 << 19));
    MFL_INLINE static int edge(int bin) { return (int)(__umul24((uint32_t)bin, kBinEdge) >> 19); }
    MFL_INLINE double unit(int bin) const { return __builtin_ldexp(1.0, -bits - edge(bin)); }

    MFL_INLINE explicit Bins(int C)
    {
        const int wide = 32 - __builtin_clz(C);     // C < 2^wide
        bits = min(51, 62 - wide);
    }
    MFL_INLINE void set(float largest, const Filter &f)
    {
        m = largest;
        scale = (float)fmin(f.inv_t * (BINS / kUnits), 1e30);
        weight = {m, f.inv_t * kLog2eD};
    }
    // (the smaller one before the conversion: -inf has no integer)
    MFL_INLINE int bin_of(float x) const { return (int)fminf((m - x) * scale, (float)(BINS - 1)); }
    MFL_INLINE uint64_t mass(float x, int bin) const
    {
        // 2^52 + an integer below 2^52: the low bits of the sum are that integer
        const double v = weight.scaled(x, bits + edge(bin)) + 4503599627370496.0;
        return __builtin_bit_cast(uint64_t, v) & 0xfffffffffffffull;
    }
    // The lowest score of bins 0 .. b (they grow as the score falls); b = -1: none
    MFL_INLINE float lowest_of(int b) const
    {
        if (b < 0) return INFINITY;
        // hi is in, lo is not; 64 places between them at a time, one a lane
        long long lo = score_key(-INFINITY), hi = score_key(m);
        if (bin_of(-INFINITY) <= b) return -INFINITY;
#pragma unroll 1
        while (hi - lo > 1) {
            const long long step = (hi - lo + 63) >> 6, at = min(lo + ((threadIdx.x & 63) + 1) * step, hi);
            const int in = __ffsll((unsigned long long)__ballot(bin_of(key_score((int)at)) <= b)) - 1;
            hi = min(lo + (in + 1) * step, hi);
            lo += in * step;
        }
        return key_score((int)hi);
    }
};

template <typename T, int NT> struct BlockRow : Bins<4 * NT> {
    using Bins<4 * NT>::kBins;
    using Bins<4 * NT>::m;
    using Bins<4 * NT>::weight;
    using Bins<4 * NT>::bin_of;
    using Bins<4 * NT>::mass;
    using Bins<4 * NT>::lowest_of;
    using Bins<4 * NT>::unit;
    static constexpr int V = kVec<T>, step = 64 * V, waves = NT / 64;
    struct Shared {
        uint32_t counts[kBins];
        unsigned long long masses[kBins];
        unsigned long long key[kBinList], key_mass[kBinList];
        double runs[kRuns];
        unsigned long long more[kRuns];         // fixed point
        unsigned long long upart[NT / 64];
        double dpart[NT / 64];
        Reach reach;
        float fpart[NT / 64];
        unsigned listed, bin;
        unsigned long long low_key, any_key;
    };
    Shared &sh;
    const T *p;
    long long sc;
    int C;
    int tiles, per, count_runs; // 64 lanes' vectors of labels, tiles a run, runs

    MFL_INLINE BlockRow(Shared &sh, const T *p, long long sc, int C) : Bins<4 * NT>(C), sh(sh), p(p), sc(sc), C(C)
    {
        tiles = (C + step - 1) / step;
        per = (tiles + kRuns - 1) / kRuns;
        count_runs = (tiles + per - 1) / per;
    }
    // f(score, label) over the row
    template <typename F> MFL_INLINE void each(F f) const
    {
        if (sc == 1) {
            constexpr int U = 2;
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

    MFL_INLINE float largest()
    {
        float v = -INFINITY;
        each([&](float x, int) __attribute__((always_inline)) { v = max_or_nan(v, x); });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v = max_or_nan(v, __shfl_xor(v, o));
        if ((threadIdx.x & 63) == 0) sh.fpart[threadIdx.x >> 6] = v;
        __syncthreads();
        for (int w = 0; w < NT / 64; ++w) v = max_or_nan(v, sh.fpart[w]);
        return v;
    }

    // A lane's vector of a tile (behind the last label: -inf)
    MFL_INLINE void load_tile(float (&x)[V], int t) const
    {
        const int c = t * step + (threadIdx.x & 63) * V;
        if (sc == 1 && c + V <= C) {
            load_vec(p + c, x);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = c + i < C ? to_float(p[(c + i) * sc]) : -INFINITY;
        }
    }
    // sh.runs = sums of f(vector, its first label) over the runs.  A wave takes U runs at a time, to have U loads in flight.
    // f is called by whole waves.
    template <int U, typename F> MFL_INLINE void sum_runs(F f)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 1
        for (int e = wave; e < count_runs; e += U * waves) {
            double sum[U] = {};
#pragma unroll 1
            for (int t = 0; t < per; ++t) {
                float x[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u) load_tile(x[u], min((e + u * waves) * per + t, tiles - 1));
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = (e + u * waves) * per + t;
                    if (at < tiles) sum[u] += f(x[u], at * step + lane * V);
                }
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
#pragma unroll
                for (int u = 0; u < U; ++u) sum[u] += __shfl_xor(sum[u], o);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (lane == 0 && e + u * waves < count_runs) sh.runs[e + u * waves] = sum[u];
        }
    }

    // sh.runs = the runs' weights of at least min_p of scores from `sure` on, and, unless LIST, of scores from `open` on
    // whose key is at least cut; with LIST those labels between are listed
    template <bool LIST> MFL_INLINE void sweep(float sure, float open, uint64_t cut, double min_p)
    {
        sum_runs<4>([&](const float (&x)[V], int c) __attribute__((always_inline)) {
            uint32_t todo = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) todo |= x[i] >= open ? 1u << i : 0u;
            if (c + V > C) todo &= (1u << max(C - c, 0)) - 1;
            double sum = 0;
            // every lane its first, then its second: seldom more, where few are kept
#pragma unroll 1
            while (__any(todo != 0)) {
                const int i = __ffs(todo) - 1;
                float v = x[0];
#pragma unroll
                for (int j = 1; j < V; ++j) v = i == j ? x[j] : v;
                bool keep = todo != 0;
                todo &= todo - 1;
                if (keep && !(v >= sure)) {
                    const uint64_t key = rank_key(score_key(v), c + i);
                    keep = key >= cut;
                    if (LIST && keep) {
                        keep = false;
                        const unsigned at = atomicAdd(&sh.listed, 1u);
                        if (at < (unsigned)kBinList) sh.key[at] = key;
                    }
                }
                const double w = weight(v);
                sum += keep && w >= min_p ? w : 0.0;
            }
            return sum;
        });
        __syncthreads();
    }

    // How many labels of the mass `each` reach what is left
    MFL_INLINE unsigned long long share_of(double left, double one, unsigned long long each) const
    {
        unsigned long long n = (unsigned long long)fmin(fmax(1.0, __builtin_ceil(left / ((double)each * one))), (double)C);
        while (n > 1 && (double)((n - 1) * each) * one >= left) --n;
        while (n < (unsigned long long)C && (double)(n * each) * one < left) ++n;
        return n;
    }
    // The rank key of the n-th label of one score, in label order (of the last one, if there are fewer)
    MFL_INLINE uint64_t nth_of_score(float score, unsigned long long n)
    {
        // (two at a time: with four, the kernel's registers leave two waves a SIMD instead of three)
        sum_runs<2>([&](const float (&x)[V], int c) __attribute__((always_inline)) {
            double found = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) found += x[i] == score && c + i < C ? 1.0 : 0.0;
            return found;
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            double left = (double)n;
            int run = 0, label = -1;
            for (; run < count_runs - 1 && sh.runs[run] < left; ++run) left -= sh.runs[run];
            for (int t = run * per; t < min(tiles, (run + 1) * per); ++t) {
                float x[V];
                load_tile(x, t);
                const int c = t * step + lane * V;
                int own = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) own += x[i] == score && c + i < C;
                int upto = own;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int other = __shfl_up(upto, o);
                    if (lane >= o) upto += other;
                }
                const uint64_t past = __ballot(own > 0 && upto >= left), holds = __ballot(own > 0);
                if (holds) {
                    const int who = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)holds);
                    int at = upto - own, l = -1;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const bool here = x[i] == score && c + i < C && !(l >= 0 && at >= left);
                        at += here;
                        l = here ? c + i : l;
                    }
                    label = __shfl(l, who);
                }
                if (past) break;
                left -= __shfl(upto, 63);
            }
            if (lane == 0) sh.low_key = rank_key(score_key(score), label);
        }
        __syncthreads();
        return sh.low_key;
    }

    // The lowest rank key that top_k and top_p keep (0: all); sh.runs becomes the runs' kept weights
    MFL_INLINE uint64_t cut_of(const Filter &f)
    {
        const bool by_count = f.top_k < C, by_mass = f.top_p < 1;
        int bin = 0;
        float sure = -INFINITY, open = -INFINITY;
        uint64_t cut = 0;
        bool summed = false;
        if (by_count || by_mass) {
            for (int i = threadIdx.x; i < kBins; i += NT) sh.counts[i] = 0, sh.masses[i] = 0;
            __syncthreads();
            each([&](float x, int) __attribute__((always_inline)) {
                const int b = bin_of(x);
                if (by_count) atomicAdd(&sh.counts[b], 1u);
                if (by_mass) {
                    const uint64_t v = mass(x, b);
                    if (v) atomicAdd(&sh.masses[b], (unsigned long long)v);
                }
            });
            __syncthreads();
        }
        // first by number, then by mass among what is left
#pragma unroll 1
        for (int stage = by_count ? 0 : 1; stage < (by_mass ? 2 : 1); ++stage) {
            const bool count = stage == 0, final = stage == 1 || !by_mass;
            // the bin it falls into, and what the bins in front of it leave of the goal
            constexpr int each_bins = kBins / NT;
            const auto held = [&](int b) __attribute__((always_inline)) { return count ? (double)sh.counts[b] : (double)sh.masses[b] * unit(b); };
            if (threadIdx.x == 0) sh.reach.first = ~0u, sh.reach.last = 0, sh.listed = 0, sh.low_key = ~0ull;
            for (int i = threadIdx.x; i < kRuns; i += NT) sh.more[i] = 0;
            // (this thread's bins.  Made anew in each stage, or their steps are kept in registers throughout, which there are none for)
            int own = threadIdx.x * each_bins;
            asm volatile("" : "+v"(own));
            double mine = 0, all;
            for (int i = 0; i < each_bins; ++i) mine += held(own + i);
            const double front = block_front<double, NT>(mine, sh.dpart, all);
            // labels stay while what lies in front of them is below the goal
            const double goal = count ? (double)f.top_k : f.top_p * all;
            find_bin(each_bins, front, mine, goal, [&](int i) __attribute__((always_inline)) { return held(own + i); }, sh.reach);
            bin = sh.reach.bin;
            sure = lowest_of(bin - 1);
            open = lowest_of(bin);
            sweep<true>(sure, open, cut, f.min_p);
            const int n = sh.listed;
            const double one = count ? 1.0 : unit(bin);
            // (rounded, but never more than the bin holds)
            const double left = fmin(sh.reach.left, held(bin));
            if (n <= kBinList) {
                for (int i = threadIdx.x; i < (n + 7) / 8 * 8; i += NT) {
                    if (i >= n) sh.key[i] = 0;
                    sh.key_mass[i] = i >= n ? 0 : count ? 1 : mass(rank_score(sh.key[i]), bin);
                }
                __syncthreads();
                for (int i = threadIdx.x; i < n; i += NT) {
                    const uint64_t key = sh.key[i];
                    const unsigned long long above = held_above(sh.key, sh.key_mass, n, key);
                    // (a goal of nothing still keeps the first label)
                    if (above == 0 || (double)above * one < left) {
                        atomicMin(&sh.low_key, key);
                        // (sums of integers: in any order)
                        if (final && weight(rank_score(key)) >= f.min_p)
                            atomicAdd(&sh.more[rank_label(key) / (step * per)], (unsigned long long)mass(rank_score(key), bin));
                    }
                }
                __syncthreads();
                cut = sh.low_key;
                if (final) {
                    for (int i = threadIdx.x; i < count_runs; i += NT) sh.runs[i] += (double)sh.more[i] * unit(bin);
                    __syncthreads();
                    summed = true;
                }
            } else {
                // the largest key from which on the bin holds what is left of the goal, bit by bit where the bin's keys differ
                if (threadIdx.x == 0) sh.low_key = ~0ull, sh.any_key = 0;
                __syncthreads();
                unsigned long long every = ~0ull, any = 0;
                each([&](float x, int c) __attribute__((always_inline)) {
                    const uint64_t key = rank_key(score_key(x), c);
                    if (bin_of(x) != bin || key < cut) return;
                    every &= key;
                    any |= key;
                });
                atomicAnd(&sh.low_key, every);
                atomicOr(&sh.any_key, any);
                __syncthreads();
                every = sh.low_key;
                any = sh.any_key;
                uint64_t best = 0;
                const bool one_score = every >> 32 == any >> 32;
                if (one_score) best = nth_of_score(rank_score(any), share_of(left, one, count ? 1 : mass(rank_score(any), bin)));
#pragma unroll 1
                for (int b = one_score ? -1 : 63; b >= 0; --b) {
                    if (!(any >> b & 1)) continue;
                    const uint64_t at = best | 1ull << b, from = at > cut ? at : cut;
                    if (every >> b & 1) {
                        best = at;
                        continue;
                    }
                    unsigned long long sum = 0;
                    each([&](float x, int c) __attribute__((always_inline)) {
                        if (bin_of(x) == bin && rank_key(score_key(x), c) >= from) sum += count ? 1 : mass(x, bin);
                    });
                    sum = block_sum<unsigned long long, NT>(sum, sh.upart);
                    if (sum && (double)sum * one >= left) best = at;
                }
                cut = best > cut ? best : cut;
            }
            if (!final) {
                // what is left of the bin, and nothing behind it
                unsigned long long kept = 0;
                each([&](float x, int c) __attribute__((always_inline)) {
                    if (bin_of(x) == bin && rank_key(score_key(x), c) >= cut) kept += mass(x, bin);
                });
                kept = block_sum<unsigned long long, NT>(kept, sh.upart);
                for (int i = threadIdx.x; i < kBins; i += NT)
                    if (i >= bin) sh.masses[i] = i == bin ? kept : 0;
                __syncthreads();
            }
        }
        if (!summed) sweep<false>(sure, open, cut, f.min_p);
        return cut;
    }

    // Step 4: sh.runs holds the runs' kept weights, cut is the lowest rank key that stays
    MFL_INLINE void draw(uint64_t cut, double min_p, float u, unsigned r, const Out &out)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, runs = count_runs;
        const float cut_score = cut ? rank_score(cut) : -INFINITY;
        // a vector's kept weights
        auto kept = [&](const float (&x)[V], int c, double (&w)[V]) {
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
            float x[V];
            load_tile(x, t);
            double w[V];
            if (!kept(x, t * step + lane * V, w)) continue;
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
sample_blocks_kernel(Rows in, Settings set, int done, const float *__restrict__ uniform, Out out)
{
    __shared__ typename BlockRow<T, NT>::Shared sh;
    const unsigned r = blockIdx.x;
    const RowOf<T> at(in, r);
    const Filter f = filter_of(set, at.n, in.C);
    if (f.top_k <= done) return;            // (a list had it)
    BlockRow<T, NT> row(sh, at.p, in.sc, in.C);
    const float m = row.largest();
    if (!(fabsf(m) < INFINITY)) {
        if (threadIdx.x == 0) put(out, r, -1, -INFINITY);
        return;
    }
    row.set(m, f);
    const uint64_t cut = row.cut_of(f);
    row.draw(cut, f.min_p, uniform[r], r, out);
}

// ---- rows of many labels without top_k and top_p: cut into parts
//
// A workgroup holds a part's scores in registers: the part's largest score, and the weights next to it (with min_p, in a
// second launch, next to the row's largest), summed.  One workgroup per row then scales the sums, finds the part that the
// draw falls into, and reads that part again.

constexpr int kPlainThreads = 256;
constexpr int kPlainPart = 8192;            // labels of a part at most
struct Part {
    double sum;
    float top;
};
template <typename T> constexpr int kPlainVecs = kPlainPart / (kPlainThreads * kVec<T>);

// A thread's vectors of a part: labels begin + (u * 256 + thread) * V
template <typename T> __device__ inline void load_part(float (&x)[kPlainVecs<T>][kVec<T>], const T *p, long long sc, int begin, int end)
{
    constexpr int V = kVec<T>, U = kPlainVecs<T>;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = begin + (u * kPlainThreads + (int)threadIdx.x) * V;
        if (sc == 1 && c + V <= end) {
            load_vec(p + c, x[u]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[u][i] = c + i < end ? to_float(p[(c + i) * sc]) : -INFINITY;
        }
    }
}
__device__ inline float block_largest(float v, float *part)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max_or_nan(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kPlainThreads / 64; ++w) v = max_or_nan(v, part[w]);
    return v;
}
// The row's largest score
__device__ inline float largest_of_parts(const Part *parts, int n, float *part)
{
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n; i += kPlainThreads) m = max_or_nan(m, parts[i].top);
    return block_largest(m, part);
}

template <typename T, bool AGAIN>
__global__ void __launch_bounds__(kPlainThreads)
plain_parts_kernel(Rows in, Settings set, int parts, int size, Part *__restrict__ ws)
{
    __shared__ float fpart[kPlainThreads / 64];
    __shared__ double dpart[kPlainThreads / 64];
    constexpr int V = kVec<T>, U = kPlainVecs<T>;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    const int begin = part * size, end = min(in.C, begin + size);
    float x[U][V];
    load_part(x, row.p, in.sc, begin, end);
    float m;
    if (AGAIN) {
        m = largest_of_parts(ws + (size_t)r * parts, parts, fpart);
    } else {
        m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) m = largest_of(x[u], m);
        m = block_largest(m, fpart);
    }
    double sum = 0;
    if (fabsf(m) < INFINITY) {
        const Weight weight = {m, f.inv_t * kLog2eD};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (begin + u * kPlainThreads * V >= end) break;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double w = weight(x[u][i]);
                sum += !AGAIN || w >= f.min_p ? w : 0.0;
            }
        }
    }
    sum = block_sum<double, kPlainThreads>(sum, dpart);
    if (threadIdx.x == 0) {
        ws[blockIdx.x].sum = sum;
        if (!AGAIN) ws[blockIdx.x].top = m;
    }
}

// Of n entries, the first whose running sum from front0 on exceeds the target, or the last that holds something; *before: the
// sum in front of it.  Unless given, all = the sum of the entries and target = its share u.
template <typename F>
__device__ inline int find_entry(int n, F value, double front0, float u, double &target, double &all, bool given, double *dpart, unsigned *first,
                                 unsigned *last, double *before)
{
    const int each = (n + kPlainThreads - 1) / kPlainThreads, from = min(n, (int)threadIdx.x * each), to = min(n, from + each);
    double mine = 0;
    int holds = -1;
    for (int i = from; i < to; ++i) {
        const double v = value(i);
        mine += v;
        if (v > 0) holds = i;
    }
    double sum, front = front0 + block_front<double, kPlainThreads>(mine, dpart, sum);
    if (!given) {
        all = sum;
        target = draw_of(u) * all;
    }
    if (threadIdx.x == 0) *first = ~0u, *last = 0;
    __syncthreads();
    if (holds >= 0) atomicMax(last, (unsigned)holds);
    if (mine > 0 && front + mine > target) {
        double run = front;
        for (int i = from; i < to; ++i) {
            run += value(i);
            if (run > target) {
                atomicMin(first, (unsigned)i);
                break;
            }
        }
    }
    __syncthreads();
    const int at = *first != ~0u ? (int)*first : (int)*last;
    if (at >= from && at < to) {
        for (int i = from; i < at; ++i) front += value(i);
        *before = front;
    }
    __syncthreads();
    return at;
}
// The label within the part that the draw falls into; kept(score, label) is what a label weighs
template <typename T, typename F>
__device__ inline void pick_in_part(const T *p, long long sc, int begin, int end, F kept, double front, double target, double total, double *sums,
                                    double *dpart, unsigned *first, unsigned *last, double *before, unsigned r, const Out &out)
{
    constexpr int V = kVec<T>, U = kPlainVecs<T>;
    float x[U][V];
    load_part(x, p, sc, begin, end);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = begin + (u * kPlainThreads + (int)threadIdx.x) * V;
        double s = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) s += kept(x[u][i], c + i);
        sums[u * kPlainThreads + threadIdx.x] = s;
    }
    __syncthreads();
    const int vec = find_entry(U * kPlainThreads, [&](int i) { return sums[i]; }, front, 0.f, target, total, true, dpart, first, last, before);
    // (its scores are still in the registers of the thread that summed it)
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (vec != u * kPlainThreads + (int)threadIdx.x) continue;
        double run = *before, got = 0;
        int label = -1;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double w = kept(x[u][i], begin + vec * V + i);
            const bool open = w > 0 && !(label >= 0 && run > target);
            run += open ? w : 0.0;
            label = open ? begin + vec * V + i : label;
            got = open ? w : got;
        }
        put(out, r, label, log(got / total));
    }
}

template <typename T, bool AGAIN>
__global__ void __launch_bounds__(kPlainThreads)
plain_pick_kernel(Rows in, Settings set, int parts, int size, const Part *__restrict__ ws, const float *__restrict__ uniform, Out out)
{
    __shared__ float fpart[kPlainThreads / 64];
    __shared__ double dpart[kPlainThreads / 64], sums[kPlainVecs<T> * kPlainThreads], before;
    __shared__ unsigned first, last;
    const unsigned r = blockIdx.x;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    ws += (size_t)r * parts;
    const float m = largest_of_parts(ws, parts, fpart);
    if (!(fabsf(m) < INFINITY)) {
        if (threadIdx.x == 0) put(out, r, -1, -INFINITY);
        return;
    }
    const Weight weight = {m, f.inv_t * kLog2eD};
    double target = 0, total = 0;
    const int part = find_entry(parts, [&](int i) { return AGAIN ? ws[i].sum : ws[i].sum * weight(ws[i].top); }, 0.0, uniform[r], target, total, false,
                                dpart, &first, &last, &before);
    const double front = before;
    __syncthreads();
    auto kept = [&](float v, int) {
        const double w = weight(v);
        return w >= f.min_p ? w : 0.0;
    };
    pick_in_part<T>(row.p, in.sc, part * size, min(in.C, part * size + size), kept, front, target, total, sums, dpart, &first, &last, &before, r, out);
}

// ---- few rows of many labels that top_p cuts: the workgroup's steps, spread over the card
//
// (1 x 128000 bf16: 47 us against 118 by one workgroup, 64 rows 84 against 124; at 256 rows, one for each CU, 183 against 133,
// so from kSplitRows on a row gets its workgroup.)
//
//   1  the parts' largest scores               2  the histogram: a part's in LDS, then added to the row's (integers)
//   3  every workgroup finds the row's bin for itself; its part's sure weights summed, the bin's labels listed
//   4  one workgroup per row: the cut within the list, the part, the label.  (A list that overflowed, or a top_k of the row's
//      own: all of the workgroup's steps.)

constexpr int kSplitBins = 4096;
constexpr int kSplitParts = 512;
constexpr unsigned kSplitRows = 128;
struct SplitRow {
    unsigned long long masses[kSplitBins], keys[kBinList];
    double left;                // of the goal, for the bin that the cut falls into
    int bin;
    unsigned listed;
};
struct SplitSpace {
    SplitRow *rows;
    Part *parts;
};

template <typename T>
__global__ void __launch_bounds__(kPlainThreads)
split_largest_kernel(Rows in, int parts, int size, SplitSpace ws)
{
    __shared__ float fpart[kPlainThreads / 64];
    constexpr int V = kVec<T>, U = kPlainVecs<T>;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const RowOf<T> row(in, r);
    float x[U][V], m = -INFINITY;
    load_part(x, row.p, in.sc, part * size, min(in.C, (int)part * size + size));
    for (int b = part * kPlainThreads + threadIdx.x; b < kSplitBins; b += parts * kPlainThreads) ws.rows[r].masses[b] = 0;
    if (part == 0 && threadIdx.x == 0) ws.rows[r].listed = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) m = largest_of(x[u], m);
    m = block_largest(m, fpart);
    if (threadIdx.x == 0) ws.parts[blockIdx.x].top = m;
}

template <typename T>
__global__ void __launch_bounds__(kPlainThreads)
split_histogram_kernel(Rows in, Settings set, int parts, int size, SplitSpace ws)
{
    __shared__ unsigned long long masses[kSplitBins];
    __shared__ float fpart[kPlainThreads / 64];
    constexpr int V = kVec<T>, U = kPlainVecs<T>;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    if (f.top_k < in.C || f.top_p >= 1) return;
    const int begin = part * size, end = min(in.C, begin + size);
    float x[U][V];
    load_part(x, row.p, in.sc, begin, end);
    const float m = largest_of_parts(ws.parts + (size_t)r * parts, parts, fpart);
    if (!(fabsf(m) < INFINITY)) return;
    Bins<kSplitBins> bins(in.C);
    bins.set(m, f);
    for (int b = threadIdx.x; b < kSplitBins; b += kPlainThreads) masses[b] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = begin + (u * kPlainThreads + (int)threadIdx.x) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int b = bins.bin_of(x[u][i]);
            const uint64_t v = c + i < end ? bins.mass(x[u][i], b) : 0;
            if (v) atomicAdd(&masses[b], (unsigned long long)v);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < kSplitBins; b += kPlainThreads)
        if (masses[b]) atomicAdd(&ws.rows[r].masses[b], masses[b]);
}

template <typename T>
__global__ void __launch_bounds__(kPlainThreads)
split_sweep_kernel(Rows in, Settings set, int parts, int size, SplitSpace ws)
{
    __shared__ float fpart[kPlainThreads / 64];
    __shared__ double dpart[kPlainThreads / 64];
    __shared__ Reach reach;
    constexpr int V = kVec<T>, U = kPlainVecs<T>, each_bins = kSplitBins / kPlainThreads;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const RowOf<T> row(in, r);
    const Filter f = filter_of(set, row.n, in.C);
    if (f.top_k < in.C) return;
    const int begin = part * size, end = min(in.C, begin + size);
    float x[U][V];
    load_part(x, row.p, in.sc, begin, end);
    SplitRow &state = ws.rows[r];
    const float m = largest_of_parts(ws.parts + (size_t)r * parts, parts, fpart);
    if (!(fabsf(m) < INFINITY)) return;
    Bins<kSplitBins> bins(in.C);
    bins.set(m, f);
    float sure = -INFINITY, open = -INFINITY;
    if (f.top_p < 1) {
        if (threadIdx.x == 0) reach.first = ~0u, reach.last = 0;
        const auto held = [&](int i) {
            const int b = threadIdx.x * each_bins + i;
            return (double)state.masses[b] * bins.unit(b);
        };
        double mine = 0, all;
        for (int i = 0; i < each_bins; ++i) mine += held(i);
        const double front = block_front<double, kPlainThreads>(mine, dpart, all);
        find_bin(each_bins, front, mine, f.top_p * all, held, reach);        // (the one thread reads its bins again)
        sure = bins.lowest_of(reach.bin - 1);
        open = bins.lowest_of(reach.bin);
        if (part == 0 && threadIdx.x == 0) state.bin = reach.bin, state.left = reach.left;
    }
    double sum = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = begin + (u * kPlainThreads + (int)threadIdx.x) * V;
        uint32_t todo = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) todo |= x[u][i] >= open && c + i < end ? 1u << i : 0u;
#pragma unroll 1
        while (__any(todo != 0)) {
            const int i = __ffs(todo) - 1;
            float v = x[u][0];
#pragma unroll
            for (int j = 1; j < V; ++j) v = i == j ? x[u][j] : v;
            const bool keep = todo != 0 && v >= sure;
            if (todo != 0 && !keep) {
                const unsigned at = atomicAdd(&state.listed, 1u);
                if (at < (unsigned)kBinList) state.keys[at] = rank_key(score_key(v), c + i);
            }
            todo &= todo - 1;
            const double w = bins.weight(v);
            sum += keep && w >= f.min_p ? w : 0.0;
        }
    }
    sum = block_sum<double, kPlainThreads>(sum, dpart);
    if (threadIdx.x == 0) ws.parts[blockIdx.x].sum = sum;
}

template <typename T>
__global__ void __launch_bounds__(kPlainThreads)
split_pick_kernel(Rows in, Settings set, int done, int parts, int size, SplitSpace ws, const float *__restrict__ uniform, Out out)
{
    constexpr int U = kPlainVecs<T>, NT = kPlainThreads;
    __shared__ typename BlockRow<T, NT>::Shared sh;
    __shared__ unsigned long long more[kSplitParts];
    __shared__ double sums[U * NT], before;
    __shared__ unsigned first, last;
    const unsigned r = blockIdx.x;
    const RowOf<T> at(in, r);
    const Filter f = filter_of(set, at.n, in.C);
    if (f.top_k <= done) return;            // (a list had it)
    const Part *part_of = ws.parts + (size_t)r * parts;
    const SplitRow &state = ws.rows[r];
    const float m = largest_of_parts(part_of, parts, sh.fpart);
    if (!(fabsf(m) < INFINITY)) {
        if (threadIdx.x == 0) put(out, r, -1, -INFINITY);
        return;
    }
    BlockRow<T, NT> row(sh, at.p, in.sc, in.C);
    row.set(m, f);
    const bool ranked = f.top_p < 1;
    const unsigned n = f.top_k < in.C ? ~0u : ranked ? state.listed : 0;
    if (n > (unsigned)kBinList) {
        const uint64_t cut = row.cut_of(f);
        row.draw(cut, f.min_p, uniform[r], r, out);
        return;
    }
    // the cut within the list
    uint64_t cut = 0;
    Bins<kSplitBins> bins(in.C);
    bins.set(m, f);
    const int bin = ranked ? state.bin : 0;
    for (int i = threadIdx.x; i < parts; i += NT) more[i] = 0;
    if (ranked) {
        if (threadIdx.x == 0) sh.low_key = ~0ull;
        for (unsigned i = threadIdx.x; i < (n + 7) / 8 * 8; i += NT) {
            sh.key[i] = i < n ? state.keys[i] : 0;
            sh.key_mass[i] = i < n ? bins.mass(rank_score(sh.key[i]), bin) : 0;
        }
        __syncthreads();
        const double left = state.left, one = bins.unit(bin);
        for (unsigned i = threadIdx.x; i < n; i += NT) {
            const uint64_t key = sh.key[i];
            const unsigned long long above = held_above(sh.key, sh.key_mass, n, key);
            if (above == 0 || (double)above * one < left) {
                atomicMin(&sh.low_key, key);
                if (row.weight(rank_score(key)) >= f.min_p) atomicAdd(&more[rank_label(key) / size], sh.key_mass[i]);
            }
        }
    }
    __syncthreads();
    if (ranked) cut = sh.low_key;
    const float cut_score = cut ? rank_score(cut) : -INFINITY;
    auto kept = [&](float x, int c) {
        if (!(x >= cut_score) || rank_key(score_key(x), c) < cut) return 0.0;
        const double w = row.weight(x);
        return w >= f.min_p ? w : 0.0;
    };
    double target = 0, total = 0;
    const int part = find_entry(parts, [&](int i) { return part_of[i].sum + (double)more[i] * bins.unit(bin); }, 0.0, uniform[r], target, total,
                                false, sh.dpart, &first, &last, &before);
    const double front = before;
    __syncthreads();
    pick_in_part<T>(at.p, in.sc, part * size, min(in.C, part * size + size), kept, front, target, total, sums, sh.dpart, &first, &last, &before, r, out);
}

int plain_part_labels(unsigned rows, int C)
{
    // a quarter of the full size where that leaves the card short of workgroups
    return (unsigned long long)rows * ((C + kPlainPart - 1) / kPlainPart) >= 1024 ? kPlainPart : kPlainPart / 4;
}
int plain_parts(unsigned rows, int C) { return (int)(((long long)C + plain_part_labels(rows, C) - 1) / plain_part_labels(rows, C)); }

// top_k for all rows, and short enough for a list (temperature 0: the best one)
int list_length(const Settings &set)
{
    if (set.top_k_n) return 0;
    if (!set.t_n && set.t == 0) return 1;
    return set.top_k >= 1 && set.top_k <= MFL_MAX_TOP_LABELS ? set.top_k : 0;
}

constexpr int kShortRow = 4096;             // a workgroup of 256 up to here, of 1024 above

enum Way { LONE, LANES, LIST_LANES, ANY_LANES, PLAIN, WAVES, SPLIT, BLOCKS };
struct Plan {
    Way way;
    int k;                      // length of the list, 0: none
    bool two;                   // WAVES, then SPLIT or BLOCKS for the rows whose own top_k is not that short
    bool split;
    size_t bytes;
};
Plan plan_of(const Rows &in, const Settings &set)
{
    const bool no_k = !set.top_k_n && (set.top_k == 0 || set.top_k >= in.C), no_p = !set.top_p_n && set.top_p == 1;
    const bool plain = no_k && no_p && !set.t_n && set.t > 0 && !set.min_p_n;
    const int k = list_length(set) < in.C ? list_length(set) : 0;
    const auto keys = [&](int k) {
        const int parts = row_per_wave(in.rows, in.C) ? 1 : top_parts(in.rows, in.C);
        return parts > 1 ? (size_t)in.rows * parts * part_keys(k) * sizeof(uint64_t) : 0;
    };
    // lanes: short rows, and planes of many rows.  Lanes / rows of neighbouring labels, fp32, without filters, top_k 8 and top_p,
    // us: 4096 x 64 19 / 40, 14 / 15, 52 / 73; 4096 x 256 42 / 35, 35 / 22, 309 / 72; 16384 x 256 42 / 123, 34 / 64, 310 / 255.
    // (Many rows of 256 and more labels would do better with lanes: 131072 x 256 83 / 959, 79 / 421, 487 / 1991.)
    if (!(in.sc == 1 && in.C >= 256) && !(in.C >= 1024 && in.rows <= 4096)) {
        const int list = k ? k : no_k && in.C <= 32 ? in.C : 0;
        if (plain) return {in.C <= kLoneBlock ? LONE : LANES, 0, false, false, 0};
        if (list && list <= 32 && in.C <= kBestLabels) return {LIST_LANES, list, false, false, 0};
        // (few rows of many labels to rank: a workgroup each)
        if (in.C <= kBestLabels && (in.rows > 2048 || in.C <= 64)) return {ANY_LANES, 0, false, false, 0};
    }
    if (plain && in.C > 4096) return {PLAIN, 0, false, false, (size_t)in.rows * plain_parts(in.rows, in.C) * sizeof(Part)};
    if (k) return {WAVES, k, false, false, keys(k)};
    // (a top_k for all rows that is too long for a list is the workgroup's to count)
    const bool split = in.C > 8192 && in.rows <= kSplitRows && (no_k || set.top_k_n) && plain_parts(in.rows, in.C) <= kSplitParts;
    const size_t space = split ? (size_t)in.rows * (sizeof(SplitRow) + plain_parts(in.rows, in.C) * sizeof(Part)) : 0;
    if (set.top_k_n && in.C > MFL_MAX_TOP_LABELS) return {WAVES, MFL_MAX_TOP_LABELS, true, split, space + keys(MFL_MAX_TOP_LABELS)};
    return {split ? SPLIT : BLOCKS, 0, false, split, space};
}

template <typename T>
int run(const Rows &in, const Settings &set, const float *uniform, const Out &out, void *workspace, hipStream_t st)
{
    const Plan plan = plan_of(in, set);
    const int k = plan.k;
    // the threads that a row takes in the largest of the launches
    unsigned threads_a_row = 1;
    if (plan.way == WAVES) threads_a_row = row_per_wave(in.rows, in.C) ? 64 : kWaveTopThreads * top_parts(in.rows, in.C);
    if (plan.way == PLAIN || plan.split) threads_a_row = max(threads_a_row, (unsigned)(kPlainThreads * plain_parts(in.rows, in.C)));
    else if (plan.way == BLOCKS || plan.two) threads_a_row = max(threads_a_row, in.C <= kShortRow ? 256u : 1024u);
    if (!launchable(in.rows, threads_a_row)) return MFL_ERR_TOO_LARGE;
    const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
#define MFL_LANES(...) hipLaunchKernelGGL(__VA_ARGS__, grid, block, 0, st, in, set, uniform, out)
    switch (plan.way) {
    case LONE:
        if (in.C <= 8) MFL_LANES((plain_lone_kernel<T, 8>));
        else if (in.C <= 16) MFL_LANES((plain_lone_kernel<T, 16>));
        else MFL_LANES((plain_lone_kernel<T, kLoneBlock>));
        break;
    case LANES: MFL_LANES((plain_lanes_kernel<T>)); break;
    case LIST_LANES:
        if (in.C <= 32 && k > 4) {
            if (in.C <= 8) MFL_LANES((list_lanes_kernel<T, 8, true>));
            else if (in.C <= 16) MFL_LANES((list_lanes_kernel<T, 16, true>));
            else if (in.C <= 24) MFL_LANES((list_lanes_kernel<T, 24, true>));
            else MFL_LANES((list_lanes_kernel<T, 32, true>));
        } else if (k <= 1) MFL_LANES((list_lanes_kernel<T, 1, false>));
        else if (k <= 4) MFL_LANES((list_lanes_kernel<T, 4, false>));
        else if (k <= 8) MFL_LANES((list_lanes_kernel<T, 8, false>));
        else if (k <= 16) MFL_LANES((list_lanes_kernel<T, 16, false>));
        else MFL_LANES((list_lanes_kernel<T, 32, false>));
        break;
    case ANY_LANES: MFL_LANES((any_lanes_kernel<T>)); break;
#undef MFL_LANES
    case PLAIN: {
        const int parts = plain_parts(in.rows, in.C), size = plain_part_labels(in.rows, in.C);
        Part *ws = (Part *)workspace;
        const dim3 all(in.rows * parts), one(in.rows), threads(kPlainThreads);
        hipLaunchKernelGGL((plain_parts_kernel<T, false>), all, threads, 0, st, in, set, parts, size, ws);
        if (set.min_p > 0) {
            hipLaunchKernelGGL((plain_parts_kernel<T, true>), all, threads, 0, st, in, set, parts, size, ws);
            hipLaunchKernelGGL((plain_pick_kernel<T, true>), one, threads, 0, st, in, set, parts, size, ws, uniform, out);
        } else {
            hipLaunchKernelGGL((plain_pick_kernel<T, false>), one, threads, 0, st, in, set, parts, size, ws, uniform, out);
        }
        break;
    }
    case WAVES: {
        const size_t space = plan.split ? (size_t)in.rows * (sizeof(SplitRow) + plain_parts(in.rows, in.C) * sizeof(Part)) : 0;
        if (row_per_wave(in.rows, in.C)) {
            const unsigned per = kWaveTopThreads / 64;
            hipLaunchKernelGGL(list_waves_kernel<T>, dim3((in.rows + per - 1) / per), dim3(kWaveTopThreads), 0, st, in, set, k, uniform, out);
        } else {
            const int parts = top_parts(in.rows, in.C);
            uint64_t *keys = (uint64_t *)((char *)workspace + space);
            hipLaunchKernelGGL(list_parts_kernel<T>, dim3(in.rows * parts), dim3(kWaveTopThreads), 0, st, in, set, k, parts, uniform, keys, out);
            if (parts > 1)
                hipLaunchKernelGGL(list_join_kernel, dim3(in.rows), dim3(kWaveTopThreads), 0, st, in, set, k, parts, uniform, keys, out);
        }
        if (!plan.two) break;
        [[fallthrough]];
    }
    case SPLIT:
    case BLOCKS:
        if (plan.split) {
            const int parts = plain_parts(in.rows, in.C), size = plain_part_labels(in.rows, in.C);
            const SplitSpace ws = {(SplitRow *)workspace, (Part *)((SplitRow *)workspace + in.rows)};
            const dim3 all(in.rows * parts), one(in.rows), threads(kPlainThreads);
            hipLaunchKernelGGL(split_largest_kernel<T>, all, threads, 0, st, in, parts, size, ws);
            hipLaunchKernelGGL(split_histogram_kernel<T>, all, threads, 0, st, in, set, parts, size, ws);
            hipLaunchKernelGGL(split_sweep_kernel<T>, all, threads, 0, st, in, set, parts, size, ws);
            hipLaunchKernelGGL(split_pick_kernel<T>, one, threads, 0, st, in, set, k, parts, size, ws, uniform, out);
            break;
        }
        if (in.C <= kShortRow) hipLaunchKernelGGL((sample_blocks_kernel<T, 256>), dim3(in.rows), dim3(256), 0, st, in, set, k, uniform, out);
        else hipLaunchKernelGGL((sample_blocks_kernel<T, 1024>), dim3(in.rows), dim3(1024), 0, st, in, set, k, uniform, out);
    }
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

// (for any strides and settings: the most that a call of this size takes)
size_t mfl_sample_labels_workspace_bytes(int N, int C, int S, int dtype)
{
    Rows in;
    if (make_rows(in, "", dtype, N, C, S, 0, 1, 0)) return 0;
    size_t most = 0;
    // no filters; a short list; top_p; a top_k of every row's own
    const int some = 0;
    const Settings sets[4] = {{1.0, 1.0, 0.0, 0, nullptr, nullptr, nullptr, nullptr}, {1.0, 1.0, 0.0, MFL_MAX_TOP_LABELS, nullptr, nullptr, nullptr, nullptr},
                              {1.0, 0.5, 0.0, 0, nullptr, nullptr, nullptr, nullptr}, {1.0, 1.0, 0.0, 0, nullptr, nullptr, nullptr, &some}};
    for (int i = 0; i < 8; ++i) {
        in.sc = i & 1 ? 1 : 2;
        const size_t n = plan_of(in, sets[i >> 1]).bytes;
        most = n > most ? n : most;
    }
    return most;
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
    const Settings set = {temperature, top_p, min_p, top_k, temperature_n, top_p_n, min_p_n, top_k_n};
    const size_t need = plan_of(in, set).bytes;
    if (need && (!workspace || workspace_bytes < need)) return MFL_ERR_WORKSPACE;
    const Out out = {labels, label_bytes, logprob};
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run<float>(in, set, uniform, out, workspace, st);
    case MFL_BF16: return run<bf16_t>(in, set, uniform, out, workspace, st);
    default: return run<f16_t>(in, set, uniform, out, workspace, st);
    }
}

}  // extern "C"
