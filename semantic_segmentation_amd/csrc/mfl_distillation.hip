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
//   stats[0] = m,  stats[1] = Z - m / T,  stats[2] = m_O, the largest score in O,  stats[3] = Z_O - m_O / T,  stats[4] = Z_O - Z
// without anything in O: m_O and Z_O - Z are -inf, Z_O - m_O / T is 0; a row without loss: the same of m and Z - m / T too; a
// row with a NaN score: all NaN.  Up to kLoneBlock labels nothing is kept, the backward pass finds them anew.
//
// Both passes are bound by memory: the forward pass reads the scores, the backward pass reads them again and writes the
// gradient.  Measured on MI355X, forward / backward: 8 x 21 x 512 x 512 fp32, k = 4 with rest 64 / 98 us (4.1 / 4.4 TB/s);
// 2 x 19 x 1024 x 2048 bf16, k = 3 73 / 111 us (3.5 / 3.7 TB/s: two bytes a lane and the vector unit's share); 2048 x 128000
// bf16, k = 64 with rest 103 / 211 us (5.1 / 5.0 TB/s: the backward pass starts with the rows that the forward pass read last,
// part of which is still in the last-level cache, and streams its gradient past it; rows from the first on 316, cached gradient
// 377 us for both).  16 x 32000: 21 us in three launches, of which the bytes take one, in a call that takes the host about 105
// with autograd's round trip.  Channels-last maps are the lanes' as well, and their stores of single scores C apart, streamed
// past the caches, do badly: 8 x 21 x 512 x 512 73 / 1459 us in fp32, 55 / 719 in bf16.
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

// The teacher's distribution of a row.  log p_j = (t_j - m) / T - l, log p_rest = rest - m / T - l
struct Target {
    float m, l, log_p_rest, p_rest;
    float s;                    // l = log(1 + s)
    bool any;                   // it holds something
};
// sum: the entries with a label of the row (named: there are some); rest: -inf for none
__device__ inline Target target_of(const Teacher &t, Excess sum, bool named, float rest)
{
    Target g;
    if (sum.m == -INFINITY && rest != -INFINITY) sum.m = rest * t.t;
    const float above = fmaf(-sum.m, t.inv_t, rest);       // the rest next to the largest entry
    g.s = rest == -INFINITY ? sum.s : sum.s + __builtin_amdgcn_exp2f(above * kLog2e);
    g.l = rest == -INFINITY || above <= 0 ? log_1p(g.s) : above + log_1p((1.f + sum.s) * __builtin_amdgcn_exp2f(-above * kLog2e));
    g.m = sum.m;
    g.any = named && !(sum.m == -INFINITY && sum.s == -1.f);
    const float ratio = (1.f + sum.s) * __builtin_amdgcn_exp2f(-above * kLog2e);        // the record next to the rest
    g.log_p_rest = rest == -INFINITY ? -INFINITY : ratio == INFINITY ? above - g.l : -log_1p(ratio);
    if (g.s != g.s) g.log_p_rest = NAN;         // (a NaN among the values leaves no share a number, an empty rest's neither)
    g.p_rest = __builtin_amdgcn_exp2f(g.log_p_rest * kLog2e);
    return g;
}
__device__ inline float log_share(const Teacher &t, const Target &g, float value) { return (value - g.m) * t.inv_t - g.l; }

// p T d; nothing where p is 0.  (A share that fp32 does not hold still counts next to a difference near the largest number, but
// not next to an infinite one.)
__device__ inline float share_term(float log_p, float t, float d)
{
    const float e = log_p * kLog2e;
    const bool tiny = e < -100.f && fabsf(d) < INFINITY;
    const float p = __builtin_amdgcn_exp2f(tiny ? e + 60.f : e);
    return p == 0.f ? 0.f : p * t * (tiny ? d * 0x1p-60f : d);
}
// T^2 p (log p - log q) of an entry.  log p - log q = ((t - m_p) - (score - m_q)) / T -
// log((1 + s_p) / (1 + s_q)), in this order, since close to the teacher the two logarithms agree in most of their digits, and
// times T, since a score of the type's lowest number over T may be no fp32 number where T times it is one
__device__ inline float entry_term(const Teacher &t, const Target &g, float log_sums, float m, float value, float x)
{
    return share_term(log_share(t, g, value), t.t, fmaf(-log_sums, t.t, (value - g.m) - (x - m)));
}

struct Stats {
    float m, z, mo, zo, log_q_rest;     // as above
    float s;                            // z = log(1 + s); not kept
};
constexpr Stats kNoStats = {-INFINITY, 0.f, -INFINITY, 0.f, -INFINITY, 0.f};
// ... of the rest (without it log p_rest is -inf)
__device__ inline float rest_term(const Teacher &t, const Target &g, const Stats &a)
{
    const float d = a.log_q_rest == -INFINITY && a.mo != -INFINITY ? fmaf(g.log_p_rest - (a.zo - a.z), t.t, a.m - a.mo) : (g.log_p_rest - a.log_q_rest) * t.t;
    return share_term(g.log_p_rest, t.t, d);
}
// log((1 + s_p) / (1 + s_q))
__device__ inline float log_sums(const Target &g, const Stats &a)
{
    const float d = (g.s - a.s) / (1.f + a.s);
    return fabsf(d) < 0.5f ? log_1p(d) : g.l - a.z;
}
// top: the record's labels, each once; out: all others
__device__ inline Stats stats_of(Excess top, LogSum out, const Teacher &t)
{
    const Excess all = join(top, Excess{out.m, out.s - 1.f}, t.c2);
    if (all.m == -INFINITY && all.s == -1.f) return kNoStats;
    // (a NaN score is in the sum, whatever the largest score came to without it)
    if (all.s != all.s) return {NAN, NAN, NAN, NAN, NAN, NAN};
    Stats a = {all.m, log_1p(all.s), -INFINITY, 0.f, -INFINITY, all.s};
    if (out.m == -INFINITY && out.s == 0.f) return a;
    a.mo = out.m;
    a.zo = logf(out.s);
    const float ratio = (1.f + top.s) * __builtin_amdgcn_exp2f((top.m - out.m) * t.c2) / out.s;
    a.log_q_rest = ratio == INFINITY ? (a.mo - a.m) * t.inv_t + (a.zo - a.z) : -log_1p(ratio);
    return a;
}
__device__ inline void put(float *loss, float *stats, size_t rows, unsigned r, float l, const Stats &a)
{
    loss[r] = l;
    if (!stats) return;
    stats[r] = a.m;
    stats[rows + r] = a.z;
    stats[2 * rows + r] = a.mo;
    stats[3 * rows + r] = a.zo;
    stats[4 * rows + r] = a.log_q_rest;
}
__device__ inline Stats load_stats(const float *stats, size_t rows, unsigned r)
{
    return {stats[r], stats[rows + r], stats[2 * rows + r], stats[3 * rows + r], stats[4 * rows + r], 0.f};
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
            // q_rest - p_rest = p_rest (exp(d) - 1), exp(d) - 1 from the rounded exponential and its own logarithm (Kahan)
            const float d = a.log_q_rest - g.log_p_rest, e = __builtin_amdgcn_exp2f(d * kLog2e);
            const float grow = e == 1.f ? d : (e - 1.f) * (d / logf(e));
            s.f_out = s.up * (fabsf(d) < 0.5f ? g.p_rest * grow : __builtin_amdgcn_exp2f(a.log_q_rest * kLog2e) - g.p_rest);
            s.m_out = a.mo;
            s.o_out = -a.zo * kLog2e;
        }
    }
    return s;
}
// taken: the record's share of the label, -1 where it is not named
__device__ inline float slope(const Slope &s, float x, float taken, float c2)
{
    const bool named = !(taken < 0.f);          // (a share may be NaN)
    const float e = __builtin_amdgcn_exp2f((x - (named ? s.m_top : s.m_out)) * c2 + (named ? s.o_top : s.o_out));
    return named ? s.up * (e - taken) : s.f_out * e;
}

// ---- one lane per row (see mfl_top_labels.hip for the two shapes of work)
//
// A lane takes its labels CB at a time and its record's entries KB at a time, all loads of a block in flight at once; the
// student's scores of the record are fetched by label beside the stream.  With KB >= k the record stays in registers, with
// CB >= C the scores do, and the backward pass then finds the softmax statistics by itself instead of reading them back
// (16 bytes of 200 a pixel at 21 labels).

constexpr int kLoneBlock = MFL_DISTILLATION_LONE_LABELS;        // up to this many labels a lane's scores stay in registers

// Entries j0 .. j0 + KB of a row's record; x: the student's scores of their labels
template <typename T, int KB> struct Block {
    int label[KB];              // -1: none, or no label of the row
    float value[KB], x[KB];
    __device__ Block(const Rows &in, const Teacher &t, size_t base, int j0)
    {
        auto at = [&](int j) { return base + (size_t)min(j0 + j, t.k - 1) * in.S; };
#pragma unroll
        for (int j = 0; j < KB; ++j) label[j] = t.labels[at(j)];
        load_any(value, t.values, t.dtype, at);
    }
    __device__ void fetch(const Rows &in, const Teacher &t, const T *p, int j0)
    {
        T raw[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            label[j] = j0 + j < t.k && (unsigned)label[j] < (unsigned)in.C ? label[j] : -1;
            raw[j] = p[max(label[j], 0) * in.sc];
        }
#pragma unroll
        for (int j = 0; j < KB; ++j) x[j] = to_float(raw[j]);
    }
};

// valid and rest of a row, read from some address without a branch, so that nothing waits for them before they are used
struct RowFlags {
    unsigned char v;
    float r;
    __device__ RowFlags(const Teacher &t, unsigned row)
        : v(*(t.valid ? t.valid + row : (const unsigned char *)t.labels)), r(*(t.rest ? t.rest + row : (const float *)t.labels)) {}
    __device__ bool valid(const Teacher &t) const { return !t.valid || v; }
    __device__ float rest(const Teacher &t) const { return t.rest ? r : -INFINITY; }
};

// The used ones of KB scores as one Excess: the largest first, so that its own 1 is never added
template <int KB> __device__ inline Excess excess_of(const float (&v)[KB], const bool (&used)[KB], float c2)
{
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int j = 0; j < KB; ++j) m = used[j] ? fmaxf(m, v[j]) : m;
    const float ref = finite_or_zero(m);
    bool found = false;
#pragma unroll
    for (int j = 0; j < KB; ++j) {
        const bool first = used[j] && v[j] == m && !found;
        found |= first;
        s += used[j] && !first ? __builtin_amdgcn_exp2f((v[j] - ref) * c2) : 0.f;
    }
    return {m, m == -INFINITY && s == 0.f ? -1.f : s};
}

// A record as one lane goes over it: f(block) for all of it, from registers where it fits
template <typename T, int KB, bool ALL> struct LaneRecord {
    const Rows &in;
    const Teacher &t;
    const T *p;
    size_t base;
    Block<T, KB> first;
    __device__ LaneRecord(const Rows &in, const Teacher &t, const T *p, size_t base) : in(in), t(t), p(p), base(base), first(in, t, base, 0) {}
    __device__ void fetch() { first.fetch(in, t, p, 0); }
    template <typename F> __device__ void each(F f) const
    {
        f(first);
        if constexpr (!ALL)
            for (int j0 = KB; j0 < t.k; j0 += KB) {
                Block<T, KB> b(in, t, base, j0);
                b.fetch(in, t, p, j0);
                f(b);
            }
    }
    __device__ Target target(float rest) const
    {
        Excess sum = kNoExcess;
        bool named = false;
        each([&](const Block<T, KB> &b) {
            bool used[KB];
#pragma unroll
            for (int j = 0; j < KB; ++j) named |= used[j] = b.label[j] >= 0;
            const Excess e = excess_of(b.value, used, t.c2);
            sum = ALL ? e : join(sum, e, t.c2);
        });
        return target_of(t, sum, named, rest);
    }
};

// Labels c0 .. c0 + CB of a row (what lies behind the last one: -inf).  The first SURE of them are there.
template <int CB, bool LONE> constexpr int kSure = LONE && CB > 8 ? CB - 3 : 1;
template <int SURE, typename T, int CB> __device__ inline void load_labels(float (&x)[CB], const Rows &in, const T *p, int c0)
{
    T raw[CB];
    const T *q = p + c0 * in.sc;
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        raw[i] = *q;
        q += i + 1 < SURE || c0 + i + 1 < in.C ? in.sc : 0;         // (the last one again)
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) x[i] = i < SURE || c0 + i < in.C ? to_float(raw[i]) : -INFINITY;
}

// Adds a block of labels to the two sums: the record's into top (each once), the others into out
template <typename T, int CB, bool LONE, int KB, bool ALL>
__device__ inline void add_labels(const LaneRecord<T, KB, ALL> &record, const float (&x)[CB], int c0, float c2, LogSum &out, Excess &top)
{
    static_assert(CB <= 32, "one word of marks");
    uint32_t marks = 0;
    record.each([&](const Block<T, KB> &b) {
        bool used[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            const int i = b.label[j] - c0;
            const uint32_t bit = b.label[j] >= 0 && (LONE || (unsigned)i < (unsigned)CB) ? 1u << (i & 31) : 0u;
            used[j] = (bit & ~marks) != 0;
            marks |= bit;
        }
        const Excess e = excess_of(b.x, used, c2);
        top = LONE && ALL ? e : join(top, e, c2);
    });
    float m = out.m, y[CB];
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        y[i] = minus_inf_where(marks, i, x[i]);
        m = fmaxf(m, y[i]);
    }
    const float ref = finite_or_zero(m);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < CB; ++i) sum += __builtin_amdgcn_exp2f((y[i] - ref) * c2);
    out = {m, fmaf(out.s, __builtin_amdgcn_exp2f((out.m - ref) * c2), sum)};
}

// LONE: C <= CB
template <typename T, int CB, bool LONE, int KB, bool ALL>
__global__ void __launch_bounds__(kLaneThreads)
forward_lanes_kernel(Rows in, Teacher t, float *__restrict__ loss, float *__restrict__ stats)
{
    const unsigned r = blockIdx.x * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    constexpr int SURE = kSure<CB, LONE>;
    // (everything is asked for before anything is looked at)
    LaneRecord<T, KB, ALL> record(in, t, p, (size_t)n * t.k * in.S + s);
    float x[CB];
    load_labels<SURE>(x, in, p, 0);
    const RowFlags flags(t, r);
    record.fetch();
    LogSum out = {-INFINITY, 0.f};
    Excess top = kNoExcess;
    for (int c0 = 0;;) {
        add_labels<T, CB, LONE>(record, x, c0, t.c2, out, top);
        c0 += CB;
        if (LONE || c0 >= in.C) break;
        load_labels<SURE>(x, in, p, c0);
    }
    const Target g = record.target(flags.rest(t));
    const Stats a = stats_of(top, out, t);
    if (!flags.valid(t) || !g.any || a.m == -INFINITY) return put(loss, LONE ? nullptr : stats, in.rows, r, 0.f, kNoStats);
    const float dl = log_sums(g, a);
    float sum = rest_term(t, g, a);
    record.each([&](const Block<T, KB> &b) {
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            sum += b.label[j] >= 0 ? entry_term(t, g, dl, a.m, b.value[j], b.x[j]) : 0.f;
        }
    });
    put(loss, LONE ? nullptr : stats, in.rows, r, sum, a);
}

// What the record takes from each label of a block lies in LDS, one column per lane (-1: not named).
template <typename T, int CB, bool LONE, int KB, bool ALL>
__global__ void __launch_bounds__(kLaneThreads)
backward_lanes_kernel(Rows in, Teacher t, const float *__restrict__ stats, const float *__restrict__ grad_loss, T *__restrict__ grad,
                      long long gn, long long gc, long long gs)
{
    __shared__ float taken[CB][kLaneThreads];
    constexpr int SURE = kSure<CB, LONE>;
    // (from the last row on: what the forward pass read last is still in the last-level cache)
    const unsigned r = (gridDim.x - 1 - blockIdx.x) * kLaneThreads + threadIdx.x;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    T *out = grad + (long long)n * gn + (long long)s * gs;
    LaneRecord<T, KB, ALL> record(in, t, p, (size_t)n * t.k * in.S + s);
    float x[CB];
    load_labels<SURE>(x, in, p, 0);
    const RowFlags flags(t, r);
    const float up = grad_loss[r];
    record.fetch();
    Stats a;
    if constexpr (LONE) {
        LogSum other = {-INFINITY, 0.f};
        Excess top = kNoExcess;
        add_labels<T, CB, LONE>(record, x, 0, t.c2, other, top);
        a = stats_of(top, other, t);
    } else {
        a = load_stats(stats, in.rows, r);
    }
    const Target g = record.target(flags.rest(t));
    if (!flags.valid(t) || a.m == -INFINITY || !g.any) {
        for (int c = 0; c < in.C; ++c) from_float(0.f, out[c * gc]);
        return;
    }
    const Slope sl = slope_of(a, t, g, up);
#pragma unroll
    for (int i = 0; i < CB; ++i) taken[i][threadIdx.x] = -1.f;
    for (int c0 = 0; c0 < (LONE ? 1 : in.C); c0 += CB) {
        if (c0) load_labels<SURE>(x, in, p, c0);
        record.each([&](const Block<T, KB> &b) {
#pragma unroll
            for (int j = 0; j < KB; ++j) {
                const int i = b.label[j] - c0;
                if (b.label[j] < 0 || (unsigned)i >= (unsigned)CB) continue;
                taken[i][threadIdx.x] = fmaxf(taken[i][threadIdx.x], 0.f) + __builtin_amdgcn_exp2f(log_share(t, g, b.value[j]) * kLog2e);
            }
        });
        T *w = out + c0 * gc;
#pragma unroll
        for (int i = 0; i < CB; ++i) {
            const float share = taken[i][threadIdx.x];
            if (i < SURE || c0 + i < in.C) store_once(slope(sl, x[i], share, t.c2), w + i * gc);
            if (!(share < 0.f)) taken[i][threadIdx.x] = -1.f;
        }
    }
}

// ---- one or more workgroups per row (class stride 1)
//
// Rows of many labels are cut into parts, as many as it takes to have work for the whole card: a part's running sum over
// the labels outside the record goes to the workspace, and one wave per row joins them and adds the record's side.

constexpr int kRowThreads = 256;
constexpr int kSegment = 1 << 16;       // labels marked at a time by a workgroup: 8 KB of bits
constexpr int kMaxParts = 64;
constexpr int kMinPart = 8192;

__host__ __device__ inline int part_labels(int C, int parts) { return (((C + parts - 1) / parts) + 2047) & ~2047; }
int parts_of(const Rows &in, unsigned enough)
{
    const unsigned most = (unsigned)((in.C + kMinPart - 1) / kMinPart), want = (enough + in.rows - 1) / in.rows;
    const unsigned n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > kMaxParts ? kMaxParts : n);
}

// Marks the record's labels in [c0, c1) as bits
__device__ inline void mark(uint32_t *bits, const Teacher &t, size_t base, size_t step, int c0, int c1)
{
    for (int w = threadIdx.x; w < (c1 - c0 + 31) / 32; w += kRowThreads) bits[w] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < t.k; j += kRowThreads) {
        const int i = t.labels[base + (size_t)j * step];
        if (i >= c0 && i < c1) atomicOr(&bits[(i - c0) >> 5], 1u << ((i - c0) & 31));
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
outside_parts_kernel(Rows in, Teacher t, int parts, LogSum *__restrict__ sums)
{
    extern __shared__ uint32_t bits[];
    __shared__ LogSum wave_sum[kRowThreads / 64];
    constexpr int V = kVec<T>;
    const unsigned r = blockIdx.x / parts, part = blockIdx.x - r * parts;
    const unsigned n = r / in.S, s = r - n * in.S;
    if (t.valid && !t.valid[r]) return;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const size_t base = (size_t)n * t.k * in.S + s;
    const int size = part_labels(in.C, parts);
    const int begin = min(in.C, (int)part * size), end = min(in.C, begin + size);
    LogSum out = {-INFINITY, 0.f};
    for (int c0 = begin; c0 < end; c0 += kSegment) {
        const int c1 = min(end, c0 + kSegment);
        if (c0 > begin) __syncthreads();
        mark(bits, t, base, in.S, c0, c1);
        auto take = [&](float (&x)[V], int c) {
            const uint32_t marks = ((const uint8_t *)bits)[(c - c0) >> 3] >> (V == 4 ? (c - c0) & 4 : 0);
            if (marks) {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = marks >> i & 1 ? -INFINITY : x[i];
            }
            float m = out.m;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
            const float ref = finite_or_zero(m);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * t.c2);
            out = {m, fmaf(out.s, __builtin_amdgcn_exp2f((out.m - ref) * t.c2), sum)};
        };
        constexpr int U = 4;            // vectors in flight
        int c = c0 + threadIdx.x * V;
        for (; c + (U - 1) * kRowThreads * V + V <= c1; c += U * kRowThreads * V) {
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) load_vec(p + c + u * kRowThreads * V, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) take(x[u], c + u * kRowThreads * V);
        }
        for (; c < c1; c += kRowThreads * V) {
            float x[V];
            if (c + V <= c1) {
                load_vec(p + c, x);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = c + i < c1 ? to_float(p[c + i]) : -INFINITY;
            }
            take(x, c);
        }
    }
    out = wave_join(out, t.c2);
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = out;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowThreads / 64; ++w) out = join(out, wave_sum[w], t.c2);
        sums[blockIdx.x] = out;
    }
}

// A row's record over the lanes of a wave, entries lane and lane + 64
struct Entries {
    int label[2];
    float value[2];
    bool in[2];                 // a label of the row
};
__device__ inline Entries entries_of(const Teacher &t, int C, size_t base, size_t step, int lane)
{
    Entries e;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane + 64 * h;
        e.label[h] = j < t.k ? t.labels[base + (size_t)j * step] : -1;
        e.in[h] = (unsigned)e.label[h] < (unsigned)C;
    }
    load_any(e.value, t.values, t.dtype, [&](int h) { return base + (size_t)min(lane + 64 * h, t.k - 1) * step; });
    return e;
}
__device__ inline Target target_by_wave(const Teacher &t, const Entries &e, unsigned r)
{
    Excess sum = kNoExcess;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (e.in[h]) sum = join(sum, Excess{e.value[h], 0.f}, t.c2);
    const bool named = __any(e.in[0] || e.in[1]);
    return target_of(t, wave_join(sum, t.c2), named, t.rest ? t.rest[r] : -INFINITY);
}

// One wave per row
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
finish_rows_kernel(Rows in, Teacher t, int parts, const LogSum *__restrict__ sums, float *__restrict__ loss, float *__restrict__ stats)
{
    __shared__ int labels[kRowThreads / 64][MFL_MAX_TOP_LABELS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned r = blockIdx.x * (kRowThreads / 64) + wave;
    if (r >= in.rows) return;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    const size_t base = (size_t)n * t.k * in.S + s;
    if (t.valid && !t.valid[r]) {
        if (lane == 0) put(loss, stats, in.rows, r, 0.f, kNoStats);
        return;
    }
    const Entries e = entries_of(t, in.C, base, in.S, lane);
    float x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        x[h] = e.in[h] ? to_float(p[e.label[h]]) : -INFINITY;
        labels[wave][lane + 64 * h] = e.label[h];
    }
    LogSum out = lane < parts ? sums[(size_t)r * parts + lane] : LogSum{-INFINITY, 0.f};
    out = wave_join(out, t.c2);
    const Target g = target_by_wave(t, e, r);
    if (!g.any) {
        if (lane == 0) put(loss, stats, in.rows, r, 0.f, kNoStats);
        return;
    }
    // the record's labels on the student's side: each once, by the first entry that names it
    __builtin_amdgcn_wave_barrier();
    bool again[2] = {false, false};
    for (int j = 0; j < t.k; ++j) {
        const int l = labels[wave][j];
#pragma unroll
        for (int h = 0; h < 2; ++h) again[h] |= j < lane + 64 * h && l == e.label[h];
    }
    Excess top = kNoExcess;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (e.in[h] && !again[h]) top = join(top, Excess{x[h], 0.f}, t.c2);
    top = wave_join(top, t.c2);
    const Stats a = stats_of(top, out, t);
    if (a.m == -INFINITY) {
        if (lane == 0) put(loss, stats, in.rows, r, 0.f, a);
        return;
    }
    const float dl = log_sums(g, a);
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) sum += e.in[h] ? entry_term(t, g, dl, a.m, e.value[h], x[h]) : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    sum += rest_term(t, g, a);
    if (lane == 0) put(loss, stats, in.rows, r, sum, a);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
backward_rows_kernel(Rows in, Teacher t, int parts, const float *__restrict__ stats, const float *__restrict__ grad_loss,
                     T *__restrict__ grad, long long gn, long long gs)
{
    extern __shared__ uint32_t bits[];
    __shared__ int label[MFL_MAX_TOP_LABELS];
    __shared__ float share[MFL_MAX_TOP_LABELS];
    constexpr int V = kVec<T>;
    const int lane = threadIdx.x & 63;
    // (from the last row on: what the forward pass read last is still in the last-level cache)
    const unsigned q = blockIdx.x / parts, part = blockIdx.x - q * parts, r = in.rows - 1 - q;
    const unsigned n = r / in.S, s = r - n * in.S;
    const T *p = (const T *)in.p + (long long)n * in.sn + (long long)s * in.ss;
    T *out = grad + (long long)n * gn + (long long)s * gs;
    const size_t base = (size_t)n * t.k * in.S + s;
    const int size = part_labels(in.C, parts);
    const int begin = min(in.C, (int)part * size), end = min(in.C, begin + size);
    const Stats a = load_stats(stats, in.rows, r);
    Target g;
    g.any = false;
    if (!(t.valid && !t.valid[r]) && a.m != -INFINITY) {
        const Entries e = entries_of(t, in.C, base, in.S, lane);
        g = target_by_wave(t, e, r);
        if (threadIdx.x < 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                label[lane + 64 * h] = e.label[h];
                share[lane + 64 * h] = e.in[h] ? __builtin_amdgcn_exp2f(log_share(t, g, e.value[h]) * kLog2e) : 0.f;
            }
        }
    }
    if (!g.any) {
        const float zero[V] = {};
        for (int c = begin + threadIdx.x * V; c < end; c += kRowThreads * V) {
            if (c + V <= end) {
                store_vec(out + c, zero);
            } else {
                for (int i = c; i < end; ++i) from_float(0.f, out[i]);
            }
        }
        return;
    }
    const Slope sl = slope_of(a, t, g, grad_loss[r]);
    for (int c0 = begin; c0 < end; c0 += kSegment) {
        const int c1 = min(end, c0 + kSegment);
        __syncthreads();
        mark(bits, t, base, in.S, c0, c1);
        auto turn = [&](float (&x)[V], int c) {
            const uint32_t marks = ((const uint8_t *)bits)[(c - c0) >> 3] >> (V == 4 ? (c - c0) & 4 : 0);
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = sl.f_out * __builtin_amdgcn_exp2f(fmaf(x[i] - sl.m_out, t.c2, sl.o_out));
            if (marks & ((1 << V) - 1)) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (!(marks >> i & 1)) continue;
                    float sum = 0.f;
                    for (int j = 0; j < t.k; ++j) sum += label[j] == c + i ? share[j] : 0.f;
                    y[i] = slope(sl, x[i], sum, t.c2);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = y[i];
        };
        constexpr int U = 4;
        int c = c0 + threadIdx.x * V;
        for (; c + (U - 1) * kRowThreads * V + V <= c1; c += U * kRowThreads * V) {
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) unpack<T>(load_words_once(p + c + u * kRowThreads * V), x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                turn(x[u], c + u * kRowThreads * V);
                store_vec(out + c + u * kRowThreads * V, x[u]);
            }
        }
        for (; c < c1; c += kRowThreads * V) {
            float x[V];
            if (c + V <= c1) {
                load_vec(p + c, x);
                turn(x, c);
                store_vec(out + c, x);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = c + i < c1 ? to_float(p[c + i]) : 0.f;
                turn(x, c);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (c + i < c1) from_float(x[i], out[c + i]);
            }
        }
    }
}

// (few short rows as well: a lane alone takes its time over a long record.)  Lanes / rows, fp32, k = 8 with rest, both passes, us:
// 4096 x 64 37 / 37, 16384 x 64 51 / 85, 16384 x 128 95 / 87, 4096 x 256 103 / 37, 16384 x 512 329 / 97, 131072 x 128 728 / 616.
// (Many rows of 128 to 511 labels would do better by rows, for the gradient's stores: 131072 x 256 1664 / 616.)
bool by_rows(const Rows &in) { return in.sc == 1 && (in.C >= 512 || (in.C >= 64 && in.rows <= 16384)); }
size_t mark_bytes(int C, int parts)
{
    const int size = part_labels(C, parts);
    return (size_t)(size < kSegment ? size : kSegment) / 8;
}
constexpr unsigned kEnough = 8192;      // workgroups: 32 for each of 256 CUs, so that the last ones end together

// labels and entries a lane takes at a time
#define MFL_BY_SIZE(C, k, LAUNCH)                                                             \
    do {                                                                                      \
        if (C <= kLoneBlock) {                                                                \
            if (k <= 4) {                                                                     \
                if (C <= 8) LAUNCH(8, true, 4, true);                                         \
                else if (C <= 12) LAUNCH(12, true, 4, true);                                  \
                else if (C <= 16) LAUNCH(16, true, 4, true);                                  \
                else if (C <= 20) LAUNCH(20, true, 4, true);                                  \
                else LAUNCH(24, true, 4, true);                                               \
            } else {                                                                          \
                if (C <= 8) LAUNCH(8, true, 8, false);                                        \
                else if (C <= 12) LAUNCH(12, true, 8, false);                                 \
                else if (C <= 16) LAUNCH(16, true, 8, false);                                 \
                else if (C <= 20) LAUNCH(20, true, 8, false);                                 \
                else LAUNCH(24, true, 8, false);                                              \
            }                                                                                 \
        } else {                                                                              \
            if (k <= 4) LAUNCH(32, false, 4, true);                                           \
            else if (k <= 8) LAUNCH(32, false, 8, true);                                      \
            else LAUNCH(32, false, 8, false);                                                 \
        }                                                                                     \
    } while (0)

template <typename T>
int run_forward(const Rows &in, const Teacher &t, float *loss, float *stats, void *workspace, hipStream_t st)
{
    if (by_rows(in)) {
        const int parts = parts_of(in, kEnough);
        if (!launchable((unsigned long long)in.rows * parts, kRowThreads)) return MFL_ERR_TOO_LARGE;
        hipLaunchKernelGGL(outside_parts_kernel<T>, dim3(in.rows * parts), dim3(kRowThreads), mark_bytes(in.C, parts), st, in, t, parts,
                           (LogSum *)workspace);
        const unsigned per = kRowThreads / 64;
        hipLaunchKernelGGL(finish_rows_kernel<T>, dim3((in.rows + per - 1) / per), dim3(kRowThreads), 0, st, in, t, parts,
                           (const LogSum *)workspace, loss, stats);
        return (int)hipGetLastError();
    }
    const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
#define MFL_LANES(CB, LONE, KB, ALL) \
    hipLaunchKernelGGL((forward_lanes_kernel<T, CB, LONE, KB, ALL>), grid, block, 0, st, in, t, loss, stats)
    MFL_BY_SIZE(in.C, t.k, MFL_LANES);
#undef MFL_LANES
    return (int)hipGetLastError();
}

template <typename T>
int run_backward(const Rows &in, const Teacher &t, const float *stats, const float *grad_loss, void *grad, const Rows &out, hipStream_t st)
{
    if (by_rows(in) && out.sc == 1) {
        const int parts = parts_of(in, kEnough);
        if (!launchable((unsigned long long)in.rows * parts, kRowThreads)) return MFL_ERR_TOO_LARGE;
        hipLaunchKernelGGL(backward_rows_kernel<T>, dim3(in.rows * parts), dim3(kRowThreads), mark_bytes(in.C, parts), st, in, t, parts,
                           stats, grad_loss, (T *)grad, out.sn, out.ss);
        return (int)hipGetLastError();
    }
    const dim3 grid((in.rows + kLaneThreads - 1) / kLaneThreads), block(kLaneThreads);
#define MFL_LANES(CB, LONE, KB, ALL) \
    hipLaunchKernelGGL((backward_lanes_kernel<T, CB, LONE, KB, ALL>), grid, block, 0, st, in, t, stats, grad_loss, (T *)grad, out.sn, out.sc, \
                       out.ss)
    MFL_BY_SIZE(in.C, t.k, MFL_LANES);
#undef MFL_LANES
    return (int)hipGetLastError();
}

int make_teacher(Teacher &t, const void *values, int dtype, const int *labels, const float *rest, const unsigned char *valid, int k,
                 double temperature)
{
    // (the loss is T^2 times a sum: an ordinary fp32 number as well, or a loss of 0 becomes a NaN)
    if (!values || !labels || k < 1 || k > MFL_MAX_TOP_LABELS || !(temperature >= 1e-18 && temperature <= 1e18)) return MFL_ERR_INVALID_ARGUMENT;
    if (dtype != MFL_F32 && dtype != MFL_BF16 && dtype != MFL_F16) return MFL_ERR_INVALID_ARGUMENT;
    t = {values, dtype, labels, rest, valid, k, (float)(kLog2eD / temperature), (float)(1.0 / temperature), (float)temperature};
    return MFL_OK;
}

}  // namespace

extern "C" {

// (for any strides: a size that the lanes serve is not worth telling apart)
size_t mfl_distillation_workspace_bytes(int N, int C, int S, int dtype, int k)
{
    Rows in;
    if (make_rows(in, "", dtype, N, C, S, 0, 1, 0) || k < 1 || !by_rows(in)) return 0;
    return (size_t)in.rows * parts_of(in, kEnough) * sizeof(LogSum);
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
    if (by_rows(in) && (!workspace || workspace_bytes < mfl_distillation_workspace_bytes(N, C, S, dtype, k))) return MFL_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case MFL_F32: return run_forward<float>(in, t, loss, stats, workspace, st);
    case MFL_BF16: return run_forward<bf16_t>(in, t, loss, stats, workspace, st);
    default: return run_forward<f16_t>(in, t, loss, stats, workspace, st);
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
    case MFL_F32: return run_backward<float>(in, t, stats, grad_loss, d_scores, out, st);
    case MFL_BF16: return run_backward<bf16_t>(in, t, stats, grad_loss, d_scores, out, st);
    default: return run_backward<f16_t>(in, t, stats, grad_loss, d_scores, out, st);
    }
}

}  // extern "C"
