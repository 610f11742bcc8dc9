// The k <= 128 largest scores of a run of labels, by one wave in one pass (mfl_top_labels.hip, mfl_sample_labels.hip).
//
// The wave keeps a list of candidates in LDS, as rank keys, and a bound below which no label can be among the k best any
// more.  A vector of scores with none above the bound costs a compare each; scores above it are appended.  When
// the list has grown, a binary search over the keys (held in registers, counted by ballots) finds a bound that
// leaves between k and about 2 k of them, and the others leave.  Before the first search a look at the first part's largest
// score per lane gives a bound.  For scores in random order a few hundred labels are appended at all; for rising ones every
// label is, at one search per few hundred.  Everything that never enters or
// leaves the list goes into the rest's running sum exactly once.  Appending follows the order of the labels and every count
// is the wave's own: no atomics, the same result every time.
//
// Measured, 1024 rows of 32001 bf16 scores, k = 64: a list that starts with the first 512 scores, four independent waves a
// row and a second launch to join them 75 us; with the look at the first scores 65; the four waves agreeing on it and
// joining in place 36.
#ifndef MFL_WAVE_TOP_H
#define MFL_WAVE_TOP_H

#include "mfl_scores.h"

namespace mfl_scores {

constexpr int kWaveTopThreads = 256;
constexpr int kListKeys = 1024;

// Keys a search leaves at most, and a part of a row hands on
__host__ __device__ inline int part_keys(int k) { return k < 64 ? 2 * k + 32 : k + k / 2; }

typedef __attribute__((address_space(3))) uint64_t lds_key;

template <bool REST> struct WaveTop {
    lds_key *list;              // kListKeys, this wave's own
    int k, count;
    uint64_t bound;             // keys up to it are out
    float bound_score;
    float c2;
    LogSum rest;                // this lane's share

    __device__ WaveTop(uint64_t *list, int k, float c2)
        : list((lds_key *)list), k(k), count(0), bound(0), bound_score(-INFINITY), c2(c2), rest{-INFINITY, 0.f} {}

    // Leaves between `least` (<= count) and `most` keys in the list
    __device__ void shrink(int least, int most)
    {
        constexpr int R = kListKeys / 128;          // registers of half a list
        const int lane = threadIdx.x & 63;
        const bool both = count > kListKeys / 2;    // the second half holds something
        uint64_t r[2][R];
        __builtin_amdgcn_wave_barrier();
        auto load = [&](uint64_t (&h)[R], int from) {
#pragma unroll
            for (int i = 0; i < R; ++i) h[i] = from + 64 * i + lane < count ? list[from + 64 * i + lane] : 0;
        };
        load(r[0], 0);
        if (both) load(r[1], kListKeys / 2);
        auto scores_above = [&](const uint64_t (&h)[R], uint32_t at) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < R; ++i) n += __popcll(__ballot((uint32_t)(h[i] >> 32) > at));
            return n;
        };
        auto keys_above = [&](const uint64_t (&h)[R], uint64_t at) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < R; ++i) n += __popcll(__ballot(h[i] > at));
            return n;
        };
        // by the scores first: more than `most` above lo, fewer than `least` above hi
        uint32_t lo = (uint32_t)(bound >> 32), hi = ~0u, at = lo;
        bool found = false;
        while (hi - lo > 1) {
            at = lo + (hi - lo) / 2;
            int above = scores_above(r[0], at);
            if (both) above += scores_above(r[1], at);
            if (above > most) {
                lo = at;
            } else if (above < least) {
                hi = at;
            } else {
                found = true;
                break;
            }
        }
        if (found) {
            bound = (uint64_t)at << 32 | 0xffffffffu;
        } else {
            // too many share one score: by their labels (the scores up to lo are out, those above hi are in)
            uint64_t mid = lo == (uint32_t)(bound >> 32) ? bound : (uint64_t)lo << 32 | 0xffffffffu;
            uint64_t end = (uint64_t)hi << 32 | 0xffffffffu;
            while (end - mid > 1) {
                const uint64_t m = mid + (end - mid) / 2;
                int above = keys_above(r[0], m);
                if (both) above += keys_above(r[1], m);
                if (above < least) {
                    end = m;
                } else {
                    mid = m;
                    if (above <= most) break;
                }
            }
            bound = mid;
        }
        count = 0;
        auto keep = [&](const uint64_t (&h)[R]) {
            float out[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool stay = h[i] > bound;
                const uint64_t who = __ballot(stay);
                if (stay) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = h[i];
                count += __popcll(who);
                out[i] = stay || !h[i] ? -INFINITY : rank_score(h[i]);
            }
            if (REST) add_to_rest(out);
        };
        keep(r[0]);
        if (both) keep(r[1]);
        bound_score = rank_score(bound);
        __builtin_amdgcn_wave_barrier();
    }
    __device__ int most() const { return part_keys(k); }

    // Keeps the list short: its bound is only as tight as the last search
    __device__ void room()
    {
        if (count >= most() + 128) shrink(k, most());
    }
    // Appends this lane's key if it brings one; returns whether it went in
    __device__ bool append(uint64_t key, bool bring)
    {
        bring = bring && key > bound;
        const uint64_t who = __ballot(bring);
        if (bring) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key;
        count += __popcll(who);
        return bring;
    }
    template <int V> __device__ void add_to_rest(const float (&x)[V])
    {
        float top = rest.m;
#pragma unroll
        for (int i = 0; i < V; ++i) top = max_or_nan(top, x[i]);
        const float ref = finite_or_zero(top);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * c2);
        rest = {top, fmaf(rest.s, __builtin_amdgcn_exp2f((rest.m - ref) * c2), sum)};
    }

    template <int V> __device__ void take(float (&x)[V], int c, int end)
    {
        static_assert(MFL_MAX_TOP_LABELS * 3 / 2 + 128 + 64 * V <= kListKeys, "a vector fits behind a list that room() leaves");
        room();
        // (a NaN is not below the bound either)
        uint32_t open = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) open |= !(x[i] < bound_score) ? 1u << i : 0u;
        if (c + V > end) open &= (1u << max(end - c, 0)) - 1;
        // every lane brings its first open score, then its second: a turn or two once the bound is tight
        uint32_t in = 0;
        while (__any(open != 0)) {
            const int i = __ffs(open) - 1;
            float v = x[0];
#pragma unroll
            for (int j = 1; j < V; ++j) v = i == j ? x[j] : v;
            if (append(rank_key(score_key(v), c + i), open != 0)) in |= 1u << i;
            open &= open - 1;
        }
        if (REST) {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = minus_inf_where(in, j, x[j]);
            add_to_rest(x);
        }
    }

    // The largest scores of four disjoint sets a lane, among the first `vectors` of the labels at p + begin
    template <typename T> __device__ static void look(const T *p, int begin, int vectors, float (&m)[4])
    {
        constexpr int V = kVec<T>;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < 4; ++u) m[u] = -INFINITY;
        int v = 0;
        for (; v + 4 <= vectors; v += 4) {
            float x[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) load_vec(p + begin + ((v + u) * 64 + lane) * V, x[u]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < V; ++i) m[u] = fmaxf(m[u], x[u][i]);
        }
        for (; v < vectors; ++v) {
            float x[V];
            load_vec(p + begin + (v * 64 + lane) * V, x);
#pragma unroll
            for (int i = 0; i < V; ++i) m[0] = fmaxf(m[0], x[i]);
        }
    }
    // A bound to begin with, from the largest scores of 256 disjoint sets of labels, four a lane: where k sets hold a score
    // that large, k labels do.
    __device__ void foresee(const float (&m)[4])
    {
        uint32_t seen[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) seen[u] = (uint32_t)score_key(m[u]) ^ 0x80000000u;
        uint32_t lo = 0, hi = ~0u;                  // at least k sets reach lo, fewer hi
        while (hi - lo > 1) {
            const uint32_t at = lo + (hi - lo) / 2;
            int n = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) n += __popcll(__ballot(seen[u] >= at));
            if (n >= k) {
                lo = at;
                if (n == k) break;
            } else {
                hi = at;
            }
        }
        if (lo) {
            bound = ((uint64_t)lo << 32) - 1;
            bound_score = key_score((int)(lo ^ 0x80000000u));
        }
    }

    // Labels begin .. end of a row at p
    template <typename T> __device__ void stream(const T *p, long long sc, int begin, int end)
    {
        constexpr int V = kVec<T>;
        const int lane = threadIdx.x & 63;
        if (sc == 1) {
            // (one copy of the loop's body: three vectors ahead, kept as bits)
            constexpr int step = 64 * V;
            const int whole = begin + (end - begin) / step * step;
            if (begin < whole) {
                // (past the last one: the last one again, so that the count of loads in flight is the same all the way)
                auto ahead = [&](int c) { return load_words(p + min(c, whole - step) + lane * V); };
                words4 a = ahead(begin), b = ahead(begin + step), d = ahead(begin + 2 * step);
#pragma unroll 1
                for (int c = begin; c < whole; c += step) {
                    float x[V];
                    unpack<T>(a, x);
                    a = b;
                    b = d;
                    d = ahead(c + 3 * step);
                    take(x, c + lane * V, end);
                }
            }
            if (whole < end) {
                const int at = whole + lane * V;
                float x[V];
#pragma unroll
                for (int i = 0; i < V; ++i) x[i] = at + i < end ? to_float(p[at + i]) : -INFINITY;
                take(x, at, end);
            }
        } else {
#pragma unroll 1
            for (int c = begin; c < end; c += 64) {
                float x[1] = {c + lane < end ? to_float(p[(c + lane) * sc]) : -INFINITY};
                take(x, c + lane, end);
            }
        }
    }

    // Keys that other waves found (0: none)
    template <typename Key> __device__ void join(Key *keys, int n)
    {
        const int lane = threadIdx.x & 63;
        if (n <= 0) return;
        auto ahead = [&](int i) { return (uint64_t)keys[min(i + lane, n - 1)]; };
        uint64_t next[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) next[u] = ahead(64 * u);
#pragma unroll 1
        for (int i = 0; i < n; i += 64) {
            const uint64_t key = i + lane < n ? next[0] : 0;
#pragma unroll
            for (int u = 0; u < 3; ++u) next[u] = next[u + 1];
            next[3] = ahead(i + 4 * 64);
            room();
            const bool in = append(key, key != 0);
            if (REST && __any(!in && key)) add_score(rest, !in && key ? rank_score(key) : -INFINITY, c2);
        }
    }

    // Down to at most as many as ranked() and a draw take
    __device__ void cut()
    {
        if (count > MFL_MAX_TOP_LABELS) shrink(k, MFL_MAX_TOP_LABELS);
    }

    // f(rank, key) for the k best of at most 128 keys, by counting what is above each; the others go to the rest
    template <typename F> __device__ void ranked(F f)
    {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_wave_barrier();
        const uint64_t a = lane < count ? list[lane] : 0, b = lane + 64 < count ? list[lane + 64] : 0;
        int above_a = 0, above_b = 0;
        for (int j = 0; j < count; ++j) {
            const uint64_t key = list[j];
            above_a += key > a;
            above_b += key > b;
        }
        if (a && above_a < k) f(above_a, a);
        if (b && above_b < k) f(above_b, b);
        const float out[2] = {a && above_a >= k ? rank_score(a) : -INFINITY, b && above_b >= k ? rank_score(b) : -INFINITY};
        if (REST) add_to_rest(out);
    }
};

// ---- a workgroup's four waves on one part of a row, or on four rows
//
// Four waves on one part agree on the bound to begin with: every lane brings the largest of up to 64 scores.  At k = 64 of 256
// such sets the bound lets 0.5 % of scores in random order through, where a wave's own look lets 1.8 % through.  The first
// wave then joins the four lists.

struct TopShared {
    uint64_t lists[kWaveTopThreads / 64][kListKeys];
    float seen[kWaveTopThreads];
    LogSum rest[kWaveTopThreads / 64];
    int count[kWaveTopThreads / 64];
};

// The first wave takes over the four lists.  After it its list holds the part's k best and perhaps more (no more than
// most()), and its lanes the shares of the rest; the other waves are done (false).
template <bool REST> __device__ inline bool join_waves(WaveTop<REST> &top, TopShared &sh)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (top.count > kListKeys / 2) top.shrink(top.k, top.most());
    const LogSum rest = wave_join(top.rest, top.c2);
    if (lane == 0) {
        sh.count[wave] = top.count;
        sh.rest[wave] = rest;
    }
    __syncthreads();
    if (wave) return false;
    for (int w = 1; w < kWaveTopThreads / 64; ++w) {
        top.join((lds_key *)sh.lists[w], sh.count[w]);
        if (REST && lane == 0) top.rest = join(top.rest, sh.rest[w], top.c2);
    }
    if (top.count > top.most()) top.shrink(top.k, top.most());
    return true;
}
// Every lane brings the largest score it has seen
template <bool REST> __device__ inline void agree(WaveTop<REST> &top, TopShared &sh, float seen)
{
    const int lane = threadIdx.x & 63;
    sh.seen[threadIdx.x] = seen;
    __syncthreads();
    float m[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) m[u] = sh.seen[lane + 64 * u];
    top.foresee(m);
}

template <bool REST, typename T>
__device__ inline bool top_of_part(WaveTop<REST> &top, TopShared &sh, const T *p, long long sc, int begin, int end)
{
    const int wave = threadIdx.x >> 6;
    constexpr int step = 64 * kVec<T>;
    // three waves take whole steps, the last one what is left
    const int even = (end - begin) / 4 / step * step, quarter = even ? even : step;
    const int from = min(end, begin + wave * quarter), to = wave == 3 ? end : min(end, from + quarter);
    if (sc == 1 && even) {
        float m[4];
        WaveTop<REST>::look(p, from, min(even / step, 8), m);
        agree(top, sh, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    }
    top.stream(p, sc, from, to);
    return join_waves(top, sh);
}

// ... of the keys that parts of a row left (0: none)
template <bool REST> __device__ inline bool top_of_keys(WaveTop<REST> &top, TopShared &sh, const uint64_t *keys, int n)
{
    uint64_t best = 0;
    for (int i = threadIdx.x; i < n; i += 8 * kWaveTopThreads) {
        uint64_t key[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = i + u * kWaveTopThreads < n ? keys[i + u * kWaveTopThreads] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) best = key[u] > best ? key[u] : best;
    }
    agree(top, sh, best ? rank_score(best) : -INFINITY);
    const int wave = threadIdx.x >> 6, quarter = (n + 3) / 4;
    const int from = min(n, wave * quarter), to = min(n, from + quarter);
    top.join(keys + from, to - from);
    return join_waves(top, sh);
}

// Parts a row is cut into: enough workgroups for the card (four on each of 256 CUs), at least kPartLabels labels each
constexpr int kPartLabels = 2048;
__host__ __device__ inline int top_part_labels(int C, int parts) { return (((C + parts - 1) / parts) + 511) & ~511; }
inline int top_parts(unsigned rows, int C)
{
    const unsigned most = (unsigned)(C / kPartLabels), want = (1024 + rows - 1) / rows;
    const unsigned n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}
// One wave per row does where rows are short, or many and not long
inline bool row_per_wave(unsigned rows, int C) { return C < kPartLabels || (C < 8192 && rows > 1024); }

}  // namespace mfl_scores

#endif
