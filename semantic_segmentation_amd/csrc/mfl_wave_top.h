// The k <= 128 largest scores of a run of labels, by one wave in one pass (mfl_top_labels.hip, mfl_sample_labels.hip).
//
// The wave keeps a list of candidates in LDS, as rank keys, and a bound below which no label can be among the k best any
// more.  A vector of scores with none above the bound costs a maximum and a compare; scores above it are appended.  When
// the list is full, a binary search over the keys (held in registers, eight a lane, counted by ballots) finds a bound that
// leaves between k and about 2 k of them, and the others leave.  For scores in random order about k ln(C / 512) of C labels
// are appended at all; for rising ones every label is, at one search per few hundred.  Everything that never enters or
// leaves the list goes into the rest's running sum exactly once.  Appending follows the order of the labels and every count
// is the wave's own: no atomics, the same result every time.
#ifndef MFL_WAVE_TOP_H
#define MFL_WAVE_TOP_H

#include "mfl_scores.h"

namespace mfl_scores {

constexpr int kWaveTopThreads = 256;
constexpr int kListKeys = 512;
constexpr int kListRegs = kListKeys / 64;

template <bool REST> struct WaveTop {
    uint64_t *list;             // LDS, kListKeys, this wave's own
    int k, count;
    uint64_t bound;             // keys up to it are out
    float bound_score;
    float c2;
    LogSum rest;                // this lane's share

    __device__ WaveTop(uint64_t *list, int k, float c2)
        : list(list), k(k), count(0), bound(0), bound_score(-INFINITY), c2(c2), rest{-INFINITY, 0.f} {}

    // Leaves between `least` (<= count) and `most` keys in the list
    __device__ void shrink(int least, int most)
    {
        const int lane = threadIdx.x & 63;
        uint64_t r[kListRegs];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kListRegs; ++i) r[i] = lane + 64 * i < count ? list[lane + 64 * i] : 0;
        uint64_t lo = bound, hi = ~0ull;            // more than `most` above lo, fewer than `least` above hi
        uint64_t mid;
        for (;;) {
            mid = lo + (hi - lo) / 2;               // (keys differ: least = most is always met)
            int above = 0;
#pragma unroll
            for (int i = 0; i < kListRegs; ++i) above += __popcll(__ballot(r[i] > mid));
            if (above > most) lo = mid;
            else if (above < least) hi = mid;
            else break;
            if (hi - lo <= 1) {                     // (the key ~0, a NaN on label 0, is above nothing: keep from it on)
                mid = lo;
                break;
            }
        }
        count = 0;
#pragma unroll
        for (int i = 0; i < kListRegs; ++i) {
            const bool stay = r[i] > mid;
            const uint64_t who = __ballot(stay);
            if (stay) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = r[i];
            count += __popcll(who);
            if (REST && !stay && r[i]) add_score(rest, rank_score(r[i]), c2);
        }
        bound = mid;
        bound_score = rank_score(mid);
        __builtin_amdgcn_wave_barrier();
    }
    __device__ int most() const { return k < 64 ? 2 * k + 32 : k + k / 2; }

    // Appends the keys of the lanes that bring one; returns whether this lane's went in
    __device__ bool append(uint64_t key, bool bring)
    {
        bring = bring && key > bound;
        uint64_t who = __ballot(bring);
        if (!who) return false;
        if (count + __popcll(who) > kListKeys) {
            shrink(k, most());
            bring = bring && key > bound;
            who = __ballot(bring);
        }
        if (bring) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key;
        count += __popcll(who);
        return bring;
    }

    template <int V> __device__ void take(float (&x)[V], int c, int end)
    {
        float m = x[0];
#pragma unroll
        for (int i = 1; i < V; ++i) m = max_or_nan(m, x[i]);
        // (a NaN is not below the bound either)
        if (__any(!(m < bound_score))) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (append(rank_key(score_key(x[i]), c + i), c + i < end)) x[i] = -INFINITY;
        }
        if (REST) {
            float top = rest.m;
#pragma unroll
            for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
            const float ref = finite_or_zero(top);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += __builtin_amdgcn_exp2f((x[i] - ref) * c2);
            rest = {top, fmaf(rest.s, __builtin_amdgcn_exp2f((rest.m - ref) * c2), sum)};
        }
    }

    // Labels begin .. end of a row at p
    template <typename T> __device__ void stream(const T *p, long long sc, int begin, int end)
    {
        constexpr int V = kVec<T>;
        const int lane = threadIdx.x & 63;
        if (sc == 1) {
            constexpr int U = 4;                    // vectors in flight
            int c = begin;
            for (; c + U * 64 * V <= end; c += U * 64 * V) {
                float x[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u) load_vec(p + c + (u * 64 + lane) * V, x[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) take(x[u], c + (u * 64 + lane) * V, end);
            }
            for (; c < end; c += 64 * V) {
                const int at = c + lane * V;
                float x[V];
                if (at + V <= end) {
                    load_vec(p + at, x);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) x[i] = at + i < end ? to_float(p[at + i]) : -INFINITY;
                }
                take(x, at, end);
            }
        } else {
            for (int c = begin; c < end; c += 64) {
                float x[1] = {c + lane < end ? to_float(p[(c + lane) * sc]) : -INFINITY};
                take(x, c + lane, end);
            }
        }
    }

    // Keys that other waves found (0: none)
    __device__ void join(const uint64_t *keys, int n)
    {
        const int lane = threadIdx.x & 63;
        for (int i = 0; i < n; i += 64) {
            const uint64_t key = i + lane < n ? keys[i + lane] : 0;
            const bool in = append(key, key != 0);
            if (REST && !in && key) add_score(rest, rank_score(key), c2);
        }
    }

    // Down to the k best
    __device__ void cut()
    {
        if (count > k) shrink(k, k);
    }

    // f(rank, key) for each of the list's keys (at most 128), by counting what is above it
    template <typename F> __device__ void ranked(F f) const
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
        if (a) f(above_a, a);
        if (b) f(above_b, b);
    }
};

// Parts a row is cut into: enough waves for the card (16 on each of 256 CUs), at least 2048 labels each
__host__ __device__ inline int top_part_labels(int C, int parts) { return (((C + parts - 1) / parts) + 511) & ~511; }
inline int top_parts(unsigned rows, int C)
{
    const unsigned most = (unsigned)((C + 2047) / 2048), want = (4096 + rows - 1) / rows;
    const unsigned n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}

}  // namespace mfl_scores

#endif
