// What the kernels share that walk rows of logits: how logits are stored, and a wave's list of the best of them.
#pragma once
#include "common.h"

namespace {

constexpr int LIST_MAX_N = 64;                                // best ones that a list is kept of
constexpr int LIST_TAKE = 128;                                // entries that a wave takes from a step
constexpr int LIST_GROW = 40;                                 // entries beyond the n best that a list may hold between two steps
constexpr int LIST_SIZE = 256;                                // entries of a wave's list: LIST_MAX_N + LIST_GROW + LIST_TAKE fit

// Logits as stored, 16 bytes at a time
struct LogitF32 {
    static constexpr int VEC = 4, BYTES = 4, VECS = 4;        // VECS: 16-byte loads a lane and step
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return ((const float*)p)[i]; }
};
template <typename T>
struct Logit16 {
    static constexpr int VEC = 8, BYTES = 2, VECS = 2;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { unpack8<T>(v, f); }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return T::to_float(((const uint16_t*)p)[i]); }
};

// keys that order as the values do
__device__ __forceinline__ uint32_t order32(float f) {
    const uint32_t u = __float_as_uint(f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order32_back(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// c + set bits of m below this lane's
__device__ __forceinline__ int lanes_before(uint64_t m, int c) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, (uint32_t)c));
}
__device__ __forceinline__ int wave_scan_excl(int v, int& total) {
    const int lane = threadIdx.x & 63;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(incl, o, 64);
        if (lane >= o) incl += t;
    }
    total = __shfl(incl, 63, 64);
    return incl - v;
}

struct LogitList {
    float x[LIST_SIZE];
    int i[LIST_SIZE];
};

// The n best of a wave's list (entries [0, e), e >= 1) to its front, best first; returns how many there are.  Entries are held one a
// lane (and a second, third, fourth round of them) and compared with every other, which goes round as a scalar.
__device__ __forceinline__ int list_prune(LogitList& l, int e, int n) {
    constexpr int R = LIST_SIZE / 64;
    const int lane = threadIdx.x & 63;
    wave_fence();
    float x[R];
    int id[R], rank[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int at = min(lane + 64 * k, e - 1);
        x[k] = l.x[at];
        id[k] = l.i[at];
        rank[k] = lane + 64 * k < e ? 0 : LIST_SIZE;
    }
#pragma unroll
    for (int jr = 0; jr < R; ++jr) {
        const int last = min(64, e - 64 * jr);
        for (int j = 0; j < last; ++j) {
            const float xj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x[jr]), j));
            const int ij = __builtin_amdgcn_readlane(id[jr], j);
            rank[0] += xj > x[0] || (xj == x[0] && ij < id[0]);
            if (e > 64) {
#pragma unroll
                for (int k = 1; k < R; ++k) rank[k] += xj > x[k] || (xj == x[k] && ij < id[k]);
            }
        }
    }
    wave_fence();
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (rank[k] < n) {
            l.x[rank[k]] = x[k];
            l.i[rank[k]] = id[k];
        }
    wave_fence();
    return min(e, n);
}

// The list cut to the entries that reach its n-th best (e >= n), in any order; `bound` is that entry.  Found bit by bit with ballots,
// a third of the instructions that ranking takes.  Where more than LIST_GROW / 2 entries are alike there they are ranked.
template <int R>
__device__ __forceinline__ int list_cut(LogitList& l, int e, int n, float& bound) {
    const int lane = threadIdx.x & 63;
    wave_fence();
    float x[R];
    int id[R];
    uint32_t key[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int at = min(lane + 64 * k, e - 1);
        x[k] = l.x[at] + 0.f;
        id[k] = l.i[at];
        key[k] = lane + 64 * k < e ? order32(x[k]) : 0u;
    }
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = t | (1u << bit);
        int c = 0;
#pragma unroll
        for (int k = 0; k < R; ++k) c += __popcll(__ballot(key[k] >= trial));
        if (c >= n) t = trial;
    }
    bound = order32_back(t);
    int c = 0;
#pragma unroll
    for (int k = 0; k < R; ++k) c += __popcll(__ballot(key[k] >= t));
    if (c > n + LIST_GROW / 2) return list_prune(l, e, n);
    wave_fence();
    c = 0;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const bool keep = key[k] >= t;
        const uint64_t m = __ballot(keep);
        if (keep) {
            const int at = lanes_before(m, c);
            l.x[at] = x[k];
            l.i[at] = id[k];
        }
        c += __popcll(m);
    }
    wave_fence();
    return c;
}

// Takes a step's logits into a wave's list of the n best.  f: the lane's logits, VECS vectors of VEC neighbours, vector u of the step's columns
// v0 + (64 u + lane) VEC on (counted as `mis` says: column v is token v - mis; c1: the end); mx4, mx: the maxima of four and of all of
// them.  thr: a bound that n logits are known to reach once `full`; count: entries of the list.
template <typename L>
__device__ __forceinline__ void list_step(LogitList& list, const float* f, const float* mx4, float mx, int n, int v0, int mis, int c1,
                                          bool& full, float& thr, int& count) {
    constexpr int VEC = L::VEC, VECS = L::VECS, E = VECS * VEC;
    const int lane = threadIdx.x & 63;
    if (!full || __ballot(mx > thr)) {
        auto at_least = [&](float x) {                    // logits of the step that reach x
            int c = 0;
#pragma unroll
            for (int k = 0; k < E; ++k) c += __popcll(__ballot(f[k] >= x));
            return c;
        };
        if (!full) {
            const uint32_t key = order32(mx);
            uint32_t t = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = t | (1u << bit);
                if (__popcll(__ballot(key >= trial)) >= n) t = trial;
            }
            thr = order32_back(t) + 0.f;                  // (no negative zero: the values next to thr are found by its key)
        }
        // The lowest logit that is taken: above thr, at it while fewer than n are known, and no masked one.
        float low = full || thr == -INFINITY ? order32_back(order32(thr) + 1) : thr;
        // (a few lanes cannot hold too many)
        int reach = E * __popcll(__ballot(mx >= low));
        if (!full || reach > LIST_TAKE) reach = at_least(low);
        int ties = full || thr > -INFINITY ? 0 : max(n - reach, 0);        // masked ones, the lowest tokens first
        if (reach > LIST_TAKE) {                            // the step's own n-th largest logit
            uint32_t t = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = t | (1u << bit);
                if (at_least(order32_back(trial)) >= n) t = trial;
            }
            thr = low = order32_back(t) + 0.f;
            if (at_least(low) > LIST_TAKE) {                // many alike: the lowest tokens of them too
                low = order32_back(order32(thr) + 1);
                ties = n - at_least(low);
            }
        }
        full = ties == 0 || thr > -INFINITY;
#pragma unroll
        for (int k4 = 0; k4 < E; k4 += 4) {
            if (!__ballot(mx4[k4 / 4] >= low)) continue;
#pragma unroll
            for (int k = k4; k < k4 + 4; ++k) {
                const uint64_t m = __ballot(f[k] >= low);
                if (!m) continue;
                if (f[k] >= low) {
                    const int at = lanes_before(m, count);
                    list.x[at] = f[k];
                    list.i[at] = lane * VEC - mis + (v0 + (k / VEC) * 64 * VEC + k % VEC);
                }
                count += __popcll(m);
            }
        }
        // logits at thr in the order of the tokens; of masked ones, -inf and NaN, which counts as it
        for (int u = 0; u < VECS && ties > 0; ++u) {
            const int v = v0 + (u * 64 + lane) * VEC;
            int c = 0;
            bool tie[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                float fq = f[q];
#pragma unroll
                for (int uu = 1; uu < VECS; ++uu) fq = u == uu ? f[uu * VEC + q] : fq;
                tie[q] = v + q >= mis && v + q < c1 && (thr == -INFINITY ? !(fq > thr) : fq == thr);
                c += tie[q];
            }
            int all;
            int pos = wave_scan_excl(c, all);
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                if (tie[q]) {
                    if (pos < ties) {
                        list.x[count + pos] = thr;
                        list.i[count + pos] = v + q - mis;
                    }
                    ++pos;
                }
            all = min(all, ties);
            count += all;
            ties -= all;
        }
        full = full || ties == 0;                         // masked logits may have filled it
    }
    if (count > n + LIST_GROW) {
        count = count <= 128 ? list_cut<2>(list, count, n, thr) : list_cut<LIST_SIZE / 64>(list, count, n, thr);
        full = true;
    }
}

}  // namespace
