// Selection of a beam-search step: the best continuations of every group of beams over (beam, token).
//
//   score(b, v) = run[b] + (x[b, v] - m_b) - log sum_u exp(x[b, u] - m_b)          m_b: a reference, the largest logit seen
//
// One pass over the logits: a wave walks a piece of one beam's row and keeps its n best logits (order within a beam needs no
// normalisation) beside the row's running sum of exponentials; a second kernel, a workgroup a group of beams, joins the
// sums, scores what the waves kept and ranks it.  Ties go to the lowest (beam, token), but tokens of one beam are told apart by
// their logits throughout: where a logit is so large that the scores of the others are one number in float64, the waves could not
// keep the lowest of these.
//
// The order of candidates of different beams hangs on the difference of two logsums, so sums and scores are held in 64
// bits: with sums in float32 two candidates a few 1e-7 apart change places.  The vector unit runs float64 at the rate of
// (unpacked) float32, and the exponential is a polynomial of degree 7.
#include <algorithm>

#include "logit_rows.h"

namespace {

constexpr int BS_WAVES = 4;
constexpr int BS_MAX_N = 64;                                  // candidates a group, beams a group
constexpr int64_t BS_MAX_PLACES = 0x7c000000;                 // beams x vocabulary: a place, and a column a piece behind it, in 32 bits
constexpr int BS_TAKE = 128;                                  // entries that a wave takes from a step
constexpr int BS_GROW = 40;                                   // entries beyond the n best that a list may hold between two steps
constexpr int BS_LIST = 256;                                  // entries of a wave's list: 64 + BS_GROW + BS_TAKE fit

__device__ __forceinline__ uint64_t order64(double f) {
    const uint64_t u = (uint64_t)__double_as_longlong(f);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}

// e^d for -700 <= d <= 600 (below: e^-700, which no sum that holds its own reference notices; NaN too).  2^f on |f| <= 1/2 by the
// polynomial that meets it at the eight Chebyshev points: relative error below 5.6e-11.  The integer part comes out of an
// addition that leaves it in the low bits and goes into the exponent as an integer: 15 instructions.
constexpr double LOG2E = 1.4426950408889634;
__device__ __forceinline__ double exp_sum(double d) {
    constexpr double ROUND = 0x1.8p52;
    d = fmax(d, -700.0);
    const double z = fma(d, LOG2E, ROUND);
    const double f = fma(d, LOG2E, ROUND - z);
    double p = 0x1.00c0e3fcd6d55p-16;
    p = fma(p, f, 0x1.446c79f72370cp-13);
    p = fma(p, f, 0x1.5d87759a0ea3ap-10);
    p = fma(p, f, 0x1.3b29d8bafde6cp-7);
    p = fma(p, f, 0x1.c6b08da70aa5fp-5);
    p = fma(p, f, 0x1.ebfbe0aa03febp-3);
    p = fma(p, f, 0x1.62e42fef9cc7ep-1);
    p = fma(p, f, 0x1.ffffffffa7133p-1);
    return __hiloint2double(__double2hiint(p) + (__double2loint(z) << 20), __double2loint(p));
}

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

// A beam that is out of the search: its running score is no finite log probability
__device__ __forceinline__ bool dead_beam(float run) { return !(fabsf(run) < 1e30f); }

struct BeamList {
    float x[BS_LIST];
    int i[BS_LIST];
};

// The n best of a wave's list (entries [0, e), e >= 1) to its front, best first; returns how many there are.  Entries are held one a
// lane (and a second, third, fourth round of them) and compared with every other, which goes round as a scalar.
__device__ __forceinline__ int list_prune(BeamList& l, int e, int n) {
    constexpr int R = BS_LIST / 64;
    const int lane = threadIdx.x & 63;
    wave_fence();
    float x[R];
    int id[R], rank[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int at = min(lane + 64 * k, e - 1);
        x[k] = l.x[at];
        id[k] = l.i[at];
        rank[k] = lane + 64 * k < e ? 0 : BS_LIST;
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
// a third of the instructions that ranking takes.  Where more than BS_GROW / 2 entries are alike there they are ranked.
template <int R>
__device__ __forceinline__ int list_cut(BeamList& l, int e, int n, float& bound) {
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
    if (c > n + BS_GROW / 2) return list_prune(l, e, n);
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

// A wave's list takes every logit above a bound that n logits of its piece are known to reach: first the n-th largest of
// the lanes' maxima of a step (found bit by bit with ballots), later the n-th best entry, which is looked up only when the list has
// grown by some tens (a look-up costs as much as two steps; done after every step that brought an entry, the kernel took more than
// twice as long).
// Bound: the vector unit, beside the stream: 512 x 152064 float32, 16 best of 8 beams, 76 us under the profiler (4.1 TB/s; bf16 logits, half the
// bytes, take 8 us less), of about 7400 vector instructions a wave the exponentials are 4560.  A reference of 0 without its subtraction
// won nothing, the waves of a row that share the best of their bounds through LDS lost 3 us.
template <typename L>
__global__ __launch_bounds__(BS_WAVES * 64) void beam_partial_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                     const float* __restrict__ run, int vocab, int cols, int chunks,
                                                                     int n, float* __restrict__ part_ref,
                                                                     double* __restrict__ part_sum, float* __restrict__ cand_x,
                                                                     int* __restrict__ cand_tok) {
    constexpr int VEC = L::VEC, BS_VECS = L::VECS, E = BS_VECS * VEC, STEP = 64 * E;
    __shared__ BeamList lists[BS_WAVES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int chunk = blockIdx.x * BS_WAVES + w, row = blockIdx.y;
    if (chunk >= chunks) return;                              // no workgroup barrier below
    BeamList& list = lists[w];
    const uint8_t* base = (const uint8_t*)logits + row * row_stride * L::BYTES;
    // columns are counted from the 16-byte boundary at or before the row's start, `mis` elements in front of it
    const int mis = (int)(((uintptr_t)base & 15) / L::BYTES);
    const int v_end = vocab + mis;
    const int c0 = chunk * cols, c1 = min(c0 + cols, v_end);
    const int64_t pc = (int64_t)row * chunks + chunk;
    if (dead_beam(run[row])) {                                // every candidate scores -inf: the lowest tokens
        const int tok = max(c0 - mis, 0) + lane;
        if (lane < n) {
            const bool on = tok < c1 - mis;
            cand_x[pc * n + lane] = -INFINITY;
            cand_tok[pc * n + lane] = on ? tok : -1;
        }
        if (lane == 0) {
            part_ref[pc] = -INFINITY;
            part_sum[pc] = 0.0;
        }
        return;
    }
    float thr = -INFINITY, ref = 0.f;
    bool full = false;                                        // n logits at or above thr were seen
    int count = 0;                                            // entries of the list
    bool has = false;                                         // a finite logit was seen: ref is one
    double sum = 0.0;

    // A step's logits as stored, loaded one step ahead.  Always as many loads, from whole vectors inside the row (a row without one
    // reads the workspace): paths with different loads would make the compiler wait for them where the paths join.  What lies outside
    // the piece, or in a vector that is only partly inside the row, is put right where the step is unpacked.
    u32x4 raw[BS_VECS];
    const int in0 = mis ? VEC : 0, in1 = v_end / VEC * VEC - VEC;
    const uint8_t* vec0 = in1 >= in0 ? base - (int64_t)mis * L::BYTES : (const uint8_t*)part_sum;
    const int lo = in1 >= in0 ? in0 : 0, hi = in1 >= in0 ? in1 : 0;
    auto whole = [&](int v0) { return v0 >= mis && v0 + STEP <= c1; };     // uniform
    auto load = [&](int v0) {
        if (whole(v0)) {
            const uint8_t* at = base + (int64_t)(v0 - mis) * L::BYTES;         // uniform
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u) raw[u] = __builtin_nontemporal_load((const u32x4*)(at + (uint32_t)(1024 * u + 16 * lane)));
        } else {
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u) {
                const int v = min(max(v0 + (u * 64 + lane) * VEC, lo), hi);
                raw[u] = __builtin_nontemporal_load((const u32x4*)(vec0 + (int64_t)v * L::BYTES));
            }
        }
    };
    load(c0);
    for (int v0 = c0; v0 < c1; v0 += STEP) {
        float f[E];
#pragma unroll
        for (int u = 0; u < BS_VECS; ++u) L::unpack(raw[u], f + u * VEC);
        if (!whole(v0)) {
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u) {
                const int v = v0 + (u * 64 + lane) * VEC;
                if (!(v >= mis && v + VEC <= c1))
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        f[u * VEC + e] = v + e >= mis && v + e < c1 ? L::at(base, v + e - mis) : -INFINITY;
            }
        }
        load(v0 + STEP);                                      // on its way behind this step's work
        float mx4[E / 4], mx = -INFINITY;                     // of four logits, of all
#pragma unroll
        for (int k = 0; k < E / 4; ++k) {
            mx4[k] = fmaxf(fmaxf(f[4 * k], f[4 * k + 1]), fmaxf(f[4 * k + 2], f[4 * k + 3]));
            mx = fmaxf(mx, mx4[k]);
        }
        if (__ballot(mx == INFINITY)) {                       // +inf counts as the largest finite value
#pragma unroll
            for (int k = 0; k < E; ++k) f[k] = f[k] == INFINITY ? 3.402823466e38f : f[k];
            mx = mx == INFINITY ? 3.402823466e38f : mx;
#pragma unroll
            for (int k = 0; k < E / 4; ++k) mx4[k] = mx4[k] == INFINITY ? 3.402823466e38f : mx4[k];
        }
        // ---- the sum: the reference of a lane moves when a logit would leave the range of a double.  (Their difference: the sum ref + 600
        // may round up to a logit that is a step of 1024 away.)
        const bool moves = mx > -INFINITY && (!has || mx - ref > 600.f);
        if (__ballot(moves)) {
            if (moves) {
                sum = has ? sum * exp_sum((double)ref - (double)mx) : 0.0;
                ref = mx;
                has = true;
            }
        }
        const double r = (double)ref;
#pragma unroll
        for (int k = 0; k < E; ++k) sum += exp_sum((double)f[k] - r);

        // ---- the list
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
            if (!full || reach > BS_TAKE) reach = at_least(low);
            int ties = full || thr > -INFINITY ? 0 : max(n - reach, 0);        // masked ones, the lowest tokens first
            if (reach > BS_TAKE) {                            // the step's own n-th largest logit
                uint32_t t = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t trial = t | (1u << bit);
                    if (at_least(order32_back(trial)) >= n) t = trial;
                }
                thr = low = order32_back(t) + 0.f;
                if (at_least(low) > BS_TAKE) {                // many alike: the lowest tokens of them too
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
            for (int u = 0; u < BS_VECS && ties > 0; ++u) {
                const int v = v0 + (u * 64 + lane) * VEC;
                int c = 0;
                bool tie[VEC];
#pragma unroll
                for (int q = 0; q < VEC; ++q) {
                    float fq = f[q];
#pragma unroll
                    for (int uu = 1; uu < BS_VECS; ++uu) fq = u == uu ? f[uu * VEC + q] : fq;
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
        if (count > n + BS_GROW) {
            count = count <= 128 ? list_cut<2>(list, count, n, thr) : list_cut<BS_LIST / 64>(list, count, n, thr);
            full = true;
        }
    }
    if (count > n) count = list_cut<2>(list, count, n, thr);  // no more than n + BS_GROW here
    if (count) count = list_prune(list, count, n);
    // ---- the wave's sum, and what it kept
    float m = has ? ref : -INFINITY;
    m = wave_max(m);
    double s = has ? sum * exp_sum((double)ref - (double)m) : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) {
        part_ref[pc] = m;
        part_sum[pc] = s;
    }
    if (lane < n) {
        cand_x[pc * n + lane] = lane < count ? list.x[lane] : -INFINITY;
        cand_tok[pc * n + lane] = lane < count ? list.i[lane] : -1;
    }
}

// Joins the pieces of a group's beams and ranks their candidates.  What bounds it: a chain of dependent reads and reductions, a
// workgroup a group (64 groups of 8 beams, 16 candidates: a call takes 84 us with the entries ranked by sixteen lanes each and a bound of 20
// bits, 90 with a lane each and all 32).  HELD: the candidates fit the registers, and are read once, beside the pieces' sums.
constexpr int BJ_THREADS = 1024;
constexpr int BJ_WAVES = BJ_THREADS / 64;
constexpr int BJ_HELD = 4;                                    // candidates a thread
constexpr int BJ_LIST = 1024;
template <bool HELD>
__global__ __launch_bounds__(BJ_THREADS) void beam_join_kernel(const float* __restrict__ part_ref, const double* __restrict__ part_sum,
                                                               const float* __restrict__ cand_x, const int* __restrict__ cand_tok,
                                                               const float* __restrict__ run, int beams, int vocab, int chunks, int n,
                                                               int eos, float* __restrict__ scores, int* __restrict__ out_beam,
                                                               int* __restrict__ out_tok, float* __restrict__ next_scores,
                                                               int* __restrict__ next_rows, int* __restrict__ next_tok) {
    __shared__ double s_m[BS_MAX_N], s_log[BS_MAX_N];         // per beam: reference, log of the sum
    __shared__ float s_run[BS_MAX_N];
    __shared__ double l_score[BJ_LIST];
    __shared__ int l_at[BJ_LIST];
    __shared__ float l_x[BJ_LIST];
    __shared__ double best_score[BS_MAX_N];
    __shared__ int best_at[BS_MAX_N];
    __shared__ uint64_t w_key[BJ_WAVES];
    __shared__ uint32_t w_bound[BJ_WAVES];
    __shared__ int w_at[BJ_WAVES];
    __shared__ float w_x[BJ_WAVES];
    __shared__ int s_count;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int per_beam = chunks * n, all = beams * per_beam;
    const int64_t first = (int64_t)g * all;
    float hx[BJ_HELD];
    int ht[BJ_HELD];
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < BJ_HELD; ++c) {
            const int i = tid + c * BJ_THREADS;
            ht[c] = i < all ? cand_tok[first + i] : -1;
            hx[c] = i < all ? cand_x[first + i] : 0.f;
        }
    }
    for (int b = w; b < beams; b += BJ_WAVES) {
        const int64_t p0 = ((int64_t)g * beams + b) * chunks;  // at most 64 pieces: one a lane
        const float r = lane < chunks ? part_ref[p0 + lane] : -INFINITY;
        const double ps = lane < chunks ? part_sum[p0 + lane] : 0.0;
        const float m = wave_max(r);
        double s = r > -INFINITY ? ps * exp_sum((double)r - (double)m) : 0.0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0) {
            s_m[b] = m;
            s_log[b] = log(s);
            s_run[b] = run[g * beams + b];
        }
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
    auto score_of = [&](int b, float x) -> double {
        const float r = s_run[b];
        return x == -INFINITY || dead_beam(r) ? -INFINITY : (double)r + (((double)x - s_m[b]) - s_log[b]);
    };
    // candidate i: its place b V + v (-1: none) and score
    auto candidate = [&](int i, double& score) -> int {
        const int tok = cand_tok[first + i];
        if (tok < 0) return -1;
        const int b = i / per_beam;
        score = score_of(b, cand_x[first + i]);
        return b * vocab + tok;
    };
    double hs[BJ_HELD];
    int ha[BJ_HELD];
    // A bound that at least n candidates reach: the largest of the waves' n-th largest lane maxima.  Taken on scores rounded to
    // float32, which keep their order.
    uint32_t key = 0;
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < BJ_HELD; ++c) {
            ha[c] = -1;
            if (ht[c] >= 0) {
                const int b = (tid + c * BJ_THREADS) / per_beam;
                hs[c] = score_of(b, hx[c]);
                ha[c] = b * vocab + ht[c];
                key = max(key, order32((float)hs[c] + 0.f));
            }
        }
    } else {
        for (int i = tid; i < all; i += BJ_THREADS) {
            double s;
            if (candidate(i, s) >= 0) key = max(key, order32((float)s + 0.f));
        }
    }
    uint32_t t = 0;
    for (int bit = 31; bit >= 12; --bit) {                    // a lower bound does as well: the last bits keep few candidates away
        const uint32_t trial = t | (1u << bit);
        if (__popcll(__ballot(key >= trial)) >= n) t = trial;
    }
    if (lane == 0) w_bound[w] = t;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BJ_WAVES; ++i) t = max(t, w_bound[i]);
    auto keep = [&](double s, float x, int at) {
        if (order32((float)s + 0.f) >= t) {
            const int p = atomicAdd(&s_count, 1);
            if (p < BJ_LIST) {
                l_score[p] = s;
                l_at[p] = at;
                l_x[p] = x;
            }
        }
    };
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < BJ_HELD; ++c)
            if (ha[c] >= 0) keep(hs[c], hx[c], ha[c]);
    } else {
        for (int i = tid; i < all; i += BJ_THREADS) {
            double s;
            const int at = candidate(i, s);
            if (at >= 0) keep(s, cand_x[first + i], at);
        }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= BJ_LIST) {
        for (int i0 = 0; i0 < count; i0 += BJ_THREADS / 16) { // sixteen lanes an entry
            const int i = min(i0 + tid / 16, count - 1);
            const double s = l_score[i];
            const int at = l_at[i];
            int rank = 0;
            for (int j = tid & 15; j < count; j += 16) {
                rank += l_score[j] > s;
                if (l_score[j] == s && j != i) {              // rare
                    const int aj = l_at[j], bi = at / vocab, bj = aj / vocab;
                    const float x = l_x[i], xj = l_x[j];
                    rank += bj < bi || (bj == bi && (xj > x || (xj == x && aj < at)));
                }
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) rank += __shfl_xor(rank, o, 64);
            if (rank < n) {                                   // (lanes of one entry, and those past the last, write the same)
                best_score[rank] = s;
                best_at[rank] = at;
            }
        }
        __syncthreads();
    } else {                                                  // more ties than the list holds: one after the other
        struct Entry {
            uint64_t k;
            float x;
            int at;
        };
        auto before = [&](const Entry& a, const Entry& b) -> bool {
            if (a.k != b.k) return a.k > b.k;
            const int ba = a.at / vocab, bb = b.at / vocab;
            return ba != bb ? ba < bb : (a.x != b.x ? a.x > b.x : a.at < b.at);
        };
        Entry last = {~0ull, 0.f, 0};                         // no score has this key
        for (int r = 0; r < n; ++r) {
            Entry top = {0, 0.f, 0x7fffffff};
            for (int i = tid; i < all; i += BJ_THREADS) {
                double s;
                const int c = candidate(i, s);
                if (c < 0) continue;
                const Entry e = {order64(s), cand_x[first + i], c};
                if (before(last, e) && before(e, top)) top = e;
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const Entry e = {__shfl_xor((unsigned long long)top.k, o, 64), __shfl_xor(top.x, o, 64), __shfl_xor(top.at, o, 64)};
                if (before(e, top)) top = e;
            }
            __syncthreads();
            if (lane == 0) {
                w_key[w] = top.k;
                w_x[w] = top.x;
                w_at[w] = top.at;
            }
            __syncthreads();
            for (int i = 0; i < BJ_WAVES; ++i) {
                const Entry e = {w_key[i], w_x[i], w_at[i]};
                if (before(e, top)) top = e;
            }
            last = top;
            if (tid == 0) {
                best_score[r] = __longlong_as_double((long long)((top.k >> 63) ? top.k ^ 0x8000000000000000ull : ~top.k));
                best_at[r] = top.at;
            }
        }
        __syncthreads();
    }
    if (w) return;
    const bool on = lane < n;
    const int at = on ? best_at[lane] : 0;
    const float s = on ? (float)best_score[lane] : 0.f;       // rounded once, to the type of the running scores
    const int b = at / vocab, tok = at - b * vocab;
    if (on) {
        scores[(int64_t)g * n + lane] = s;
        out_beam[(int64_t)g * n + lane] = b;
        out_tok[(int64_t)g * n + lane] = tok;
    }
    const bool goes_on = on && tok != eos;
    const uint64_t m = __ballot(goes_on);
    const int place = __popcll(m & ((1ull << lane) - 1ull));
    if (goes_on && place < beams) {
        next_scores[(int64_t)g * beams + place] = s;
        next_rows[(int64_t)g * beams + place] = g * beams + b;
        next_tok[(int64_t)g * beams + place] = tok;
    }
}

// Columns of a row that a wave walks: about 4096 waves where there is that much to read, at least 1024 columns and at most as many as give a
// row 64 pieces (the join reads n candidates of each).
int beam_cols(int64_t rows, int vocab, int vec) {
    const int64_t span = (int64_t)vocab + vec - 1;
    int64_t cols = std::max<int64_t>(1024, rows * span / 4096);
    cols = std::max(cols, (span + 63) / 64);
    const int64_t step = 64 * 16;                             // logits of a step, of either width
    return (int)(cols > step ? (cols + step - 1) / step * step : (cols + 511) / 512 * 512);
}
struct BeamPlan {
    int cols, chunks;
    size_t sum, ref, x, tok, bytes;
};
BeamPlan beam_plan(int64_t rows, int vocab, int n, int dtype) {
    const int vec = dtype == MF_FP32 ? 4 : 8;
    BeamPlan p;
    p.cols = beam_cols(rows, vocab, vec);
    p.chunks = (vocab + vec - 1 + p.cols - 1) / p.cols;
    const size_t pieces = (size_t)rows * p.chunks;
    p.sum = 0;
    p.ref = p.sum + pieces * 8;
    p.x = p.ref + pieces * 4;
    p.tok = p.x + pieces * n * 4;
    p.bytes = p.tok + pieces * n * 4;
    return p;
}

}  // namespace

extern "C" size_t mf_beam_search_workspace_bytes(int groups, int beams, int vocab, int n, int dtype) {
    if (groups <= 0 || beams <= 0 || vocab <= 0 || n <= 0 || dtype < 0 || dtype > MF_FP32) return 0;
    return beam_plan((int64_t)groups * beams, vocab, n, dtype).bytes;
}

extern "C" int mf_beam_search_select(float* scores, int32_t* beam_ids, int32_t* tokens, float* next_scores, int32_t* next_rows,
                                     int32_t* next_tokens, const void* logits, int64_t row_stride, const float* beam_scores,
                                     int groups, int beams, int vocab, int n, int eos, int dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    MF_REQUIRE(dtype == MF_BF16 || dtype == MF_FP16 || dtype == MF_FP32, "beam_search_select: dtype must be bf16, fp16 or fp32");
    MF_REQUIRE(groups >= 0 && beams > 0 && vocab > 0, "beam_search_select: bad sizes");
    if (groups == 0) return 0;
    MF_REQUIRE(beams <= BS_MAX_N && n > 0 && n <= BS_MAX_N, "beam_search_select: up to %d beams and candidates, got %d and %d", BS_MAX_N,
               beams, n);
    MF_REQUIRE(n >= (eos >= 0 ? 2 : 1) * beams && (int64_t)n <= (int64_t)beams * vocab,
               "beam_search_select: %d candidates of %d beams x %d tokens: at least one a beam (two with an end token) and no more than there are",
               n, beams, vocab);
    MF_REQUIRE((int64_t)groups * beams <= 65535 && (int64_t)beams * vocab <= BS_MAX_PLACES, "beam_search_select: %d x %d beams of %d tokens",
               groups, beams, vocab);
    if (row_stride <= 0) row_stride = vocab;
    MF_REQUIRE(row_stride >= vocab, "beam_search_select: row stride %lld below the vocabulary's %d", (long long)row_stride, vocab);
    MF_REQUIRE(scores && beam_ids && tokens && next_scores && next_rows && next_tokens && logits && beam_scores,
               "beam_search_select: null argument");
    MF_REQUIRE(((uintptr_t)logits & (dtype == MF_FP32 ? 3 : 1)) == 0, "beam_search_select: logits must be aligned to their type");
    const int rows = groups * beams;
    const BeamPlan p = beam_plan(rows, vocab, n, dtype);
    MF_REQUIRE(workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 7) == 0,
               "beam_search_select: 8-byte aligned workspace of %zu bytes needed, %zu given", p.bytes, workspace_bytes);
    uint8_t* ws = (uint8_t*)workspace;
    double* part_sum = (double*)(ws + p.sum);
    float *part_ref = (float*)(ws + p.ref), *cand_x = (float*)(ws + p.x);
    int* cand_tok = (int*)(ws + p.tok);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)((p.chunks + BS_WAVES - 1) / BS_WAVES), (unsigned)rows);
#define BS_LAUNCH(L)                                                                                                        \
    hipLaunchKernelGGL(beam_partial_kernel<L>, grid, dim3(BS_WAVES * 64), 0, st, logits, row_stride, beam_scores, vocab, p.cols, \
                       p.chunks, n, part_ref, part_sum, cand_x, cand_tok)
    if (dtype == MF_FP32) BS_LAUNCH(LogitF32);
    else if (dtype == MF_BF16) BS_LAUNCH(Logit16<BF16>);
    else BS_LAUNCH(Logit16<FP16>);
#undef BS_LAUNCH
    const int rc = MF_LAUNCH_CHECK();
    if (rc) return rc;
#define BJ_LAUNCH(HELD)                                                                                                      \
    hipLaunchKernelGGL(beam_join_kernel<HELD>, dim3(groups), dim3(BJ_THREADS), 0, st, part_ref, part_sum, cand_x, cand_tok, beam_scores, \
                       beams, vocab, p.chunks, n, eos, scores, beam_ids, tokens, next_scores, next_rows, next_tokens)
    if ((int64_t)beams * p.chunks * n <= BJ_HELD * BJ_THREADS) BJ_LAUNCH(true);
    else BJ_LAUNCH(false);
#undef BJ_LAUNCH
    return MF_LAUNCH_CHECK();
}
