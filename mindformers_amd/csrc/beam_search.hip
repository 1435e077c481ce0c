// Selection of a beam-search step: the best continuations of every group of beams over (beam, token).
//
//   score(b, v) = run[b] + (x[b, v] - m_b) - log sum_u exp(x[b, u] - m_b)          m_b: a reference, the largest logit seen
//
// One pass over the logits: a wave walks a piece of one beam's row and keeps its n best logits (order within a beam needs no
// normalisation) beside the row's running sum of exponentials; a second kernel, a workgroup a group of beams, joins the
// sums, scores what the waves kept and ranks it.  Ties go to the lowest (beam, token).
//
// The order of candidates of different beams hangs on the difference of two logsums, so sums and scores are held in 64
// bits: with sums in float32 two candidates a few 1e-7 apart change places.  The vector unit runs float64 at the rate of
// (unpacked) float32, and the exponential is a polynomial of degree 7, about 15 instructions a logit.
#include <algorithm>

#include "common.h"

namespace {

constexpr int BS_WAVES = 4;
constexpr int BS_MAX_N = 64;                                  // candidates a group, beams a group
constexpr int BS_APPEND = 192;                                // new entries that a wave takes beside its list at a time
constexpr int BS_LIST = BS_MAX_N + BS_APPEND;
constexpr int BS_VECS = 4;                                    // 16-byte loads a lane and step

// Logits as stored, 16 bytes at a time
struct LogitF32 {
    static constexpr int VEC = 4, BYTES = 4;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return ((const float*)p)[i]; }
};
template <typename T>
struct Logit16 {
    static constexpr int VEC = 8, BYTES = 2;
    static __device__ __forceinline__ void unpack(const u32x4& v, float* f) { unpack8<T>(v, f); }
    static __device__ __forceinline__ float at(const void* p, int64_t i) { return T::to_float(((const uint16_t*)p)[i]); }
};

// keys that order as the values do
__device__ __forceinline__ uint32_t order32(float f) {
    const uint32_t u = __float_as_uint(f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order32_back(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t order64(double f) {
    const uint64_t u = (uint64_t)__double_as_longlong(f);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}

// 2^t for t <= 1000 (below -1074: 0).  2^f on |f| <= 1/2 by the polynomial that meets it at the eight Chebyshev points: relative error
// below 5.6e-11.
__device__ __forceinline__ double exp2_sum(double t) {
    t = fmax(t, -1100.0);                                     // also for NaN
    const double n = rint(t), f = t - n;
    double p = 0x1.00c0e3fcd6d55p-16;
    p = fma(p, f, 0x1.446c79f72370cp-13);
    p = fma(p, f, 0x1.5d87759a0ea3ap-10);
    p = fma(p, f, 0x1.3b29d8bafde6cp-7);
    p = fma(p, f, 0x1.c6b08da70aa5fp-5);
    p = fma(p, f, 0x1.ebfbe0aa03febp-3);
    p = fma(p, f, 0x1.62e42fef9cc7ep-1);
    p = fma(p, f, 0x1.ffffffffa7133p-1);
    return ldexp(p, (int)n);
}
constexpr double LOG2E = 1.4426950408889634;

__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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

// The n best of a wave's list (entries [0, e)) to its front, best first.
__device__ __forceinline__ int list_prune(BeamList& l, int e, int n) {
    const int lane = threadIdx.x & 63;
    wave_fence();
    float x[BS_LIST / 64];
    int id[BS_LIST / 64], rank[BS_LIST / 64];
#pragma unroll
    for (int k = 0; k < BS_LIST / 64; ++k) {
        const int at = min(lane + 64 * k, e - 1);
        x[k] = l.x[at];
        id[k] = l.i[at];
        rank[k] = lane + 64 * k < e ? 0 : BS_LIST;
    }
    for (int j = 0; j < e; ++j) {
        const float xj = l.x[j];
        const int ij = l.i[j];
#pragma unroll
        for (int k = 0; k < BS_LIST / 64; ++k) rank[k] += xj > x[k] || (xj == x[k] && ij < id[k]);
    }
    wave_fence();
#pragma unroll
    for (int k = 0; k < BS_LIST / 64; ++k)
        if (rank[k] < n) {
            l.x[rank[k]] = x[k];
            l.i[rank[k]] = id[k];
        }
    wave_fence();
    return min(e, n);
}

template <typename L>
__global__ __launch_bounds__(BS_WAVES * 64) void beam_partial_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                     const float* __restrict__ run, int vocab, int cols, int chunks,
                                                                     int n, float* __restrict__ part_ref,
                                                                     double* __restrict__ part_sum, float* __restrict__ cand_x,
                                                                     int* __restrict__ cand_tok) {
    constexpr int VEC = L::VEC, E = BS_VECS * VEC, STEP = 64 * E;
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
    int count = 0;
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
    bool has = false;                                         // a finite logit was seen: ref is one
    double sum = 0.0;
    for (int v0 = c0; v0 < c1; v0 += STEP) {
        float f[E];
        const bool whole = v0 >= mis && v0 + STEP <= c1;      // uniform
        if (whole) {
            u32x4 raw[BS_VECS];
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u)
                raw[u] = __builtin_nontemporal_load((const u32x4*)(base + (int64_t)(v0 - mis + (u * 64 + lane) * VEC) * L::BYTES));
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u) L::unpack(raw[u], f + u * VEC);
        } else {
#pragma unroll
            for (int u = 0; u < BS_VECS; ++u) {
                const int v = v0 + (u * 64 + lane) * VEC;
                if (v >= mis && v + VEC <= c1) {
                    const u32x4 raw = __builtin_nontemporal_load((const u32x4*)(base + (int64_t)(v - mis) * L::BYTES));
                    L::unpack(raw, f + u * VEC);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        f[u * VEC + e] = v + e >= mis && v + e < c1 ? L::at(base, v + e - mis) : -INFINITY;
                }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < E; ++k) mx = fmaxf(mx, f[k]);
        if (__ballot(mx == INFINITY)) {                       // +inf counts as the largest finite value
#pragma unroll
            for (int k = 0; k < E; ++k) f[k] = f[k] == INFINITY ? 3.402823466e38f : f[k];
            mx = mx == INFINITY ? 3.402823466e38f : mx;
        }
        // ---- the sum: the reference of a lane moves when a logit would leave the range of a double
        const bool moves = mx > -INFINITY && (!has || mx > ref + 600.f);
        if (__ballot(moves)) {
            if (moves) {
                sum = has ? sum * exp2_sum(((double)ref - mx) * LOG2E) : 0.0;
                ref = mx;
                has = true;
            }
        }
#pragma unroll
        for (int k = 0; k < E; ++k) sum += exp2_sum(((double)f[k] - (double)ref) * LOG2E);

        // ---- the list
        const bool full = count == n;
        if (full && !__ballot(mx > thr)) continue;
        float least = thr;                                    // entries are the logits above it (and, while the list fills, some at it)
        auto more = [&]() {
            int c = 0;
#pragma unroll
            for (int k = 0; k < E; ++k) c += f[k] > least;
            return c;
        };
        if (!full) {                                          // the n-th largest of the lanes' maxima
            const uint32_t key = order32(mx);
            uint32_t t = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = t | (1u << bit);
                if (__popcll(__ballot(key >= trial)) >= n) t = trial;
            }
            least = order32_back(t);
        }
        int mine = more(), total;
        int at = wave_scan_excl(mine, total);
        int ties = full ? 0 : max(n - total, 0);
        if (total > BS_APPEND) {                              // the step's n-th largest logit itself
            uint32_t t = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = t | (1u << bit);
                int c = 0;
#pragma unroll
                for (int k = 0; k < E; ++k) c += order32(fmaxf(f[k], -INFINITY)) >= trial;   // NaN counts as -inf
                int all;
                (void)wave_scan_excl(c, all);
                if (all >= n) t = trial;
            }
            least = order32_back(t);
            mine = more();
            at = wave_scan_excl(mine, total);
            ties = n - total;
        }
        at += count;
        if (mine) {
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (f[k] > least) {
                    list.x[at] = f[k];
                    list.i[at] = v0 + ((k / VEC) * 64 + lane) * VEC + k % VEC - mis;
                    ++at;
                }
        }
        int e = count + total;
        // logits at the bound, in the order of the tokens (masked ones are all alike: -inf, and NaN, which counts as it)
        for (int u = 0; u < BS_VECS && ties > 0; ++u) {
            const int v = v0 + (u * 64 + lane) * VEC;
            int c = 0;
            bool tie[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) {
                float fq = f[q];
#pragma unroll
                for (int uu = 1; uu < BS_VECS; ++uu) fq = u == uu ? f[uu * VEC + q] : fq;
                tie[q] = v + q >= mis && v + q < c1 && (least == -INFINITY ? !(fq > least) : fq == least);
                c += tie[q];
            }
            int all;
            int pos = wave_scan_excl(c, all);
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                if (tie[q]) {
                    if (pos < ties) {
                        list.x[e + pos] = least;
                        list.i[e + pos] = v + q - mis;
                    }
                    ++pos;
                }
            all = min(all, ties);
            e += all;
            ties -= all;
        }
        if (e > count) {
            count = list_prune(list, e, n);
            if (count == n) thr = list.x[n - 1];
        }
    }
    // ---- the wave's sum, and what it kept
    float m = has ? ref : -INFINITY;
    m = wave_max(m);
    double s = has ? sum * exp2_sum(((double)ref - (double)m) * LOG2E) : 0.0;
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

// Joins the pieces of a group's beams and ranks their candidates.
constexpr int BJ_THREADS = 256;
constexpr int BJ_LIST = 1024;
__global__ __launch_bounds__(BJ_THREADS) void beam_join_kernel(const float* __restrict__ part_ref, const double* __restrict__ part_sum,
                                                               const float* __restrict__ cand_x, const int* __restrict__ cand_tok,
                                                               const float* __restrict__ run, int beams, int vocab, int chunks, int n,
                                                               int eos, float* __restrict__ scores, int* __restrict__ out_beam,
                                                               int* __restrict__ out_tok, float* __restrict__ next_scores,
                                                               int* __restrict__ next_rows, int* __restrict__ next_tok) {
    __shared__ double s_m[BS_MAX_N], s_log[BS_MAX_N];         // per beam: reference, log of the sum
    __shared__ double l_score[BJ_LIST];
    __shared__ int l_at[BJ_LIST];
    __shared__ double best_score[BS_MAX_N];
    __shared__ int best_at[BS_MAX_N];
    __shared__ uint64_t w_key[BJ_THREADS / 64];
    __shared__ int w_at[BJ_THREADS / 64];
    __shared__ int s_count;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    for (int b = w; b < beams; b += BJ_THREADS / 64) {
        const int64_t p0 = ((int64_t)g * beams + b) * chunks;
        float m = -INFINITY;
        for (int c = lane; c < chunks; c += 64) m = fmaxf(m, part_ref[p0 + c]);
        m = wave_max(m);
        double s = 0.0;
        if (m > -INFINITY)
            for (int c = lane; c < chunks; c += 64) {
                const float r = part_ref[p0 + c];
                if (r > -INFINITY) s += part_sum[p0 + c] * exp2_sum(((double)r - (double)m) * LOG2E);
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0) {
            s_m[b] = m;
            s_log[b] = log(s);
        }
    }
    if (tid == 0) s_count = 0;
    __syncthreads();
    const int per_beam = chunks * n, all = beams * per_beam;
    const int64_t first = (int64_t)g * all;
    // candidate i: its place b V + v (-1: none) and score
    auto candidate = [&](int i, double& score) -> int {
        const int tok = cand_tok[first + i];
        if (tok < 0) return -1;
        const int b = i / per_beam;
        const float x = cand_x[first + i], r = run[g * beams + b];
        score = x == -INFINITY || dead_beam(r) ? -INFINITY : (double)r + (((double)x - s_m[b]) - s_log[b]);
        return b * vocab + tok;
    };
    // a bound that at least n candidates reach: the largest of the waves' n-th largest lane maxima
    uint64_t key = 0;
    for (int i = tid; i < all; i += BJ_THREADS) {
        double s;
        if (candidate(i, s) >= 0) {
            const uint64_t k = order64(s);
            key = k > key ? k : key;
        }
    }
    uint64_t t = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t trial = t | (1ull << bit);
        if (__popcll(__ballot(key >= trial)) >= n) t = trial;
    }
    if (lane == 0) w_key[w] = t;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BJ_THREADS / 64; ++i) t = w_key[i] > t ? w_key[i] : t;
    for (int i = tid; i < all; i += BJ_THREADS) {
        double s;
        const int at = candidate(i, s);
        if (at >= 0 && order64(s) >= t) {
            const int p = atomicAdd(&s_count, 1);
            if (p < BJ_LIST) {
                l_score[p] = s;
                l_at[p] = at;
            }
        }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= BJ_LIST) {
        for (int i = tid; i < count; i += BJ_THREADS) {
            const double s = l_score[i];
            const int at = l_at[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += l_score[j] > s || (l_score[j] == s && l_at[j] < at);
            if (rank < n) {
                best_score[rank] = s;
                best_at[rank] = at;
            }
        }
        __syncthreads();
    } else {                                                  // more ties than the list holds: one after the other
        uint64_t last = ~0ull;
        int last_at = -1;
        for (int r = 0; r < n; ++r) {
            uint64_t k = 0;
            int at = 0x7fffffff;
            for (int i = tid; i < all; i += BJ_THREADS) {
                double s;
                const int c = candidate(i, s);
                if (c < 0) continue;
                const uint64_t ks = order64(s);
                const bool after = ks < last || (ks == last && c > last_at);
                if (after && (ks > k || (ks == k && c < at))) {
                    k = ks;
                    at = c;
                }
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const uint64_t ok = __shfl_xor((unsigned long long)k, o, 64);
                const int oa = __shfl_xor(at, o, 64);
                if (ok > k || (ok == k && oa < at)) {
                    k = ok;
                    at = oa;
                }
            }
            __syncthreads();
            if (lane == 0) {
                w_key[w] = k;
                w_at[w] = at;
            }
            __syncthreads();
            for (int i = 0; i < BJ_THREADS / 64; ++i)
                if (w_key[i] > k || (w_key[i] == k && w_at[i] < at)) {
                    k = w_key[i];
                    at = w_at[i];
                }
            last = k;
            last_at = at;
            if (tid == 0) {
                best_score[r] = __longlong_as_double((long long)((k >> 63) ? k ^ 0x8000000000000000ull : ~k));
                best_at[r] = at;
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
    const int64_t step = 64 * BS_VECS * vec;
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
    MF_REQUIRE((int64_t)groups * beams <= 65535 && (int64_t)beams * vocab <= 0x7fffffffLL, "beam_search_select: %d x %d beams of %d tokens",
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
    hipLaunchKernelGGL(beam_join_kernel, dim3(groups), dim3(BJ_THREADS), 0, st, part_ref, part_sum, cand_x, cand_tok, beam_scores, beams,
                       vocab, p.chunks, n, eos, scores, beam_ids, tokens, next_scores, next_rows, next_tokens);
    return MF_LAUNCH_CHECK();
}
