// Log probabilities of given tokens, with their ranks, the entropy of the distribution and its most likely tokens:
//
//   lp(v) = x[v] - m - log Z,   Z = sum_u exp(x[u] - m),   H = log Z - (1 / Z) sum_u (x[u] - m) exp(x[u] - m)
//   rank(v) = number of tokens u with x[u] > x[v], or x[u] = x[v] and u < v
//
// One pass over the logits.  A wave walks a piece of a row and keeps the two sums about a reference m of each lane's own (moved when a
// logit passes it by more than 8: the sums stay in range and H loses no more than that), the count of the rank and, where asked for, a
// list of its best logits.  The waves of a workgroup join in LDS; a row of one workgroup is done then, others take a second kernel.
// Sums in float32: their errors are of the size of the rounding of what comes out.
#include <algorithm>

#include "logit_rows.h"

namespace {

constexpr int TL_WAVES = 4;
constexpr int TL_MAX_GROUPS = 64;                             // workgroups of a row
constexpr int64_t TL_MAX_VOCAB = 0x7c000000;                  // a column a piece behind the last in 32 bits

struct RowSums {
    float m, z, w;                                            // reference (-inf: no finite logit), sum, weighted sum
    int above;                                                // tokens in front of the given one
};
struct LogprobOut {
    float* logprobs;
    int* ranks;
    float* entropy;
    int* top_tokens;
    float* top_logprobs;
};

__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }      // d >= -104

// the sums moved to a reference m at or above their own
__device__ __forceinline__ void sums_to(RowSums& s, float m) {
    const float d = s.m > -INFINITY ? fmaxf(s.m - m, -104.f) : -104.f;
    const float e = s.m > -INFINITY ? exp_neg(d) : 0.f;
    s.w = e * fmaf(d, s.z, s.w);
    s.z *= e;
    s.m = m;
}

struct TokenGiven {
    int token;                                                // -1: none
    float x;                                                  // its logit; +inf: no token
};
__device__ __forceinline__ float log_prob(float x, const RowSums& s, float log_z) { return x > -INFINITY ? (x - s.m) - log_z : -INFINITY; }

__device__ __forceinline__ void write_row(const LogprobOut& o, int64_t row, const TokenGiven& t, const RowSums& s, float log_z) {
    o.logprobs[row] = t.token < 0 ? -INFINITY : log_prob(t.x, s, log_z);
    o.ranks[row] = t.token < 0 ? -1 : s.above + (t.x > -INFINITY ? 0 : t.token);      // all in front of a masked token count
    o.entropy[row] = s.z > 0.f ? fmaxf(log_z - s.w / s.z, 0.f) : 0.f;
}

// a logit as it counts: +inf as the largest float, NaN as -inf
__device__ __forceinline__ float counted(float x) { return x > -INFINITY ? fminf(x, 3.402823466e38f) : -INFINITY; }

template <typename L>
__device__ __forceinline__ TokenGiven given(const uint8_t* base, int token, int vocab) {
    TokenGiven t = {-1, INFINITY};
    if (token >= 0 && token < vocab) {
        t.token = token;
        t.x = counted(L::at(base, token));
    }
    return t;
}

__device__ u32x4 tl_nothing;                                  // what a row without a whole vector loads in its place

// How many of a list, best first and `n` long, come in front of x; of equals those of lists in front
__device__ __forceinline__ int in_front(const float* l, int n, float x, bool lower) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (l[mid] > x || (lower && l[mid] == x)) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename L, bool TOP>
__global__ __launch_bounds__(TL_WAVES * 64) void logprob_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                const int* __restrict__ tokens, int vocab, int cols, int groups, int n,
                                                                const LogprobOut out, RowSums* __restrict__ part,
                                                                float* __restrict__ cand_x, int* __restrict__ cand_tok) {
    constexpr int VEC = L::VEC, VECS = L::VECS, E = VECS * VEC, STEP = 64 * E;
    __shared__ LogitList lists[TOP ? TL_WAVES : 1];
    __shared__ RowSums w_sums[TL_WAVES];
    __shared__ int w_count[TL_WAVES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t row = blockIdx.x / groups;
    const int group = (int)(blockIdx.x - row * groups);
    const uint8_t* base = (const uint8_t*)logits + row * row_stride * L::BYTES;
    // columns are counted from the 16-byte boundary at or before the row's start, `mis` elements in front of it
    const int mis = (int)(((uintptr_t)base & 15) / L::BYTES);
    const int v_end = vocab + mis;
    const int64_t piece = (int64_t)(group * TL_WAVES + w) * cols;
    const int c0 = (int)min(piece, (int64_t)v_end), c1 = (int)min(piece + cols, (int64_t)v_end);

    u32x4 raw[VECS];                                          // a step's logits as stored, loaded one step ahead
    const int in0 = mis ? VEC : 0, in1 = v_end / VEC * VEC - VEC;
    const uint8_t* vec0 = in1 >= in0 ? base - (int64_t)mis * L::BYTES : (const uint8_t*)&tl_nothing;
    const int lo = in1 >= in0 ? in0 : 0, hi = in1 >= in0 ? in1 : 0;
    auto whole = [&](int v0) { return v0 >= mis && v0 + STEP <= c1; };
    auto load = [&](int v0) {
        if (whole(v0)) {
            const uint8_t* at = base + (int64_t)(v0 - mis) * L::BYTES;
#pragma unroll
            for (int u = 0; u < VECS; ++u) raw[u] = __builtin_nontemporal_load((const u32x4*)(at + (uint32_t)(1024 * u + 16 * lane)));
        } else {
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
                const int v = min(max(v0 + (u * 64 + lane) * VEC, lo), hi);
                raw[u] = __builtin_nontemporal_load((const u32x4*)(vec0 + (int64_t)v * L::BYTES));
            }
        }
    };
    load(c0);
    const int token = tokens[row];
    const TokenGiven tok = given<L>(base, token, vocab);
    // Logits above `after` count for the rank, in vectors that end in front of the token those at it too: above `before`.  (A masked
    // token: all in front of it count, which is added in the end.)
    const float after = tok.x;
    const float before = !(tok.x > -INFINITY) || tok.token < 0 ? INFINITY : order32_back(order32(tok.x == 0.f ? -0.f : tok.x) - 1);
    const int tok_v = tok.token < 0 ? -1 : tok.token + mis;   // its column
    int above = 0;
    if (tok_v >= c0 && tok_v < c1) {                          // of the token's own vector, those in front of it: the equal ones, or, of
        const int v = tok_v / VEC * VEC + lane;               // a masked token, those that would count twice
        if (lane < VEC && v >= mis && v < tok_v) {
            const float x = counted(L::at(base, v - mis));
            above = tok.x > -INFINITY ? x == tok.x : -(int)(x > -INFINITY);
        }
    }

    float thr = -INFINITY;
    bool full = false;
    int count = 0;
    bool has = false;                                         // a finite logit was seen: ref is one
    float ref = 0.f, z = 0.f, ws = 0.f;
    for (int v0 = c0; v0 < c1; v0 += STEP) {
        float f[E];
#pragma unroll
        for (int u = 0; u < VECS; ++u) L::unpack(raw[u], f + u * VEC);
        if (!whole(v0)) {
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
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
        const bool moves = mx > -INFINITY && (!has || mx - ref > 8.f);
        if (__ballot(moves)) {
            if (moves) {
                RowSums s = {has ? ref : -INFINITY, z, ws, 0};
                sums_to(s, mx);
                ref = mx, z = s.z, ws = s.w;
                has = true;
            }
        }
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const float d = fmaxf(f[k] - ref, -104.f);        // e^-104 is no float32 any more; -inf and NaN end there too
            const float e = exp_neg(d);
            z += e;
            ws = fmaf(d, e, ws);
        }
        if (__ballot(mx > fminf(before, after))) {
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
                const float t = v0 + (u * 64 + lane) * VEC + VEC <= tok_v ? before : after;
#pragma unroll
                for (int e = 0; e < VEC; ++e) above += f[u * VEC + e] > t;
            }
        }
        if constexpr (TOP) list_step<L>(lists[w], f, mx4, mx, n, v0, mis, c1, full, thr, count);
    }
    if constexpr (TOP) {
        if (count > n) count = list_cut<2>(lists[w], count, n, thr);
        if (count) count = list_prune(lists[w], count, n);
    }
    // ---- the wave's sums, the workgroup's
    RowSums s = {has ? ref : -INFINITY, z, ws, above};
    sums_to(s, wave_max(s.m));
    s.z = wave_sum(s.z);
    s.w = wave_sum(s.w);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s.above += __shfl_xor(s.above, o, 64);
    if (lane == 0) {
        w_sums[w] = s;
        w_count[w] = count;
    }
    __syncthreads();
    float m = w_sums[0].m;
#pragma unroll
    for (int i = 1; i < TL_WAVES; ++i) m = fmaxf(m, w_sums[i].m);
    RowSums all = {m, 0.f, 0.f, 0};
#pragma unroll
    for (int i = 0; i < TL_WAVES; ++i) {
        RowSums t = w_sums[i];
        sums_to(t, m);
        all.z += t.z;
        all.w += t.w;
        all.above += t.above;
    }
    const float log_z = logf(all.z);
    if (threadIdx.x == 0) {
        if (groups == 1) write_row(out, row, tok, all, log_z);
        else part[blockIdx.x] = all;
    }
    if constexpr (TOP) {
        int have = 0;
#pragma unroll
        for (int i = 0; i < TL_WAVES; ++i) have += w_count[i];
        const int e_w = threadIdx.x / n, e_i = threadIdx.x - e_w * n;         // an entry a thread: 4 n of them at most
        int rank = 2 * LIST_MAX_N, id = -1;
        float x = -INFINITY;
        if (e_w < TL_WAVES && e_i < w_count[e_w]) {
            x = lists[e_w].x[e_i];
            id = lists[e_w].i[e_i];
            rank = e_i;
            for (int i = 0; i < TL_WAVES; ++i)
                if (i != e_w) rank += in_front(lists[i].x, w_count[i], x, i < e_w);
        }
        if (groups == 1) {
            if (rank < n) {
                out.top_tokens[row * n + rank] = id;
                out.top_logprobs[row * n + rank] = log_prob(x, all, log_z);
            }
        } else {
            const int64_t at = (int64_t)blockIdx.x * n;
            if (rank < n) {
                cand_x[at + rank] = x;
                cand_tok[at + rank] = id;
            }
            if ((int)threadIdx.x >= have && (int)threadIdx.x < n) {           // fewer tokens than that in the group
                cand_x[at + threadIdx.x] = -INFINITY;
                cand_tok[at + threadIdx.x] = -1;
            }
        }
    }
}

// Joins the workgroups of a row.  Every group's list is in order, so an entry's rank is its place and a search in each other list; only
// entries at or above the best of the lists' last ones can be among the n.
constexpr int TJ_THREADS = 256;
template <typename L, bool TOP>
__global__ __launch_bounds__(TJ_THREADS) void logprob_join_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                  const int* __restrict__ tokens, int vocab, int groups, int n,
                                                                  const LogprobOut out, const RowSums* __restrict__ part,
                                                                  const float* __restrict__ cand_x, const int* __restrict__ cand_tok) {
    extern __shared__ float l_x[];                            // [groups x n] logits, tokens behind them, then the entries in question
    __shared__ int l_count[TL_MAX_GROUPS], s_count;
    __shared__ float s_bound[TJ_THREADS / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, entries = groups * n;
    int* l_tok = (int*)(l_x + entries);
    uint16_t* l_at = (uint16_t*)(l_tok + entries);
    const TokenGiven tok = given<L>((const uint8_t*)logits + row * row_stride * L::BYTES, tokens[row], vocab);
    if constexpr (TOP) {
        for (int i = tid; i < groups; i += TJ_THREADS) l_count[i] = 0;
        if (tid == 0) s_count = 0;
        __syncthreads();
        float bound = -INFINITY;
        for (int i = tid; i < entries; i += TJ_THREADS) {
            const float x = cand_x[row * entries + i];
            const int t = cand_tok[row * entries + i], g = i / n;
            l_x[i] = x;
            l_tok[i] = t;
            if (t >= 0) {
                atomicAdd(&l_count[g], 1);
                if (i - g * n == n - 1) bound = fmaxf(bound, x);
            }
        }
        bound = wave_max(bound);
        if (lane == 0) s_bound[tid >> 6] = bound;
    }
    RowSums s = {-INFINITY, 0.f, 0.f, 0};
    if (lane < groups) s = part[row * groups + lane];
    sums_to(s, wave_max(s.m));
    s.z = wave_sum(s.z);
    s.w = wave_sum(s.w);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s.above += __shfl_xor(s.above, o, 64);
    const float log_z = logf(s.z);
    if (tid == 0) write_row(out, row, tok, s, log_z);
    if constexpr (TOP) {
        __syncthreads();
        float bound = s_bound[0];
#pragma unroll
        for (int i = 1; i < TJ_THREADS / 64; ++i) bound = fmaxf(bound, s_bound[i]);
        for (int i = tid; i < entries; i += TJ_THREADS)
            if (l_tok[i] >= 0 && l_x[i] >= bound) l_at[atomicAdd(&s_count, 1)] = (uint16_t)i;
        __syncthreads();
        const int count = s_count;
        for (int c0 = 0; c0 < count; c0 += TJ_THREADS / 16) { // sixteen lanes an entry
            const int c = c0 + tid / 16;
            const int i = l_at[min(c, count - 1)], g = i / n;
            const float x = l_x[i];
            int rank = 0;
            for (int o = tid & 15; o < groups; o += 16)
                if (o != g) rank += in_front(l_x + o * n, l_count[o], x, o < g);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) rank += __shfl_xor(rank, o, 64);
            rank += i - g * n;
            if (c < count && (tid & 15) == 0 && rank < n) {
                out.top_tokens[row * n + rank] = l_tok[i];
                out.top_logprobs[row * n + rank] = log_prob(x, s, log_z);
            }
        }
    }
}

struct LogprobPlan {
    int cols, groups;
    size_t x, tok, bytes;
};
LogprobPlan logprob_plan(int64_t rows, int64_t vocab, int n, int dtype) {
    constexpr int64_t STEP = 64 * 16;                         // logits of a wave's step, of either width
    const int64_t span = vocab + (dtype == MF_FP32 ? 3 : 7);
    int64_t cols = std::max<int64_t>(STEP, rows * span / 8192);
    cols = std::max(cols, (span + TL_MAX_GROUPS * TL_WAVES - 1) / (TL_MAX_GROUPS * TL_WAVES));
    cols = std::min((cols + STEP - 1) / STEP * STEP, (span + STEP - 1) / STEP * STEP);
    LogprobPlan p;
    p.cols = (int)cols;
    p.groups = (int)((span + cols * TL_WAVES - 1) / (cols * TL_WAVES));
    const size_t parts = p.groups == 1 ? 0 : (size_t)rows * p.groups;
    p.x = parts * sizeof(RowSums);
    p.tok = p.x + parts * n * 4;
    p.bytes = p.tok + parts * n * 4;
    return p;
}

}  // namespace

extern "C" size_t mf_token_logprobs_workspace_bytes(int rows, int vocab, int n_top, int dtype) {
    if (rows <= 0 || vocab <= 0 || n_top < 0 || n_top > LIST_MAX_N || dtype < 0 || dtype > MF_FP32) return 0;
    return logprob_plan(rows, vocab, n_top, dtype).bytes;
}

extern "C" int mf_token_logprobs(float* logprobs, int32_t* ranks, float* entropy, int32_t* top_tokens, float* top_logprobs,
                                 const void* logits, int64_t row_stride, const int32_t* tokens, int rows, int vocab, int n_top, int dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    MF_REQUIRE(dtype == MF_BF16 || dtype == MF_FP16 || dtype == MF_FP32, "token_logprobs: dtype must be bf16, fp16 or fp32");
    MF_REQUIRE(rows >= 0 && rows < (1 << 24) && vocab > 0 && vocab <= TL_MAX_VOCAB, "token_logprobs: %d rows of %d tokens", rows, vocab);
    MF_REQUIRE(n_top >= 0 && n_top <= LIST_MAX_N && n_top <= vocab, "token_logprobs: %d alternatives of %d tokens, up to %d", n_top, vocab,
               LIST_MAX_N);
    if (rows == 0) return 0;
    if (row_stride <= 0) row_stride = vocab;
    MF_REQUIRE(row_stride >= vocab, "token_logprobs: row stride %lld below the vocabulary's %d", (long long)row_stride, vocab);
    MF_REQUIRE(logprobs && ranks && entropy && logits && tokens && (n_top == 0 || (top_tokens && top_logprobs)), "token_logprobs: null argument");
    MF_REQUIRE(((uintptr_t)logits & (dtype == MF_FP32 ? 3 : 1)) == 0, "token_logprobs: logits must be aligned to their type");
    const LogprobPlan p = logprob_plan(rows, vocab, n_top, dtype);
    MF_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && ((uintptr_t)workspace & 15) == 0),
               "token_logprobs: 16-byte aligned workspace of %zu bytes needed, %zu given", p.bytes, workspace_bytes);
    uint8_t* ws = (uint8_t*)workspace;
    RowSums* part = (RowSums*)ws;
    float* cand_x = (float*)(ws + p.x);
    int* cand_tok = (int*)(ws + p.tok);
    const LogprobOut out = {logprobs, ranks, entropy, top_tokens, top_logprobs};
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)rows * (unsigned)p.groups);
    const size_t lds = (size_t)p.groups * n_top * 10;
#define TL_LAUNCH2(L, TOP)                                                                                                              \
    do {                                                                                                                                \
        hipLaunchKernelGGL((logprob_kernel<L, TOP>), grid, dim3(TL_WAVES * 64), 0, st, logits, row_stride, tokens, vocab, p.cols, p.groups, \
                           n_top, out, part, cand_x, cand_tok);                                                                         \
        const int rc = MF_LAUNCH_CHECK();                                                                                               \
        if (rc || p.groups == 1) return rc;                                                                                             \
        hipLaunchKernelGGL((logprob_join_kernel<L, TOP>), dim3(rows), dim3(TJ_THREADS), lds, st, logits, row_stride, tokens, vocab, p.groups, \
                           n_top, out, part, cand_x, cand_tok);                                                                         \
        return MF_LAUNCH_CHECK();                                                                                                       \
    } while (0)
#define TL_LAUNCH(L)                        \
    do {                                    \
        if (n_top) TL_LAUNCH2(L, true);     \
        else TL_LAUNCH2(L, false);          \
    } while (0)
    if (dtype == MF_FP32) TL_LAUNCH(LogitF32);
    else if (dtype == MF_BF16) TL_LAUNCH(Logit16<BF16>);
    else TL_LAUNCH(Logit16<FP16>);
#undef TL_LAUNCH
#undef TL_LAUNCH2
}
