// Log probabilities of given tokens, with their ranks, the entropy of the distribution and its most likely tokens:
//
//   lp(v) = x[v] - m - log Z,   Z = sum_u exp(x[u] - m),   H = log Z - (1 / Z) sum_u (x[u] - m) exp(x[u] - m)
//   rank(v) = number of tokens u with x[u] > x[v], or x[u] = x[v] and u < v
//
// One pass over the logits for the sums, the rank and the largest logit of every lane's steps; the best ones are looked for behind it, in
// those groups of a lane's steps whose largest reaches the n-th largest of the workgroup's 256 lanes.  A group is one step of 16 logits for
// each 98304 columns of the piece or part of them (24 groups a lane at most), so that is n times 16, 32, ... logits, read once more, and those of
// groups whose largest has the upper 16 bits of that bound.  (4137 x 152064 bf16 with 5, 20 and 64 alternatives: 211, 215 and 228 us; whole lanes read again, of whose 16 bytes a step
// memory gives 128, 220, 297 and 403; a list kept on the way 280, 347 and 545; without alternatives 215; of rows of equal logits, which
// reach it all, 233, 230 and 235.)  The waves of a workgroup take the steps of a piece of a
// row in turn; each lane's sums are about a reference m of its own (moved when a logit passes it by more than 8: the sums stay
// in range and H loses no more than that).  A row of one workgroup is done then, others are joined by a second kernel.  Sums in
// float32: their errors are of the size of the rounding of what comes out.
#include <algorithm>

#include "logit_rows.h"

namespace {

constexpr int TL_WAVES = 4;
constexpr int TL_MAX_GROUPS = 64;                             // workgroups of a row
constexpr int TL_MAX_N = 64;                                  // alternatives
constexpr int TL_LIST = 512;                                  // logits that a workgroup ranks at a time
constexpr int TL_TURNS = 24;                                  // groups of steps that lanes' largest logits are kept of
constexpr int TL_LATE = 8;                                    // steps whose sums are added up by themselves
constexpr int TL_HITS = 1024;                                 // (lane, group)s that are looked into at once
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

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float FAR = 65536.f;                                // references whose product with LOG2E is rounded by 2^-8 at most
__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }      // d >= -104

// the sums moved to a reference m at or above their own
__device__ __forceinline__ void sums_to(RowSums& s, float m) {
    const float d = s.m > -INFINITY ? fmaxf(s.m - m, -104.f) : -104.f;
    const float e = s.m > -INFINITY ? exp_neg(d) : 0.f;
    s.w = e * fmaf(d, s.z, s.w);
    s.z *= e;
    s.m = m;
}

// A lane's sums while it walks, in units of log 2: an exponent is x LOG2E - refl, one operation, with the product ref LOG2E rounded
// once, to refl; `rest` is what that left out, which the sums make good when they are taken out.  The logits of a step are added up by
// themselves, and TL_LATE steps of them: hundreds of like terms of a rounding's size beside one sum would all be rounded one way
// (147000 logits 18 below a peak: log probabilities off by 3e-5).
struct LaneSums {
    float ref = 0.f, refl = 0.f, rest = 0.f, z = 0.f, w = 0.f, late_z = 0.f, late_w = 0.f;
    bool has = false;                                         // a finite logit was seen: ref is one
    __device__ __forceinline__ void take_late() {
        z += late_z;
        w += late_w;
        late_z = late_w = 0.f;
    }
    __device__ __forceinline__ RowSums out(int above) const {
        const float e = __builtin_amdgcn_exp2f(-rest);
        return {has ? ref : -INFINITY, z * e, (w - rest * z) * e * LN2, above};
    }
    __device__ __forceinline__ void move(float to) {
        take_late();
        RowSums s = out(0);
        sums_to(s, to);
        has = true;
        ref = to;
        refl = fabsf(to) < FAR ? to * LOG2E : 0.f;            // far: not used
        rest = fabsf(to) < FAR ? fmaf(to, LOG2E, -refl) : 0.f;
        const float e = __builtin_amdgcn_exp2f(rest);         // out(), backwards
        z = s.z * e;
        w = s.w * e * LOG2E + rest * z;
    }
};

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

// the float below x; of zeros of both signs, the one below them
__device__ __forceinline__ float below(float x) { return order32_back(order32(x == 0.f ? -0.f : x) - 1); }

__device__ u32x4 tl_nothing;                                  // what a row without a whole vector loads in its place

// the largest of a wave's values, in every lane
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define TL_DPP(ctrl) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false))
    TL_DPP(0x111);                                            // from 1, 2, 4, 8 lanes below within sixteen
    TL_DPP(0x112);
    TL_DPP(0x114);
    TL_DPP(0x118);
    TL_DPP(0x142);                                            // the last lane of sixteen to the next sixteen, of 32 to the next 32
    TL_DPP(0x143);
#undef TL_DPP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The columns of a row that a workgroup has, and how its lanes take them: lane l of wave w has, of step k, vectors u at columns
// c0 + (k TL_WAVES + w) STEP + (64 u + l) VEC.  Columns are counted from the 16-byte boundary at or before the row's start, `mis` elements in
// front of it.
struct RowPiece {
    const uint8_t* base;
    int mis, vocab, c0, c1, in0, in1;                         // in0 .. in1: whole vectors inside the row
};

// logits of one vector, those outside the row or the piece as -inf
template <typename L>
__device__ __forceinline__ void edge_vector(const RowPiece& p, int v, float* f) {
    if ((v < p.in0 || v > p.in1) && v < p.c1)                 // not wholly inside the row: element by element
#pragma unroll
        for (int e = 0; e < L::VEC; ++e) f[e] = L::at(p.base, min(max(v + e - p.mis, 0), p.vocab - 1));
#pragma unroll
    for (int e = 0; e < L::VEC; ++e) f[e] = v + e >= p.mis && v + e < p.c1 ? f[e] : -INFINITY;
}

// the lowest bit of a key that two logits of the type differ in, but for +inf where it counts as the largest float32
template <typename L> struct LowBit { static constexpr int value = 0; };
template <> struct LowBit<Logit16<BF16>> { static constexpr int value = 16; };
template <> struct LowBit<Logit16<FP16>> { static constexpr int value = 13; };

struct TopShared {
    uint32_t key[TL_WAVES * 64];                              // of the lanes' largest logits (0: no column)
    uint16_t most[TL_TURNS][TL_WAVES * 64];                   // upper halves of those of a lane and group of steps
    uint16_t hit[TL_HITS];                                    // group x 256 + lane: those in question
    __align__(16) float x[TL_LIST];                           // logits in question, their tokens
    __align__(16) int tok[TL_LIST];
    int hits, count;
};
// the upper half of a key, of that of a float
__device__ __forceinline__ uint32_t order_high(uint16_t h) { return (uint16_t)(h ^ ((int16_t)h < 0 ? 0xffffu : 0x8000u)); }

// Calls what(x, token) for the logits of the lanes and groups whose largest may reach key k: from a list, a vector a thread (four at a time),
// or, where they are more than it takes, each lane for itself; `enough` says when to stop.  `per`: steps of a group.
template <typename L, typename F, typename G>
__device__ __forceinline__ void for_hits(const RowPiece& p, TopShared& sh, int per, uint32_t k, F&& what, G&& enough) {
    constexpr int VEC = L::VEC, VECS = L::VECS, STEP = 64 * VEC * VECS, AT_ONCE = 4;
    const int turns = (p.c1 - p.c0 + TL_WAVES * STEP - 1) / (TL_WAVES * STEP), groups = (turns + per - 1) / per;
    auto vector = [&](int g, int lane, int r) {               // column of vector r of a lane and group
        return p.c0 + ((g * per + r / VECS) * TL_WAVES + (lane >> 6)) * STEP + (r % VECS * 64 + (lane & 63)) * VEC;
    };
    auto use = [&](int v, const u32x4& raw) {
        float f[VEC];
        L::unpack(raw, f);
        edge_vector<L>(p, v, f);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (v + e >= p.mis && v + e < p.c1) what(counted(f[e]), v + e - p.mis);
    };
    auto load = [&](int v) { return v >= p.in0 && v <= p.in1 ? *(const u32x4*)(p.base + (int64_t)(v - p.mis) * L::BYTES) : (u32x4){0, 0, 0, 0}; };
    __syncthreads();
    if (threadIdx.x == 0) sh.hits = 0;
    __syncthreads();
    for (int g = 0; g < groups; ++g)
        if (order_high(sh.most[g][threadIdx.x]) >= k >> 16) {
            const int i = atomicAdd(&sh.hits, 1);
            if (i < TL_HITS) sh.hit[i] = (uint16_t)(g * TL_WAVES * 64 + threadIdx.x);
        }
    __syncthreads();
    const int hits = sh.hits, each = per * VECS, items = hits * each;
    if (hits <= TL_HITS) {
        for (int i0 = threadIdx.x; i0 < items && !enough(); i0 += AT_ONCE * TL_WAVES * 64) {
            u32x4 raw[AT_ONCE];
            int at[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int i = min(i0 + j * TL_WAVES * 64, items - 1), h = i / each;
                at[j] = vector(sh.hit[h] / (TL_WAVES * 64), sh.hit[h] % (TL_WAVES * 64), i - h * each);
                raw[j] = load(at[j]);
                if (i0 + j * TL_WAVES * 64 >= items) at[j] = p.c1;
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
                if (at[j] < p.c1) use(at[j], raw[j]);
        }
    } else {
        for (int g = 0; g < groups; ++g)
            if (order_high(sh.most[g][threadIdx.x]) >= k >> 16)
                for (int r = 0; r < each && !enough(); ++r) {
                    const int v = vector(g, threadIdx.x, r);
                    if (v < p.c1) use(v, load(v));
                }
    }
    __syncthreads();
}

// The n best logits of the piece, or all, in sh.x and sh.tok, with others beside them; returns how many there are.
template <typename L>
__device__ int best_of_piece(const RowPiece& p, TopShared& sh, int per, uint32_t key, int n) {
    const int lane = threadIdx.x & 63;
    sh.key[threadIdx.x] = key;
    __syncthreads();
    // the n-th largest of the lanes' keys, bit by bit; fewer lanes with a column than that: the lowest key
    uint32_t k4[TL_WAVES], bound = 0;
#pragma unroll
    for (int i = 0; i < TL_WAVES; ++i) k4[i] = sh.key[lane + 64 * i];
    for (int bit = 31; bit >= LowBit<L>::value; --bit) {
        const uint32_t trial = bound | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < TL_WAVES; ++i) c += __popcll(__ballot(k4[i] >= trial));
        if (c >= n) bound = trial;
        if (c == n) break;                                    // no bit below changes which lanes these are
    }
    // how many reach key k (not all of them where it is more than TL_LIST, of which the first go into the list)
    auto count_from = [&](uint32_t k) {
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        for_hits<L>(p, sh, per, k, [&](float x, int tok) {
            if (order32(x + 0.f) >= k) {
                const int i = atomicAdd(&sh.count, 1);
                if (i < TL_LIST) {
                    sh.x[i] = x;
                    sh.tok[i] = tok;
                }
            }
        }, [&] { return __hip_atomic_load(&sh.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > TL_LIST; });
        return sh.count;
    };
    int c = count_from(bound);
    if (c <= TL_LIST) return c;
    // More than fit: a higher bound that at least n reach, between `bound` and the largest key; the same in every thread.  In bits that the
    // type's keys differ in.
    constexpr int LOW = LowBit<L>::value;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < TL_WAVES; ++i) most = max(most, k4[i]);
    uint32_t lo = bound >> LOW, hi = (wave_max_u32(most) >> LOW) + 1;         // (no key is above that of +inf)
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        c = count_from(mid << LOW);
        if (c >= n && c <= TL_LIST) return c;
        if (c > TL_LIST) lo = mid;
        else hi = mid;
    }
    // Fewer than n above the logits of key `lo`, and more of those than fit: the lowest tokens of them, looked for in order.
    c = count_from(hi << LOW);
    constexpr int AT_ONCE = 4;                                // columns a thread
    auto take_equal = [&](float level) {
        for (int v0 = p.c0; v0 < p.c1 && c < n; v0 += AT_ONCE * TL_WAVES * 64) {
            float x[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
                x[j] = L::at(p.base, min(max(v0 + j * TL_WAVES * 64 + (int)threadIdx.x - p.mis, 0), p.vocab - 1));
            uint64_t tie[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int v = v0 + j * TL_WAVES * 64 + (int)threadIdx.x;
                tie[j] = __ballot(v >= p.mis && v < p.c1 && counted(x[j]) == level);
                if (lane == 0) sh.key[j * TL_WAVES + (threadIdx.x >> 6)] = __popcll(tie[j]);
            }
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                int before = c + all;
#pragma unroll
                for (int i = 0; i < TL_WAVES; ++i) {
                    if (i < (int)(threadIdx.x >> 6)) before += sh.key[j * TL_WAVES + i];
                    all += sh.key[j * TL_WAVES + i];
                }
                before += __popcll(tie[j] & ((1ull << lane) - 1ull));
                if ((tie[j] >> lane & 1) && before < n) {
                    sh.x[before] = level;
                    sh.tok[before] = v0 + j * TL_WAVES * 64 + (int)threadIdx.x - p.mis;
                }
            }
            c = min(c + all, n);
            __syncthreads();
        }
    };
    // 16 bits: +inf, which counts as the largest float32, is no value of the type and has bits below LOW.  It comes in front of the type's own
    // largest, whose upper bits it shares in bf16.
    if (LOW && lo == order32(counted(INFINITY)) >> LOW) take_equal(counted(INFINITY));
    lo <<= LOW;
    take_equal(order32_back(lo >> 31 ? lo : lo | ((1u << LOW) - 1)));     // (a key's low bits: all ones of negative values)
    return c;
}

// how many entries of a list come in front of (x, token); read four at a time, so that entries behind its end are to be list_end's
__device__ __forceinline__ int rank_in(const float* l_x, const int* l_tok, int count, float x, int token) {
    int rank = 0;
#pragma unroll 2
    for (int j = 0; j < count; j += 4) {
        const f32x4 v = *(const f32x4*)(l_x + j);
        const i32x4 t = *(const i32x4*)(l_tok + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += v[e] > x || (v[e] == x && t[e] < token);
    }
    return rank;
}
__device__ __forceinline__ void list_end(float* l_x, int* l_tok, int count, int i) {
    if (count + i < (count + 3) / 4 * 4) {
        l_x[count + i] = -INFINITY;
        l_tok[count + i] = 0x7fffffff;
    }
}

template <typename L, bool TOP>
__global__ __launch_bounds__(TL_WAVES * 64) void logprob_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                const int* __restrict__ tokens, int vocab, int cols, int groups, int n,
                                                                const LogprobOut out, RowSums* __restrict__ part,
                                                                float* __restrict__ cand_x, int* __restrict__ cand_tok) {
    constexpr int VEC = L::VEC, VECS = L::VECS, E = VECS * VEC, STEP = 64 * E;
    __shared__ TopShared sh;                                  // (without TOP: not used, no LDS)
    __shared__ RowSums w_sums[TL_WAVES];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x / groups;
    const int group = (int)(blockIdx.x - row * groups);
    RowPiece p;
    p.base = (const uint8_t*)logits + row * row_stride * L::BYTES;
    p.mis = (int)(((uintptr_t)p.base & 15) / L::BYTES);
    p.vocab = vocab;
    const int v_end = vocab + p.mis;
    p.c0 = (int)min((int64_t)group * cols, (int64_t)v_end);
    p.c1 = (int)min((int64_t)p.c0 + cols, (int64_t)v_end);
    p.in0 = p.mis ? VEC : 0;
    p.in1 = v_end / VEC * VEC - VEC;

    u32x4 raw[VECS];                                          // a step's logits as stored, loaded one step ahead, from whole vectors
    const uint8_t* vec0 = p.in1 >= p.in0 ? p.base - (int64_t)p.mis * L::BYTES : (const uint8_t*)&tl_nothing;
    const int lo = p.in1 >= p.in0 ? p.in0 : 0, hi = p.in1 >= p.in0 ? p.in1 : 0;
    auto whole = [&](int v0) { return v0 >= p.mis && v0 + STEP <= p.c1; };
    auto load = [&](int v0) {
        if (whole(v0)) {
            const uint8_t* at = p.base + (int64_t)(v0 - p.mis) * L::BYTES;
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
    const int v_first = p.c0 + w * STEP;
    load(v_first);
    const TokenGiven tok = given<L>(p.base, tokens[row], vocab);
    // Logits above `after` count for the rank, in vectors that end in front of the token those at it too: above `before`.  (A masked
    // token: all in front of it count, which is added in the end.)
    const float after = tok.x;
    const float before = !(tok.x > -INFINITY) || tok.token < 0 ? INFINITY : below(tok.x);
    const float counts = fminf(before, after);
    const int tok_v = tok.token < 0 ? -1 : tok.token + p.mis; // its column
    int above = 0;
    if (w == 0 && tok_v >= p.c0 && tok_v < p.c1) {            // of the token's own vector, those in front of it: the equal ones, or, of
        const int v = tok_v / VEC * VEC + lane;               // a masked token, those that would count twice
        if (lane < VEC && v >= p.mis && v < tok_v) {
            const float x = counted(L::at(p.base, v - p.mis));
            above = tok.x > -INFINITY ? x == tok.x : -(int)(x > -INFINITY);
        }
    }

    LaneSums sum;
    int late = 0;
    // a lane's largest logit, and that of the steps that make a group (`per` of them; one at least: a row that ends where a piece begins
    // leaves an empty one behind) with their count and the group's number
    const int turns = (p.c1 - p.c0 + TL_WAVES * STEP - 1) / (TL_WAVES * STEP), per = max((turns + TL_TURNS - 1) / TL_TURNS, 1);
    float most = -INFINITY, group_most = -INFINITY;
    int steps = 0, step_group = 0;
    auto keep_group = [&] {
        sh.most[step_group++][threadIdx.x] = (uint16_t)(__float_as_uint(group_most + 0.f) >> 16);
        most = fmaxf(most, group_most);
        group_most = -INFINITY;
        steps = 0;
    };
    for (int v0 = v_first; v0 < p.c1; v0 += TL_WAVES * STEP) {
        float f[E];
#pragma unroll
        for (int u = 0; u < VECS; ++u) L::unpack(raw[u], f + u * VEC);
        if (!whole(v0)) {                                     // the row's and the piece's ends
#pragma unroll
            for (int u = 0; u < VECS; ++u) edge_vector<L>(p, v0 + (u * 64 + lane) * VEC, f + u * VEC);
        }
        load(v0 + TL_WAVES * STEP);                           // on its way behind this step's work
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < E; k += 2) mx = fmaxf(fmaxf(f[k], f[k + 1]), mx);
        if (__ballot(mx == INFINITY)) {                       // +inf counts as the largest finite value
#pragma unroll
            for (int k = 0; k < E; ++k) f[k] = f[k] == INFINITY ? 3.402823466e38f : f[k];
            mx = mx == INFINITY ? 3.402823466e38f : mx;
        }
        if constexpr (TOP) {
            group_most = fmaxf(group_most, mx);
            if (++steps == per) keep_group();
        }
        const bool moves = mx > -INFINITY && (!sum.has || mx - sum.ref > 8.f);
        if (__ballot(moves)) {
            if (moves) sum.move(mx);
        }
        // 2^-150 is no float32 any more; -inf and NaN end there too
        float step_z[2] = {}, step_w[2] = {};
        if (!__ballot(!(fabsf(sum.ref) < FAR))) {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float d = fmaxf(fmaf(f[k], LOG2E, -sum.refl), -150.f), e = __builtin_amdgcn_exp2f(d);
                step_z[k & 1] += e;
                step_w[k & 1] = fmaf(d, e, step_w[k & 1]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float x = fabsf(sum.ref) < FAR ? fmaf(f[k], LOG2E, -sum.refl) : (f[k] - sum.ref) * LOG2E;
                const float d = fmaxf(x, -150.f), e = __builtin_amdgcn_exp2f(d);
                step_z[k & 1] += e;
                step_w[k & 1] = fmaf(d, e, step_w[k & 1]);
            }
        }
        sum.late_z += step_z[0] + step_z[1];
        sum.late_w += step_w[0] + step_w[1];
        if (++late % TL_LATE == 0) sum.take_late();
        if (__ballot(mx > counts)) {
#pragma unroll
            for (int u = 0; u < VECS; ++u) {
                const float t = v0 + (u * 64 + lane) * VEC + VEC <= tok_v ? before : after;
#pragma unroll
                for (int e = 0; e < VEC; ++e) above += f[u * VEC + e] > t;
            }
        }
    }
    // ---- the wave's sums, the workgroup's
    sum.take_late();
    RowSums s = sum.out(above);
    sums_to(s, wave_max(s.m));
    s.z = wave_sum(s.z);
    s.w = wave_sum(s.w);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s.above += __shfl_xor(s.above, o, 64);
    if (lane == 0) w_sums[w] = s;
    int kept = 0;
    if constexpr (TOP) {
        if (steps) keep_group();
        for (; step_group < (turns + per - 1) / per; ++step_group) sh.most[step_group][threadIdx.x] = 0xffffu;      // below every logit
    }
    if constexpr (TOP) kept = best_of_piece<L>(p, sh, per, v_first + lane * VEC < p.c1 ? order32(most + 0.f) : 0u, n);
    else __syncthreads();
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
        const int64_t at = (int64_t)blockIdx.x * n;
        if (threadIdx.x < 3) list_end(sh.x, sh.tok, kept, threadIdx.x);       // TL_LIST is a multiple of four
        __syncthreads();
        for (int i = threadIdx.x; i < kept; i += TL_WAVES * 64) {
            const float x = sh.x[i];
            const int id = sh.tok[i], rank = rank_in(sh.x, sh.tok, kept, x, id);
            if (rank >= n) continue;
            if (groups == 1) {
                out.top_tokens[row * n + rank] = id;
                out.top_logprobs[row * n + rank] = log_prob(x, all, log_z);
            } else {
                cand_x[at + rank] = x + 0.f;                  // no negative zero: the join goes by keys
                cand_tok[at + rank] = id;
            }
        }
        if (groups > 1 && (int)threadIdx.x >= kept && (int)threadIdx.x < n) { // fewer tokens than that in the piece
            cand_x[at + threadIdx.x] = -INFINITY;
            cand_tok[at + threadIdx.x] = -1;
        }
    }
}

// Joins the workgroups of a row: their sums, and their lists, which are in order, by taking the best head n times (a lane a list; equal
// heads: the lower list, whose tokens are the lower ones).
constexpr int TJ_THREADS = 256;
template <typename L, bool TOP>
__global__ __launch_bounds__(TJ_THREADS) void logprob_join_kernel(const void* __restrict__ logits, int64_t row_stride,
                                                                  const int* __restrict__ tokens, int vocab, int groups, int n,
                                                                  const LogprobOut out, const RowSums* __restrict__ part,
                                                                  const float* __restrict__ cand_x, const int* __restrict__ cand_tok) {
    extern __shared__ uint32_t l_key[];                       // [groups x n] keys (0: no entry), tokens behind them
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, entries = groups * n;
    int* l_tok = (int*)(l_key + entries);
    if constexpr (TOP) {
        for (int i = tid; i < entries; i += TJ_THREADS) {
            const int t = cand_tok[row * entries + i];
            l_key[i] = t >= 0 ? order32(cand_x[row * entries + i]) : 0u;
            l_tok[i] = t;
        }
    }
    RowSums s = {-INFINITY, 0.f, 0.f, 0};
    if (lane < groups) s = part[row * groups + lane];
    const TokenGiven tok = given<L>((const uint8_t*)logits + row * row_stride * L::BYTES, tokens[row], vocab);
    sums_to(s, wave_max(s.m));
    s.z = wave_sum(s.z);
    s.w = wave_sum(s.w);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s.above += __shfl_xor(s.above, o, 64);
    const float log_z = logf(s.z);
    if (tid == 0) write_row(out, row, tok, s, log_z);
    if constexpr (TOP) {
        __syncthreads();
        if (tid >= 64) return;
        // a lane's list: its head, the entry behind it (on its way), where the next one lies
        int at = lane * n + 2, id = 0;
        const int end = lane < groups ? lane * n + n : 0;
        uint32_t key = at - 2 < end ? l_key[at - 2] : 0u, key2 = at - 1 < end ? l_key[at - 1] : 0u, best = 0;
        int head = at - 2 < end ? l_tok[at - 2] : 0, head2 = at - 1 < end ? l_tok[at - 1] : 0;
        for (int i = 0; i < n; ++i) {
            const uint32_t m = wave_max_u32(key);
            const int from = (int)__builtin_ctzll(__ballot(key == m));
            const int t = __builtin_amdgcn_readlane(head, from);
            if (lane == i) {
                best = m;
                id = t;
            }
            if (lane == from) {
                key = key2;
                head = head2;
                key2 = at < end ? l_key[at] : 0u;
                head2 = at < end ? l_tok[at] : 0;
                ++at;
            }
        }
        if (lane < n) {
            out.top_tokens[row * n + lane] = id;
            out.top_logprobs[row * n + lane] = log_prob(order32_back(best), s, log_z);
        }
    }
}

// A row a workgroup up to 32768 columns, which saves the second kernel (1 x 32000 with 0, 5, 20 and 64 alternatives: 7, 11.4, 12.6 and
// 16 us, in eight pieces 5.6, 10.5, 13.3 and 23, beside a call's 3), and where there is a row for 384 columns, so that rows alone fill the
// device (1001 x 151643 fp32 91 us, in two pieces 103; 2000 x 152064 bf16 with 5 alternatives 117, in two 120; 200 x 50000 with 20 18.6, in four
// 21.6).  Otherwise equal pieces of 16384 at least (1 x 152064 with 0, 5, 20 and 64: 6.8, 12, 16 and 25 us, in pieces of 4096 5.6,
// 10.5, 14.5 and 40), for 1024 workgroups in all (300 x 152064 bf16 with 5 alternatives in one, two, four and ten: 41.0, 34.4, 30.4 and
// 34.9).
struct LogprobPlan {
    int cols, groups;
    size_t x, tok, bytes;
};
LogprobPlan logprob_plan(int64_t rows, int64_t vocab, int n, int dtype) {
    constexpr int64_t STEP = TL_WAVES * 64 * 16;              // logits of a workgroup's step, of either width
    const int64_t span = vocab + (dtype == MF_FP32 ? 3 : 7);
    int64_t pieces = 1;
    if (span > 32768 && rows * 384 < span)
        pieces = std::min({(1024 + rows - 1) / rows, (span + 16383) / 16384, (int64_t)TL_MAX_GROUPS});
    const int64_t cols = ((span + pieces - 1) / pieces + STEP - 1) / STEP * STEP;
    LogprobPlan p;
    p.cols = (int)cols;
    p.groups = (int)((span + cols - 1) / cols);
    const size_t parts = p.groups == 1 ? 0 : (size_t)rows * p.groups;
    p.x = parts * sizeof(RowSums);
    p.tok = p.x + parts * n * 4;
    p.bytes = p.tok + parts * n * 4;
    return p;
}

}  // namespace

extern "C" size_t mf_token_logprobs_workspace_bytes(int rows, int vocab, int n_top, int dtype) {
    if (rows <= 0 || vocab <= 0 || n_top < 0 || n_top > TL_MAX_N || dtype < 0 || dtype > MF_FP32) return 0;
    return logprob_plan(rows, vocab, n_top, dtype).bytes;
}

extern "C" int mf_token_logprobs(float* logprobs, int32_t* ranks, float* entropy, int32_t* top_tokens, float* top_logprobs,
                                 const void* logits, int64_t row_stride, const int32_t* tokens, int rows, int vocab, int n_top, int dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    MF_REQUIRE(dtype == MF_BF16 || dtype == MF_FP16 || dtype == MF_FP32, "token_logprobs: dtype must be bf16, fp16 or fp32");
    MF_REQUIRE(rows >= 0 && rows < (1 << 24) && vocab > 0 && vocab <= TL_MAX_VOCAB, "token_logprobs: %d rows of %d tokens", rows, vocab);
    MF_REQUIRE(n_top >= 0 && n_top <= TL_MAX_N && n_top <= vocab, "token_logprobs: %d alternatives of %d tokens, up to %d", n_top, vocab,
               TL_MAX_N);
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
    const size_t lds = (size_t)p.groups * n_top * 8;
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
