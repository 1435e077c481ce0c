// Rotary positions: pairs (a, b) of a head's columns turned by an angle that grows with the token's position,
//
//   a' = s (a cos t - b sin t),   b' = s (b cos t + a sin t),   t = position * inv_freq[i]
//
// with a, b = columns (i, i + p/2) or (2i, 2i + 1) of the p columns from `offset` on; the others pass as they are.  The turned key and
// the value go to their cache rows in the same launch.
//
// Angles in 64 bits: at position 10^6 a float32 product is off by up to 0.03 radians.  Turns (t / 2 pi) lose their whole part, the rest,
// within half a turn, goes on in float32 (an error below 2e-7 radians up to position 2^28).  A workgroup computes the cosines and sines of its rows once, for
// all heads, into LDS: one double product and one sincospi a pair and row.  Sums in float32, rounded once.
#include <algorithm>

#include "common.h"

namespace {

constexpr int RO_THREADS = 256, RO_MOST_THREADS = 512;
constexpr int RO_ROWS = 6;                                    // rows of a workgroup, at most
constexpr int RO_MAX_PAIRS = 512;

struct RotaryArgs {
    uint16_t *q_out, *k_out, *k_cache, *v_cache;              // k_out, caches: may be null
    const uint16_t *q, *k, *v;
    const int32_t *positions, *slots;
    const double* inv_freq;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride, num_slots;
    int tokens, heads, kv_heads, dim, pairs, offset, rows;    // rows: of a workgroup
    int units, v_units;                                       // of a head; of a row's values
    uint32_t unit_magic, row_magic;                           // 2^32 / units, and / units of a row, rounded up
    float scale;
};

// N 16-bit elements moved at once
template <int N>
struct Piece {
    typedef __attribute__((ext_vector_type(N / 2))) uint32_t vec;
    vec v;
    __device__ __forceinline__ void load(const uint16_t* p) { v = *(const vec*)p; }
    __device__ __forceinline__ void stream(const uint16_t* p) { v = __builtin_nontemporal_load((const vec*)p); }
    __device__ __forceinline__ void store(uint16_t* p) const { *(vec*)p = v; }
    __device__ __forceinline__ uint16_t at(int i) const { return (uint16_t)(v[i >> 1] >> (16 * (i & 1))); }
    template <typename T>
    __device__ __forceinline__ void set2(int i, float lo, float hi) { v[i >> 1] = pack2<T>(lo, hi); }
};
template <>
struct Piece<2> {
    uint32_t v;
    __device__ __forceinline__ void load(const uint16_t* p) { v = *(const uint32_t*)p; }
    __device__ __forceinline__ void store(uint16_t* p) const { *(uint32_t*)p = v; }
    __device__ __forceinline__ uint16_t at(int i) const { return (uint16_t)(v >> (16 * (i & 1))); }
    template <typename T>
    __device__ __forceinline__ void set2(int, float lo, float hi) { v = pack2<T>(lo, hi); }
};
template <>
struct Piece<1> {
    uint16_t v;
    __device__ __forceinline__ void load(const uint16_t* p) { v = *p; }
    __device__ __forceinline__ void store(uint16_t* p) const { *p = v; }
    __device__ __forceinline__ uint16_t at(int) const { return v; }
    template <typename T>
    __device__ __forceinline__ void set2(int, float lo, float) { v = T::from_float(lo); }
};

__device__ __forceinline__ void turn(float a, float b, float2 cs, float& oa, float& ob) {
    oa = fmaf(a, cs.x, -(b * cs.y));
    ob = fmaf(b, cs.x, a * cs.y);
}

// A unit of a row's work.  Of a head with neighbours in pairs (NEAR, VEC >= 2): VEC columns, of which those inside the turned part are
// turned.  Otherwise a piece of the first members with the piece of their partners, or, behind those units, VEC columns that pass;
// with VEC 1 the partner may be the neighbour.  Of the values: VEC columns to copy.
template <int VEC>
struct RotaryUnit {
    const uint16_t* in;                                       // the head, or the row of values
    uint16_t *out, *cache;                                    // where its result goes (null: not there)
    int c, d, first;                                          // columns of the two pieces (d < 0: one), number of the first pair
    Piece<VEC> x, y;
};

template <int VEC, bool NEAR>
__device__ __forceinline__ void rotary_take(const RotaryArgs& A, RotaryUnit<VEC>& U, int i, int n_q, int n_qk, int64_t row, int64_t at, bool cached) {
    U.in = nullptr;
    if (i >= n_qk) {
        if (cached) U.in = A.v + row * A.v_stride;
        U.out = nullptr, U.cache = A.v_cache + at;
        U.c = (i - n_qk) * VEC, U.d = -1, U.first = A.pairs;
        return;
    }
    const bool is_q = i < n_q;
    const int j = is_q ? i : i - n_q;
    const int head = A.units == 1 ? j : (int)__umulhi((uint32_t)j, A.unit_magic), u = j - head * A.units, hc = head * A.dim;
    const uint16_t* in = is_q ? A.q + row * A.q_stride + hc : A.k + row * A.k_stride + hc;
    U.out = is_q ? A.q_out + row * A.q_out_stride + hc : A.k_out ? A.k_out + row * A.k_out_stride + hc : nullptr;
    U.cache = !is_q && cached ? A.k_cache + at + hc : nullptr;
    U.d = -1;
    bool turned;
    if constexpr (NEAR && VEC >= 2) {
        U.c = u * VEC;
        U.first = (U.c - A.offset) >> 1;                      // offset is even
        turned = U.first + VEC / 2 > 0 && U.first < A.pairs;
    } else {
        const int n = A.pairs / VEC;
        turned = u < n;
        U.first = turned ? u * VEC : A.pairs;
        if (turned) {
            U.c = A.offset + (NEAR ? 2 * u : u * VEC);
            U.d = NEAR ? U.c + 1 : U.c + A.pairs;
        } else {
            U.c = (u - n) * VEC;
            U.c = U.c < A.offset ? U.c : U.c + 2 * A.pairs;
        }
    }
    if (!turned && U.out == in) U.out = nullptr;              // passes where it lies
    if (U.out || U.cache) U.in = in;
}

template <typename T, int VEC, bool NEAR>
__device__ __forceinline__ void rotary_finish(const RotaryArgs& A, RotaryUnit<VEC>& U, const float2* cs) {
    if constexpr (NEAR && VEC >= 2) {
        if (U.first < A.pairs && U.first + VEC / 2 > 0) {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                const int p = U.first + i;
                float a, b;
                turn(T::to_float(U.x.at(2 * i)), T::to_float(U.x.at(2 * i + 1)), cs[min(max(p, 0), A.pairs - 1)], a, b);
                const uint32_t two = pack2<T>(a, b);
                if constexpr (VEC == 2) U.x.v = p >= 0 && p < A.pairs ? two : U.x.v;
                else U.x.v[i] = p >= 0 && p < A.pairs ? two : U.x.v[i];
            }
        }
    } else if (U.d >= 0) {
        float a[VEC], b[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) turn(T::to_float(U.x.at(i)), T::to_float(U.y.at(i)), cs[U.first + i], a[i], b[i]);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            U.x.template set2<T>(i, a[i], VEC > 1 ? a[i + (VEC > 1)] : 0.f);
            U.y.template set2<T>(i, b[i], VEC > 1 ? b[i + (VEC > 1)] : 0.f);
        }
    }
    if (U.out) {
        U.x.store(U.out + U.c);
        if (U.d >= 0) U.y.store(U.out + U.d);
    }
    if (U.cache) {
        U.x.store(U.cache + U.c);
        if (U.d >= 0) U.y.store(U.cache + U.d);
    }
}

// What bounds it: memory (8191 rows of 32 + 8 heads of 128 into a cache, 202 MB: 37 us; 16001 rows of 64 + 8 heads of 80, 369 MB: 68 us; 5.4 TB/s,
// as a copy).  Two units a thread are on their way at once.  One row: 3 us, of which a launch is most.
template <typename T, int VEC, bool NEAR, bool STREAM>
__global__ __launch_bounds__(RO_MOST_THREADS) void rotary_kernel(const RotaryArgs A) {
    extern __shared__ float2 table[];                         // [rows][pairs]: s cos, s sin
    const int threads = blockDim.x;
    const int64_t row0 = (int64_t)blockIdx.x * A.rows;
    const int rows = (int)min((int64_t)A.rows, A.tokens - row0);
    for (int i = threadIdx.x; i < rows * A.pairs; i += threads) {
        const int r = i / A.pairs, p = i - r * A.pairs;
        const double turns = (double)A.positions[row0 + r] * (A.inv_freq[p] * 0.15915494309189535);
        float sn, cn;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
        table[i] = make_float2(A.scale * cn, A.scale * sn);
    }
    __syncthreads();
    const int n_q = A.heads * A.units, n_qk = n_q + A.kv_heads * A.units, each = n_qk + A.v_units, all = rows * each;
    for (int i = threadIdx.x; i < all; i += 2 * threads) {
        RotaryUnit<VEC> U[2];
        int r[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int j = min(i + k * threads, all - 1);
            r[k] = A.rows == 1 ? 0 : each == 1 ? j : (int)__umulhi((uint32_t)j, A.row_magic);
            const int64_t row = row0 + r[k], slot = A.slots ? A.slots[row] : -1;
            const bool cached = slot >= 0 && slot < A.num_slots;
            rotary_take<VEC, NEAR>(A, U[k], j - r[k] * each, n_q, n_qk, row, cached ? slot * A.kv_heads * A.dim : 0, cached);
            if (i + k * threads >= all) U[k].in = nullptr;
            if constexpr (STREAM) {
                if (U[k].in) U[k].x.stream(U[k].in + U[k].c);
                if (U[k].in && U[k].d >= 0) U[k].y.stream(U[k].in + U[k].d);
            } else if (U[k].in) {
                U[k].x.load(U[k].in + U[k].c);
                if (U[k].d >= 0) U[k].y.load(U[k].in + U[k].d);
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (U[k].in) rotary_finish<T, VEC, NEAR>(A, U[k], table + r[k] * A.pairs);
    }
}

// The widest access that every piece's start and length allows.  With partners half the part away both pieces begin VEC columns apart,
// with neighbours a pair must not lie across two.
int rotary_vec(const RotaryArgs& A, bool near) {
    uint64_t bits = (uint64_t)A.dim | A.q_stride | A.q_out_stride;
    uint64_t at = (uintptr_t)A.q | (uintptr_t)A.q_out;
    if (A.k) bits |= A.k_stride, at |= (uintptr_t)A.k;
    if (A.k_out) bits |= A.k_out_stride, at |= (uintptr_t)A.k_out;
    if (A.k_cache) bits |= A.v_stride, at |= (uintptr_t)A.k_cache | (uintptr_t)A.v_cache | (uintptr_t)A.v;
    if (near) bits |= (A.offset & 1);
    else bits |= A.offset | A.pairs;
    bits |= at >> 1;
    return bits & 1 ? 1 : bits & 2 ? 2 : bits & 4 ? 4 : 8;
}

}  // namespace

extern "C" int mf_rotary_embedding(void* query_out, void* key_out, const void* query, const void* key, const void* value, void* key_cache,
                                   void* value_cache, const int32_t* positions, const double* inv_freq, const int32_t* slot_mapping,
                                   int num_tokens, int n_heads, int n_kv_heads, int head_dim, int n_pairs, int offset, int interleaved,
                                   float scale, int64_t num_slots, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
                                   int64_t q_out_row_stride, int64_t k_out_row_stride, int dtype, void* stream) {
    MF_REQUIRE(dtype == MF_BF16 || dtype == MF_FP16, "rotary_embedding: dtype must be bf16 or fp16");
    MF_REQUIRE(num_tokens >= 0 && num_tokens < (1 << 24) && n_heads > 0 && n_kv_heads >= 0 && head_dim > 0 && n_heads <= 4096 && n_kv_heads <= 4096,
               "rotary_embedding: bad sizes");
    MF_REQUIRE(n_pairs > 0 && n_pairs <= RO_MAX_PAIRS && offset >= 0 && offset + 2 * n_pairs <= head_dim && head_dim <= 2 * RO_MAX_PAIRS,
               "rotary_embedding: %d pairs from column %d do not fit heads of %d (up to %d)", n_pairs, offset, head_dim, 2 * RO_MAX_PAIRS);
    if (num_tokens == 0) return 0;
    MF_REQUIRE(query && query_out && positions && inv_freq, "rotary_embedding: null argument");
    MF_REQUIRE((key != nullptr) == (n_kv_heads > 0) && (key || !key_out), "rotary_embedding: a key goes with its heads and its output");
    MF_REQUIRE((key_cache != nullptr) == (value_cache != nullptr) && (key_cache != nullptr) == (value != nullptr) &&
               (key_cache != nullptr) == (slot_mapping != nullptr) && (!key_cache || key),
               "rotary_embedding: caches go with a key, a value and slots");
    MF_REQUIRE(!key_cache || num_slots > 0, "rotary_embedding: caches without slots");
    MF_REQUIRE((((uintptr_t)query | (uintptr_t)query_out | (uintptr_t)key | (uintptr_t)key_out | (uintptr_t)value) & 1) == 0 &&
               ((uintptr_t)inv_freq & 7) == 0, "rotary_embedding: tensors must be aligned to their type");
    RotaryArgs A = {};
    A.q_out = (uint16_t*)query_out, A.k_out = (uint16_t*)key_out, A.k_cache = (uint16_t*)key_cache, A.v_cache = (uint16_t*)value_cache;
    A.q = (const uint16_t*)query, A.k = (const uint16_t*)key, A.v = (const uint16_t*)value;
    A.positions = positions, A.slots = slot_mapping, A.inv_freq = inv_freq;
    const int64_t qw = (int64_t)n_heads * head_dim, kw = (int64_t)n_kv_heads * head_dim;
    A.q_stride = q_row_stride > 0 ? q_row_stride : qw;
    A.q_out_stride = q_out_row_stride > 0 ? q_out_row_stride : qw;
    A.k_stride = k_row_stride > 0 ? k_row_stride : kw;
    A.k_out_stride = k_out_row_stride > 0 ? k_out_row_stride : kw;
    A.v_stride = v_row_stride > 0 ? v_row_stride : kw;
    MF_REQUIRE(A.q_stride >= qw && A.q_out_stride >= qw && A.k_stride >= kw && A.k_out_stride >= kw && A.v_stride >= kw,
               "rotary_embedding: rows overlap");
    MF_REQUIRE(num_tokens == 1 || ((query_out != query || A.q_out_stride == A.q_stride) && (!key_out || key_out != key || A.k_out_stride == A.k_stride)),
               "rotary_embedding: an output is its input with rows of another distance");
    MF_REQUIRE(query_out != key_out && query_out != key && key_out != query && (!value || (value != query_out && value != key_out)),
               "rotary_embedding: query, key and value share memory that is written");
    A.num_slots = num_slots, A.tokens = num_tokens, A.heads = n_heads, A.kv_heads = n_kv_heads, A.dim = head_dim, A.pairs = n_pairs;
    A.offset = offset, A.scale = scale;
    const int vec = rotary_vec(A, interleaved != 0);
    A.units = interleaved && vec > 1 ? head_dim / vec : n_pairs / vec + (head_dim - 2 * n_pairs) / vec;
    A.v_units = key_cache ? (int)(kw / vec) : 0;
    // exact for up to 2^32 / units units; not used for one
    auto magic = [](int64_t units) { return (uint32_t)((0x100000000ll + units - 1) / units); };
    const int64_t each = (int64_t)(n_heads + n_kv_heads) * A.units + A.v_units;
    A.unit_magic = magic(A.units), A.row_magic = magic(each);
    // Several rows a workgroup where they are short and there are enough to fill the device: as many as make a turn of its threads, two
    // units each, and no more angles than threads.  (16001 rows in 1, 2, 4 and 6 a workgroup: 8 + 2 heads of 64, 76 units a row, 18.6, 15.6,
    // 13.4 and 12.1 us; 7 + 1 of 256, 288 units, 41.0, 34.4, 35.3, 38.9; 32 + 8 of 128, 448 units, 71.1, 76.4, 79.3, 84.8.  2048 rows: 4.6,
    // 4.4, 4.8, 4.9; 7.2, 7.8, 9.1, 11.1; 10.3, 11.3, 13.2, 16.4.)
    A.rows = num_tokens < 4096 ? 1 : (int)std::min<int64_t>((2 * RO_THREADS + each / 2) / each, std::min(RO_ROWS, RO_THREADS / n_pairs));
    A.rows = std::max(A.rows, 1);
    if (each > (1 << 14)) A.rows = 1;                         // the division by them is exact up to 2^32 / each
    // long rows of few tokens: a turn of 512 threads (64 rows of 576 units 3.5 us, of 800 3.9; of 256 threads 4.3 and 4.7; 2048 rows 10.5
    // and 13.3, of 256 threads 9.7 and 13.2)
    const int threads = each > 2 * RO_THREADS && num_tokens < 2048 ? RO_MOST_THREADS : RO_THREADS;
    // Inputs that the last-level cache does not keep beside the outputs are read past the caches (32 + 8 heads of 128 behind a copy that
    // writes them, both: 16001 rows, 197 MB, 145.8 -> 140.8 us, 7000 rows, 86 MB, 54.2 -> 52.6; 4096 rows, 50 MB, 32.5 -> 32.8).  Outputs are not: what
    // that gains, the attention behind it loses (8191 rows, both 572 -> 575 us).
    const bool stream_in = (int64_t)num_tokens * (qw + kw + (key_cache ? kw : 0)) * 2 >= 80000000;
    const dim3 grid((unsigned)((num_tokens + A.rows - 1) / A.rows));
    const size_t lds = (size_t)A.rows * n_pairs * sizeof(float2);
    hipStream_t st = (hipStream_t)stream;
#define RO_LAUNCH(T, N)                                                                                                    \
    do {                                                                                                                   \
        if (vec == 8 && stream_in) hipLaunchKernelGGL((rotary_kernel<T, 8, N, true>), grid, dim3(threads), lds, st, A); \
        else if (vec == 8) hipLaunchKernelGGL((rotary_kernel<T, 8, N, false>), grid, dim3(threads), lds, st, A);        \
        else if (vec == 4) hipLaunchKernelGGL((rotary_kernel<T, 4, N, false>), grid, dim3(threads), lds, st, A);        \
        else if (vec == 2) hipLaunchKernelGGL((rotary_kernel<T, 2, N, false>), grid, dim3(threads), lds, st, A);        \
        else hipLaunchKernelGGL((rotary_kernel<T, 1, N, false>), grid, dim3(threads), lds, st, A);                      \
    } while (0)
    if (dtype == MF_BF16) {
        if (interleaved) RO_LAUNCH(BF16, true);
        else RO_LAUNCH(BF16, false);
    } else {
        if (interleaved) RO_LAUNCH(FP16, true);
        else RO_LAUNCH(FP16, false);
    }
#undef RO_LAUNCH
    return MF_LAUNCH_CHECK();
}
