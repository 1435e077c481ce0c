// Low-rank adapters of many requests beside a projection that they share:
//
//   out[t, s] = base[t, s] + scale[a] * B[a]_s (A[a]_s x[t]),   a = the adapter of row t, s = the slices of a fused projection
//
// A step's rows are sorted by adapter once (adapter_rows_kernel) into tiles of rows that share one; every projection of the step runs
// two kernels on those tiles.  The first computes h = A x, [rows, slices x rank], with the K axis cut over workgroups and waves; the
// second adds up the cuts, scales, and computes B h on top of the base rows.  Both products are on the matrix cores.  h stays in float32
// between them and enters the second product as the sum of two 16-bit values (hi + lo), which fill the 32-deep instruction with 16
// ranks: its rounding is 2^-17 of h (bf16) where one value would have 2^-9.
#include <algorithm>

#include "common.h"

namespace {

constexpr int AD_MAX_ADAPTERS = 1024;
constexpr int AD_MAX_RANK = 128;
constexpr int AD_MAX_SLICES = 8;
constexpr int AD_SORT_THREADS = 512, AD_SORT_WAVES = AD_SORT_THREADS / 64;
constexpr int AD_WAVES = 4;
constexpr int AD_GROUP = 64;                                  // columns that a wave computes at a time

struct AdapterSlices {
    int n, total;                                             // slices, columns of all
    int first[AD_MAX_SLICES], width[AD_MAX_SLICES];
};
struct AdapterTile {
    int adapter, first, count, pad;                           // adapter -1: rows without one; count 0: no tile
};

// ---- rows by adapter
int adapter_max_tiles(int64_t tokens, int64_t adapters, int tile) { return (int)(tokens / tile + std::min(tokens, adapters + 1)); }
int64_t adapter_order_ints(int64_t tokens) { return (tokens + 3) / 4 * 4; }

__device__ __forceinline__ void sort_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Lanes of the wave that have this lane's key (bits of it that any key may have: `bits`); lanes without a key are in nobody's.
__device__ __forceinline__ uint64_t same_key(int key, int bits, bool on) {
    uint64_t m = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((key >> b) & 1);
        m &= (key >> b) & 1 ? set : ~set;
    }
    return m;
}

// Counting sort in one workgroup, in the rows' order within an adapter: every wave counts, then places, a piece of the rows of its own.
// Bound by latency, ids, two scans and the placing one behind the other: ids are read 8 x 64 at a time, rows of one adapter among 64
// found by a ballot a bit (one by one, behind atomics of LDS: 5.8 us for 64 rows and 15.6 us for 8191, 4.4 and 7.7 so).
constexpr int AD_BATCH = 8;
__global__ __launch_bounds__(AD_SORT_THREADS) void adapter_rows_kernel(int* __restrict__ order, AdapterTile* __restrict__ tiles,
                                                                       const int* __restrict__ ids, int tokens, int adapters, int tile,
                                                                       int max_tiles, int bits) {
    extern __shared__ int lds[];
    const int n = adapters + 1;                               // the last: rows without an adapter
    int* hist = lds;                                          // [waves][n]
    int* start = hist + AD_SORT_WAVES * n;                    // [n + 1]
    int* tstart = start + n + 1;
    __shared__ int w_rows[AD_SORT_WAVES], w_tiles[AD_SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int piece = ((tokens + AD_SORT_WAVES - 1) / AD_SORT_WAVES + 63) / 64 * 64;
    const int r0 = min(w * piece, tokens), r1 = min(r0 + piece, tokens);
    int key[AD_BATCH];
    auto load = [&](int rb) {
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane, a = r < r1 ? ids[r] : -1;
            key[i] = a >= 0 && a < adapters ? a : adapters;
        }
    };
    load(r0);
    for (int i = tid; i < AD_SORT_WAVES * n; i += AD_SORT_THREADS) hist[i] = 0;
    __syncthreads();
    for (int rb = r0; rb < r1; rb += 64 * AD_BATCH) {
        if (rb != r0) load(rb);
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane;
            if (rb + 64 * i >= r1) break;
            const uint64_t m = same_key(key[i], bits, r < r1);
            sort_fence();
            if (r < r1 && (int)__builtin_ctzll(m) == lane) hist[w * n + key[i]] += __popcll(m);
            sort_fence();
        }
    }
    __syncthreads();
    // each thread: a run of adapters, the waves' counts turned into places within the adapter
    const int each = (n + AD_SORT_THREADS - 1) / AD_SORT_THREADS;
    const int a0 = min(tid * each, n), a1 = min(a0 + each, n);
    int rows = 0, tls = 0;
    for (int a = a0; a < a1; ++a) {
        int c = 0;
        for (int v = 0; v < AD_SORT_WAVES; ++v) {
            const int t = hist[v * n + a];
            hist[v * n + a] = c;
            c += t;
        }
        start[a] = rows;
        tstart[a] = tls;
        rows += c;
        tls += (c + tile - 1) / tile;
    }
    int pr = rows, pt = tls;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(pr, o, 64), y = __shfl_up(pt, o, 64);
        if (lane >= o) { pr += x; pt += y; }
    }
    if (lane == 63) { w_rows[w] = pr; w_tiles[w] = pt; }
    __syncthreads();
    pr -= rows;
    pt -= tls;
    int all_tiles = 0;
    for (int v = 0; v < AD_SORT_WAVES; ++v) {
        if (v < w) { pr += w_rows[v]; pt += w_tiles[v]; }
        all_tiles += w_tiles[v];
    }
    for (int a = a0; a < a1; ++a) { start[a] += pr; tstart[a] += pt; }
    if (tid == 0) start[n] = tokens;
    __syncthreads();
    for (int rb = r0; rb < r1; rb += 64 * AD_BATCH) {
        if (piece > 64 * AD_BATCH) load(rb);                  // otherwise the keys are still there
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane;
            if (rb + 64 * i >= r1) break;
            const uint64_t m = same_key(key[i], bits, r < r1);
            sort_fence();
            const int at = hist[w * n + key[i]];
            if (r < r1) order[start[key[i]] + at + __popcll(m & ((1ull << lane) - 1ull))] = r;
            sort_fence();
            if (r < r1 && (int)__builtin_ctzll(m) == lane) hist[w * n + key[i]] = at + __popcll(m);
            sort_fence();
        }
    }
    for (int i = tid; i < max_tiles; i += AD_SORT_THREADS) {
        AdapterTile t = {-1, 0, 0, 0};
        if (i < all_tiles) {
            int lo = 0, hi = n - 1;                           // the last adapter whose tiles start at or before i
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (tstart[mid] <= i) lo = mid;
                else hi = mid - 1;
            }
            t.adapter = lo < adapters ? lo : -1;
            t.first = start[lo] + (i - tstart[lo]) * tile;
            t.count = min(tile, start[lo + 1] - t.first);
        }
        tiles[i] = t;
    }
}

// ---- the two products
struct AdapterArgs {
    uint16_t* out;
    const uint16_t *x, *a, *b, *base;
    const int* order;
    const AdapterTile* tiles;
    const int* ranks;                                         // null: all of them `rank`
    const float* scales;                                      // null: 1
    float* h;                                                 // [cuts][tokens][slices x rank]
    int64_t x_stride, base_stride, out_stride;
    int tokens, k, rank, cuts, cut_units, blocks;             // cut_units: of 64 columns of x; blocks: of rank tiles
    int max_tiles;
    int groups_each;                                          // column groups of a wave
    int pitch;                                                // 16-bit values of a row of h in LDS
    int vec_io;                                               // base and out rows on 16-byte borders
    AdapterSlices s;
};

__device__ __forceinline__ int adapter_rank(const AdapterArgs& A, int a) { return A.ranks ? min(max(A.ranks[a], 0), A.rank) : A.rank; }

// h of RT x 16 rows and up to CT tiles of 16 ranks (of whatever slices), over one cut of K.  Lane l of a fragment holds rank or row
// l & 15 and 8 values from 8 (l >> 4) on, as both operands lie in memory.  The waves take units of 64 columns in turn, half a unit's
// loads on their way behind the products of the other half, and meet in LDS.  The workgroups that share x (of one tile and cut) run next
// to each other on one XCD.
template <typename T, int RT, int CT>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_shrink_kernel(const AdapterArgs A) {
    constexpr int N = RT * CT, SENT = N % 4 == 0 ? N / 2 : N;
    __shared__ f32x4 red[AD_WAVES][SENT][64];
    const int id = blockIdx.x, turn = id >> 3, item = turn / A.blocks * 8 + (id & 7), z = turn % A.blocks;
    const int cut = item / A.max_tiles;
    if (cut >= A.cuts) return;
    const AdapterTile tile = A.tiles[item - cut * A.max_tiles];
    if (tile.count <= 0 || tile.adapter < 0) return;
    const int rank = adapter_rank(A, tile.adapter);
    const int per = (rank + 15) >> 4, units = per * A.s.n, c0 = z * CT;
    if (c0 >= units) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
    const uint16_t* xr[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) xr[r] = A.x + (int64_t)A.order[tile.first + min(r * 16 + i16, tile.count - 1)] * A.x_stride + 8 * q;
    const uint16_t* ar[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {                            // tiles past the last one, ranks past the adapter's: others once more
        const int u = min(c0 + c, units - 1), s = u / per, row = min((u - s * per) * 16 + i16, rank - 1);
        ar[c] = A.a + ((int64_t)(tile.adapter * A.s.n + s) * A.rank + row) * A.k + 8 * q;
    }
    f32x4 acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int u_end = min((cut + 1) * A.cut_units, (A.k + 63) >> 6);
    const int last = A.k - 8 - 8 * q;                         // where this lane's last whole piece starts
    constexpr int NB = RT == 1 ? 4 : 2;                       // half units on their way
    u32x4 xv[NB][RT], av[NB][CT];
    auto load = [&](int b, int u) {
        const int k = u * 64 + (b & 1) * 32, at = min(k, last);       // last may be negative: then this lane's piece starts in front
#pragma unroll
        for (int r = 0; r < RT; ++r) xv[b][r] = *(const u32x4*)(xr[r] + at);
#pragma unroll
        for (int c = 0; c < CT; ++c) av[b][c] = *(const u32x4*)(ar[c] + at);
    };
    auto product = [&](int b, int u) {
        if (u * 64 + (b & 1) * 32 > last)                     // behind the row's end: nothing
#pragma unroll
            for (int r = 0; r < RT; ++r) xv[b][r] = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int c = 0; c < CT; ++c)
                acc[r * CT + c] = T::mfma16(bitcast<typename T::vec8>(av[b][c]), bitcast<typename T::vec8>(xv[b][r]), acc[r * CT + c]);
    };
    const int u0 = cut * A.cut_units + w;
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (u0 + b / 2 * AD_WAVES < u_end) load(b, u0 + b / 2 * AD_WAVES);
    for (int u = u0; u < u_end; u += NB / 2 * AD_WAVES)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int now = u + b / 2 * AD_WAVES, next = now + NB / 2 * AD_WAVES;
            if (now >= u_end) break;
            product(b, now);
            if (next < u_end) load(b, next);
        }
    const int width = A.s.n * A.rank;
    auto store = [&](int t, const f32x4& v) {
        const int r = t / CT, c = t - r * CT, u = c0 + c;
        if (u >= units) return;
        const int s = u / per, j = (u - s * per) * 16 + 4 * q, row = r * 16 + i16;       // four ranks of a row a lane
        if (row < tile.count && j < A.rank) *(f32x4*)(A.h + ((int64_t)cut * A.tokens + tile.first + row) * width + s * A.rank + j) = v;
    };
    if constexpr (N % 4 == 0) {                               // halves exchanged with wave w ^ 2, halves of those with wave w ^ 1
        f32x4 mine[N / 2], last4[N / 4];
        // (branches, not selections: those would put the accumulators into memory)
        auto exchange = [&](auto n, bool up, const f32x4* v, f32x4* kept, int other) {
            constexpr int H = decltype(n)::value;
            if (up) {
#pragma unroll
                for (int i = 0; i < H; ++i) { red[w][i][lane] = v[i]; kept[i] = v[H + i]; }
            } else {
#pragma unroll
                for (int i = 0; i < H; ++i) { red[w][i][lane] = v[H + i]; kept[i] = v[i]; }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < H; ++i) kept[i] += red[other][i][lane];
            __syncthreads();
        };
        exchange(std::integral_constant<int, N / 2>{}, w & 2, acc, mine, w ^ 2);
        exchange(std::integral_constant<int, N / 4>{}, w & 1, mine, last4, w ^ 1);
        const int t0 = (w & 2 ? N / 2 : 0) + (w & 1 ? N / 4 : 0);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) store(t0 + i, last4[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) red[w][i][lane] = acc[i];
        __syncthreads();
        for (int t = w; t < N; t += AD_WAVES) {
            f32x4 v = red[0][t][lane];
#pragma unroll
            for (int o = 1; o < AD_WAVES; ++o) v += red[o][t][lane];
            store(t, v);
        }
    }
}

// out = base + (B h) for groups of 64 columns of one slice and RT x 16 rows, h in LDS as hi and lo planes [2][RT x 16][pitch].  The product
// is taken with the columns as the matrix instruction's rows, in an order that leaves a lane twice 8 columns side by side of one
// row: base and out move in 16 bytes a lane, 64 a row and instruction.  A group's base rows and first two rank tiles are loaded
// behind the group before it.
template <typename T, int RT>
struct ColumnGroups {
    const AdapterArgs& A;
    int adapter, count, rank, per, first, cols, q, i16;
    int rows[RT];
    u32x4 bv[2][4], raw[RT][2];

    __device__ __forceinline__ ColumnGroups(const AdapterArgs& args, const AdapterTile& tile, int rk, int s)
        : A(args), adapter(tile.adapter), count(tile.count), rank(rk), per((rk + 15) >> 4), first(args.s.first[s]), cols(args.s.width[s]),
          q((threadIdx.x & 63) >> 4), i16(threadIdx.x & 15) {
#pragma unroll
        for (int r = 0; r < RT; ++r) rows[r] = A.order[tile.first + min(r * 16 + i16, count - 1)];
    }
    __device__ __forceinline__ bool whole(int c0) const { return A.vec_io && c0 + AD_GROUP <= cols && (first & 7) == 0; }
    __device__ __forceinline__ void load_b(int b, int c0, int t) {    // rank tile t of the group's columns, 8 ranks a lane
        const int k = min(t * 16 + 8 * (q & 1), A.rank - 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = min(c0 + (j >> 1) * 32 + (i16 >> 2) * 8 + (j & 1) * 4 + (i16 & 3), cols - 1);
            bv[b][j] = *(const u32x4*)(A.b + ((int64_t)adapter * A.s.total + first + n) * A.rank + k);
        }
    }
    __device__ __forceinline__ void load(int c0) {
        if (rank) {
            load_b(0, c0, 0);
            if (per > 1) load_b(1, c0, 1);
        }
        if (whole(c0))
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    raw[r][p] = *(const u32x4*)(A.base + (int64_t)rows[r] * A.base_stride + first + c0 + 32 * p + 8 * q);
    }
    // groups from column c0 on, `step` columns apart, up to `end`; load(c0) has been called
    __device__ __forceinline__ void run(int c0, int step, int end, const uint16_t* planes, int pitch, const float* factor) {
        const uint16_t* mine = planes + (((threadIdx.x & 63) >> 5) * RT * 16 + i16) * pitch + 8 * (q & 1);
        float f[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) f[r] = rank ? factor[r * 16 + i16] : 0.f;
        for (; c0 < end; c0 += step) {
            f32x4 acc[RT][4];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
            auto product = [&](int b, int t) {
                const int left = rank - (t * 16 + 8 * (q & 1));
                if (t == per - 1 && (rank & 15)) {            // behind the adapter's rank, whatever lies there
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) bv[b][j][e] &= left >= 2 * e + 2 ? 0xffffffffu : left == 2 * e + 1 ? 0xffffu : 0u;
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const u32x4 hv = *(const u32x4*)(mine + r * 16 * pitch + t * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[r][j] = T::mfma16(bitcast<typename T::vec8>(bv[b][j]), bitcast<typename T::vec8>(hv), acc[r][j]);
                }
            };
            for (int t = 0; t < per; t += 2) {
                product(0, t);
                if (t + 2 < per) load_b(0, c0, t + 2);
                if (t + 1 < per) {
                    product(1, t + 1);
                    if (t + 3 < per) load_b(1, c0, t + 3);
                }
            }
            const bool vec = whole(c0);
            u32x4 had[RT][2];
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = 0; p < 2; ++p) had[r][p] = raw[r][p];
            if (c0 + step < end) load(c0 + step);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if (r * 16 + i16 >= count) continue;
                uint16_t* out = A.out + (int64_t)rows[r] * A.out_stride + first + c0 + 8 * q;
                if (vec) {
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        float x[8];
                        unpack8<T>(had[r][p], x);
                        u32x4 o = had[r][p];
                        if (rank)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[e] = pack2<T>(fmaf(acc[r][2 * p + (e >> 1)][2 * (e & 1)], f[r], x[2 * e]),
                                                fmaf(acc[r][2 * p + (e >> 1)][2 * (e & 1) + 1], f[r], x[2 * e + 1]));
                        *(u32x4*)(out + 32 * p) = o;
                    }
                } else {
                    const uint16_t* base = A.base + (int64_t)rows[r] * A.base_stride + first + c0 + 8 * q;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int at = (e >> 3) * 32 + (e & 7);
                        if (c0 + 8 * q + at < cols)
                            out[at] = rank ? T::from_float(fmaf(acc[r][e >> 2][e & 3], f[r], T::to_float(base[at]))) : base[at];
                    }
                }
            }
        }
    }
};

// A row of h, scaled, to the planes: sixteen lanes a row, v[i] the ranks 64 i + 4 (lane & 15) .. + 3 of it; what lies at or behind the
// adapter's rank becomes zero.  `factor` gets what the products of the row are to be multiplied with.
template <typename T>
__device__ __forceinline__ void row_to_planes(f32x4* v, float scale, int rank, int row, int rows, uint16_t* planes, int pitch, float* factor) {
    constexpr int NV = AD_MAX_RANK / 64;
    const int i16 = threadIdx.x & 15;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[i][e] = 64 * i + 4 * i16 + e < rank ? v[i][e] * scale : 0.f;
            most = fmaxf(most, fabsf(v[i][e]));
        }
    float up = 1.f, down = 1.f;
    if constexpr (std::is_same_v<T, FP16>) {                  // h may pass the range of fp16: rows go in with a power of two
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        if (most > 0.f && most < INFINITY) {
            const int e = min(max(14 - ilogbf(most), -120), 120);
            up = ldexpf(1.f, e);
            down = ldexpf(1.f, -e);
        }
    }
    if (i16 == 0) factor[row] = down;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = 64 * i + 4 * i16;
        if (j >= (rank + 15) / 16 * 16) continue;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float a = v[i][2 * e] * up, b = v[i][2 * e + 1] * up;
            hi[e] = pack2<T>(a, b);
            const float ra = a - T::to_float((uint16_t)hi[e]), rb = b - T::to_float((uint16_t)(hi[e] >> 16));
            lo[e] = pack2<T>(fabsf(ra) < INFINITY ? ra : 0.f, fabsf(rb) < INFINITY ? rb : 0.f);      // infinite: hi says it
        }
        *(u32x2*)(planes + row * pitch + j) = (u32x2){hi[0], hi[1]};
        *(u32x2*)(planes + (rows + row) * pitch + j) = (u32x2){lo[0], lo[1]};
    }
}

// the slice that a block of columns lies in; block becomes its number there
__device__ __forceinline__ int slice_of(const AdapterArgs& A, int& block, int block_cols) {
    int s = 0;
    for (;; ++s) {
        const int n = (A.s.width[s] + block_cols - 1) / block_cols;
        if (block < n) return s;
        block -= n;
    }
}

// The second product by itself: a workgroup adds up the cuts of its rows' h and computes 4 x groups_each groups of columns.  The first
// group's loads are in front of those of h.
template <typename T, int RT>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_expand_kernel(const AdapterArgs A) {
    constexpr int ROWS = RT * 16, NV = AD_MAX_RANK / 64;
    extern __shared__ __align__(16) uint16_t planes[];
    __shared__ float factor[ROWS];
    const AdapterTile tile = A.tiles[blockIdx.x];
    if (tile.count <= 0) return;
    const int rank = tile.adapter < 0 ? 0 : adapter_rank(A, tile.adapter);
    if (rank == 0 && A.out == A.base) return;
    int block = blockIdx.y;
    const int block_cols = AD_GROUP * AD_WAVES * A.groups_each, s = slice_of(A, block, block_cols);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
    const int width = A.s.n * A.rank;
    ColumnGroups<T, RT> groups(A, tile, rank, s);
    const int c0 = block * block_cols + w * AD_GROUP, end = min((block + 1) * block_cols, groups.cols);
    if (c0 < end) groups.load(c0);
    if (rank) {
        const float scale = A.scales ? A.scales[tile.adapter] : 1.f;
        f32x4 v[RT][NV];
        const int64_t cut = (int64_t)A.tokens * width;
#pragma unroll
        for (int i = 0; i < NV; ++i) {                        // sixteen lanes a row, four ranks a lane
            const int j = 64 * i + 4 * i16;
#pragma unroll
            for (int r = 0; r < RT; ++r) v[r][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (j >= rank) continue;
            const float* h = A.h + (int64_t)tile.first * width + s * A.rank + j;
            for (int c = 0; c < A.cuts; c += 4) {
                f32x4 part[RT][4];
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int o = 0; o < 4; ++o)
                        part[r][o] = *(const f32x4*)(h + min((r * AD_WAVES + w) * 4 + q, tile.count - 1) * (int64_t)width + min(c + o, A.cuts - 1) * cut);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int o = 0; o < 4; ++o)
                        if (c + o < A.cuts) v[r][i] += part[r][o];
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) row_to_planes<T>(v[r], scale, rank, (r * AD_WAVES + w) * 4 + q, ROWS, planes, A.pitch, factor);
    }
    __syncthreads();
    groups.run(c0, AD_GROUP * AD_WAVES, end, planes, A.pitch, factor);
}

// How the products are cut.  Tiles of ranks a workgroup: as few workgroups that share x as the registers of RT x CT accumulators allow, evenly
// filled.  Cuts of K: 1024 workgroups where there is that much, four units a wave and cut at least; a cut is another float32 copy of h.
// Groups of columns a wave: more than one, so that the sums of h are shared, while 512 workgroups are left.
struct AdapterPlan {
    int cuts, cut_units, blocks, ct, groups_each;
};
AdapterPlan adapter_plan(int tokens, int adapters, int tile, int k, int slices, int rank, const int32_t* widths) {
    AdapterPlan p;
    const int units = slices * ((rank + 15) / 16), most = tile == 16 ? 4 : 6;
    p.blocks = (units + most - 1) / most;
    p.ct = (units + p.blocks - 1) / p.blocks;
    if (p.ct == 5) p.ct = 6;
    const int k_units = (k + 63) / 64;
    const int64_t tiles = std::min<int64_t>(adapter_max_tiles(tokens, adapters, tile), tokens);
    const int64_t want = (1024 + tiles * p.blocks - 1) / (tiles * p.blocks);
    const int cuts = (int)std::min<int64_t>(std::min<int64_t>(want, 8), std::max(1, k_units / (4 * AD_WAVES)));
    p.cut_units = (k_units + cuts - 1) / cuts;
    p.cuts = (k_units + p.cut_units - 1) / p.cut_units;
    p.groups_each = 1;
    for (; widths && p.groups_each < 4; p.groups_each *= 2) {
        int64_t blocks = 0;
        for (int i = 0; i < slices; ++i) blocks += (widths[i] + 2 * p.groups_each * AD_GROUP * AD_WAVES - 1) / (2 * p.groups_each * AD_GROUP * AD_WAVES);
        if (blocks * tiles < 512) break;
    }
    return p;
}

}  // namespace

extern "C" int64_t mf_adapter_rows_ints(int tokens, int adapters, int tile) {
    if (tokens <= 0 || adapters < 0 || (tile != 16 && tile != 64)) return 0;
    return adapter_order_ints(tokens) + 4ll * adapter_max_tiles(tokens, adapters, tile);
}

extern "C" int mf_adapter_rows(int32_t* plan, const int32_t* adapter_ids, int tokens, int adapters, int tile, void* stream) {
    MF_REQUIRE(tokens >= 0 && adapters >= 0 && adapters <= AD_MAX_ADAPTERS, "adapter_rows: up to %d adapters, got %d", AD_MAX_ADAPTERS, adapters);
    MF_REQUIRE(tokens <= (1 << 20), "adapter_rows: up to 2^20 rows, got %d", tokens);
    MF_REQUIRE(tile == 16 || tile == 64, "adapter_rows: tiles of 16 or 64 rows, got %d", tile);
    if (tokens == 0) return 0;
    MF_REQUIRE(plan && adapter_ids && ((uintptr_t)plan & 15) == 0, "adapter_rows: null or unaligned argument");
    const size_t lds = sizeof(int) * (size_t)((AD_SORT_WAVES + 2) * (adapters + 1) + 2);
    hipLaunchKernelGGL(adapter_rows_kernel, dim3(1), dim3(AD_SORT_THREADS), lds, (hipStream_t)stream, plan,
                       (AdapterTile*)(plan + adapter_order_ints(tokens)), adapter_ids, tokens, adapters, tile,
                       adapter_max_tiles(tokens, adapters, tile), 32 - __builtin_clz((unsigned)adapters | 1u));
    return MF_LAUNCH_CHECK();
}

extern "C" size_t mf_adapter_workspace_bytes(int tokens, int adapters, int tile, int k, int slices, int rank) {
    if (tokens <= 0 || adapters <= 0 || (tile != 16 && tile != 64) || k <= 0 || slices <= 0 || slices > AD_MAX_SLICES || rank <= 0 ||
        rank > AD_MAX_RANK)
        return 0;
    return sizeof(float) * (size_t)adapter_plan(tokens, adapters, tile, k, slices, rank, nullptr).cuts * tokens * slices * rank;
}

extern "C" int mf_adapter_linear(void* out, const void* x, const void* lora_a, const void* lora_b, const void* base, const int32_t* plan,
                                 const int32_t* ranks, const float* scales, const int32_t* host_widths, int slices, int tokens,
                                 int adapters, int tile, int k, int rank, int64_t x_row_stride, int64_t base_row_stride,
                                 int64_t out_row_stride, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    MF_REQUIRE(dtype == MF_BF16 || dtype == MF_FP16, "adapter_linear: dtype must be bf16 or fp16");
    MF_REQUIRE(tokens >= 0 && tokens <= (1 << 20) && adapters > 0 && adapters <= AD_MAX_ADAPTERS, "adapter_linear: up to 2^20 rows and %d adapters",
               AD_MAX_ADAPTERS);
    MF_REQUIRE(tile == 16 || tile == 64, "adapter_linear: tiles of 16 or 64 rows, got %d", tile);
    MF_REQUIRE(k > 0 && k % 8 == 0 && rank > 0 && rank % 8 == 0 && rank <= AD_MAX_RANK,
               "adapter_linear: input width %d and rank %d must be multiples of 8, the rank up to %d", k, rank, AD_MAX_RANK);
    MF_REQUIRE(host_widths && slices > 0 && slices <= AD_MAX_SLICES, "adapter_linear: 1 to %d slices, got %d", AD_MAX_SLICES, slices);
    AdapterArgs A = {};
    int64_t columns = 0;
    A.s.n = slices;
    for (int i = 0; i < slices; ++i) {
        MF_REQUIRE(host_widths[i] > 0, "adapter_linear: slice %d is %d wide", i, host_widths[i]);
        A.s.first[i] = (int)columns;
        A.s.width[i] = host_widths[i];
        columns += host_widths[i];
        MF_REQUIRE(columns <= (1 << 24), "adapter_linear: more than 2^24 columns");
    }
    if (tokens == 0) return 0;
    A.s.total = (int)columns;
    A.x_stride = x_row_stride > 0 ? x_row_stride : k;
    A.base_stride = base_row_stride > 0 ? base_row_stride : columns;
    A.out_stride = out_row_stride > 0 ? out_row_stride : columns;
    MF_REQUIRE(A.x_stride >= k && A.base_stride >= columns && A.out_stride >= columns, "adapter_linear: rows overlap");
    MF_REQUIRE(out != base || A.out_stride == A.base_stride, "adapter_linear: out is base with rows of another distance");
    MF_REQUIRE(out && x && lora_a && lora_b && base && plan, "adapter_linear: null argument");
    MF_REQUIRE((((uintptr_t)x | (uintptr_t)lora_a | (uintptr_t)lora_b | (uintptr_t)plan) & 15) == 0 && A.x_stride % 8 == 0,
               "adapter_linear: x, its rows, the adapters and the plan must lie on 16-byte borders");
    MF_REQUIRE((((uintptr_t)out | (uintptr_t)base) & 1) == 0, "adapter_linear: out and base must be aligned to their type");
    const AdapterPlan p = adapter_plan(tokens, adapters, tile, k, slices, rank, host_widths);
    const size_t need = sizeof(float) * (size_t)p.cuts * tokens * slices * rank;
    MF_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
               "adapter_linear: 16-byte aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    A.out = (uint16_t*)out, A.x = (const uint16_t*)x, A.a = (const uint16_t*)lora_a, A.b = (const uint16_t*)lora_b;
    A.base = (const uint16_t*)base, A.order = plan, A.tiles = (const AdapterTile*)(plan + adapter_order_ints(tokens));
    A.ranks = ranks, A.scales = scales, A.h = (float*)workspace;
    A.tokens = tokens, A.k = k, A.rank = rank, A.cuts = p.cuts, A.cut_units = p.cut_units, A.groups_each = p.groups_each;
    A.vec_io = ((((uintptr_t)out | (uintptr_t)base) & 15) == 0 && A.base_stride % 8 == 0 && A.out_stride % 8 == 0) ? 1 : 0;
    hipStream_t st = (hipStream_t)stream;
    const int tiles = adapter_max_tiles(tokens, adapters, tile);
    const size_t lds = (size_t)2 * tile * ((rank + 15) / 16 * 16 + 8) * 2;
    const int block_cols = AD_GROUP * AD_WAVES * p.groups_each;
    int64_t col_blocks = 0;
    for (int i = 0; i < slices; ++i) col_blocks += (A.s.width[i] + block_cols - 1) / block_cols;
    MF_REQUIRE(col_blocks <= 65535, "adapter_linear: %lld columns", (long long)columns);
    A.max_tiles = tiles, A.blocks = p.blocks, A.pitch = (rank + 15) / 16 * 16 + 8;
    const int64_t shrinks = ((int64_t)tiles * p.cuts + 7) / 8 * 8 * p.blocks;
    MF_REQUIRE(shrinks < (1 << 24), "adapter_linear: %lld workgroups", (long long)shrinks);
    const dim3 g1((unsigned)shrinks);
#define AD_SHRINK(T, RT, CT) hipLaunchKernelGGL((adapter_shrink_kernel<T, RT, CT>), g1, dim3(AD_WAVES * 64), 0, st, A)
#define AD_SHRINK_T(T)                                \
    do {                                              \
        if (tile == 16) {                             \
            if (p.ct == 1) AD_SHRINK(T, 1, 1);        \
            else if (p.ct == 2) AD_SHRINK(T, 1, 2);   \
            else if (p.ct == 3) AD_SHRINK(T, 1, 3);   \
            else AD_SHRINK(T, 1, 4);                  \
        } else {                                      \
            if (p.ct == 1) AD_SHRINK(T, 4, 1);        \
            else if (p.ct == 2) AD_SHRINK(T, 4, 2);   \
            else if (p.ct == 3) AD_SHRINK(T, 4, 3);   \
            else if (p.ct == 4) AD_SHRINK(T, 4, 4);   \
            else AD_SHRINK(T, 4, 6);                  \
        }                                             \
    } while (0)
    if (dtype == MF_BF16) AD_SHRINK_T(BF16);
    else AD_SHRINK_T(FP16);
#undef AD_SHRINK_T
#undef AD_SHRINK
    const int rc = MF_LAUNCH_CHECK();
    if (rc) return rc;
    const dim3 g2((unsigned)tiles, (unsigned)col_blocks);
#define AD_EXPAND(T, RT) hipLaunchKernelGGL((adapter_expand_kernel<T, RT>), g2, dim3(AD_WAVES * 64), lds, st, A)
    if (dtype == MF_BF16) {
        if (tile == 16) AD_EXPAND(BF16, 1);
        else AD_EXPAND(BF16, 4);
    } else {
        if (tile == 16) AD_EXPAND(FP16, 1);
        else AD_EXPAND(FP16, 4);
    }
#undef AD_EXPAND
    return MF_LAUNCH_CHECK();
}
