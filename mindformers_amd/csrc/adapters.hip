// Low-rank adapters of many requests beside a projection that they share:
//
//   out[t, s] = base[t, s] + scale[a] * B[a]_s (A[a]_s x[t]),   a = the adapter of row t, s = the slices of a fused projection
//
// A step's rows are sorted by adapter once (adapter_rows_kernel) into tiles of rows that share one; every projection of the step runs
// two kernels on those tiles (a single row one kernel, adapter_row_kernel).  The first computes h = A x, [rows, slices x rank], with the K axis cut over workgroups and waves; the
// second adds up the cuts, scales, and computes B h on top of the base rows.  Both products are on the matrix cores.  h stays in float32
// between them and enters the second product as the sum of two 16-bit values (hi + lo), which fill the 32-deep instruction with 16
// ranks: its rounding is 2^-17 of h (bf16) where one value would have 2^-9.
#include <algorithm>

#include "common.h"

namespace {

constexpr int AD_MAX_ADAPTERS = 1024;
constexpr int AD_MAX_RANK = 128;
constexpr int AD_MAX_SLICES = 8;
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

// Lanes of the wave that have this lane's key (bits of it that any key may have: `bits`); lanes without a key are in nobody's.  Prompts
// have one key a wave.
__device__ __forceinline__ uint64_t same_key(int key, int bits, bool on) {
    uint64_t m = __ballot(on);
    if (__ballot(on && key != __builtin_amdgcn_readfirstlane(key)) == 0) return m;
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((key >> b) & 1);
        m &= (key >> b) & 1 ? set : ~set;
    }
    return m;
}

// Counting sort in one workgroup, in the rows' order within an adapter: every wave counts, then places, a piece of the rows of its own.
// Bound by latency, ids, two scans and the placing one behind the other: ids are read 8 x 64 at a time, rows of one adapter among 64
// found by a ballot a bit, and one lane of theirs adds them to the wave's count; no such addition waits for the one before it.  (With
// the gap behind it, 64 rows 5.4 us and 8191 rows 8.0; counts read, waited for and written 5.8 and 10.8.)
constexpr int AD_BATCH = 8;
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void adapter_rows_kernel(int* __restrict__ order, AdapterTile* __restrict__ tiles,
                                                                       const int* __restrict__ ids, int tokens, int adapters, int tile,
                                                                       int max_tiles, int bits) {
    constexpr int THREADS = WAVES * 64;
    extern __shared__ int lds[];
    const int n = adapters + 1;                               // the last: rows without an adapter
    int* hist = lds;                                          // [waves][n]
    int* start = hist + WAVES * n;                    // [n + 1]
    int* tstart = start + n + 1;
    __shared__ int w_rows[WAVES], w_tiles[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int piece = ((tokens + WAVES - 1) / WAVES + 63) / 64 * 64;
    const int r0 = min(w * piece, tokens), r1 = min(r0 + piece, tokens);
    int key[AD_BATCH];
    uint64_t same[AD_BATCH];
    auto load = [&](int rb) {
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane, a = r < r1 ? ids[r] : -1;
            key[i] = a >= 0 && a < adapters ? a : adapters;
        }
    };
    load(r0);
    for (int i = tid; i < WAVES * n; i += THREADS) hist[i] = 0;
    __syncthreads();
    for (int rb = r0; rb < r1; rb += 64 * AD_BATCH) {
        if (rb != r0) load(rb);
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane;
            if (rb + 64 * i >= r1) break;
            same[i] = same_key(key[i], bits, r < r1);
            if (r < r1 && (int)__builtin_ctzll(same[i]) == lane) atomicAdd(&hist[w * n + key[i]], __popcll(same[i]));
        }
    }
    __syncthreads();
    // each thread: a run of adapters, the waves' counts turned into places within the adapter
    const int each = (n + THREADS - 1) / THREADS;
    const int a0 = min(tid * each, n), a1 = min(a0 + each, n);
    int rows = 0, tls = 0;
    for (int a = a0; a < a1; ++a) {
        int c = 0, of[WAVES];
#pragma unroll
        for (int v = 0; v < WAVES; ++v) of[v] = hist[v * n + a];
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            hist[v * n + a] = c;
            c += of[v];
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
    for (int v = 0; v < WAVES; ++v) {
        if (v < w) { pr += w_rows[v]; pt += w_tiles[v]; }
        all_tiles += w_tiles[v];
    }
    for (int a = a0; a < a1; ++a) { start[a] += pr; tstart[a] += pt; }
    if (tid == 0) start[n] = tokens;
    __syncthreads();
    for (int rb = r0; rb < r1; rb += 64 * AD_BATCH) {
        const bool again = piece > 64 * AD_BATCH;             // otherwise the keys are still there
        if (again) load(rb);
        int at[AD_BATCH] = {};
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {                  // (a wave's LDS operations take place in order)
            const int r = rb + 64 * i + lane;
            if (rb + 64 * i >= r1) break;
            if (again) same[i] = same_key(key[i], bits, r < r1);
            if (r < r1 && (int)__builtin_ctzll(same[i]) == lane) at[i] = atomicAdd(&hist[w * n + key[i]], __popcll(same[i]));
            sort_fence();
        }
#pragma unroll
        for (int i = 0; i < AD_BATCH; ++i) {
            const int r = rb + 64 * i + lane;
            if (rb + 64 * i >= r1) break;
            const int first = __shfl(at[i], (int)__builtin_ctzll(same[i]), 64);
            if (r < r1) order[start[key[i]] + first + __popcll(same[i] & ((1ull << lane) - 1ull))] = r;
        }
    }
    for (int i = tid; i < max_tiles; i += THREADS) {
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
    int max_tiles, subs;                                      // subs: pieces of a tile that the second product takes
    int groups_each, col_blocks;                              // column groups of a wave, workgroups of a row
    int pitch;                                                // 16-bit values of a row of h in LDS
    int vec_io;                                               // base and out rows on 16-byte borders
    AdapterSlices s;
};

__device__ __forceinline__ int adapter_rank(const AdapterArgs& A, int a) { return A.ranks ? min(max(A.ranks[a], 0), A.rank) : A.rank; }

// h of RT x 16 rows and up to CT tiles of 16 ranks (of whatever slices), over one cut of K.  The waves take units of 64 columns in turn
// and meet in LDS.  A wave's unit goes through LDS of its own: it is loaded 8 lanes a row, as it lies in memory, and read back as the
// matrix instruction wants it, a row a lane (loaded that way, every four lanes name four cache lines, and the vector memory unit takes
// as many turns: 16 bytes a clock and compute unit).  The next unit is on its way meanwhile.  The workgroups that share x (of one tile
// and cut) run next to each other on one XCD.
template <typename T, int RT, int CT>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_shrink_kernel(const AdapterArgs A) {
    constexpr int N = RT * CT, ROWS = (RT + CT) * 16, SENT = N % 4 == 0 ? N / 2 : N;
    static_assert(SENT * 64 <= ROWS * 8, "the waves' sums go where their units were");
    __shared__ u32x4 stage[AD_WAVES][ROWS * 8];               // rows of 8 pieces of 16 bytes, piece p of row r at p ^ (r & 7)
    const int id = blockIdx.x, turn = id >> 3, item = turn / A.blocks * 8 + (id & 7), z = turn % A.blocks;
    const int cut = item / A.max_tiles;
    if (cut >= A.cuts) return;
    const AdapterTile tile = A.tiles[item - cut * A.max_tiles];
    if (tile.count <= 0 || tile.adapter < 0) return;
    const int rank = adapter_rank(A, tile.adapter);
    const int per = (rank + 15) >> 4, units = per * A.s.n, c0 = z * CT;
    if (c0 >= units) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
    const int r8 = lane >> 3, p8 = lane & 7;
    const uint16_t* xr[2 * RT];
#pragma unroll
    for (int r = 0; r < 2 * RT; ++r) xr[r] = A.x + (int64_t)A.order[tile.first + min(r * 8 + r8, tile.count - 1)] * A.x_stride;
    const uint16_t* a0 = A.a + (int64_t)tile.adapter * A.s.n * A.rank * A.k;
    int64_t ar[2 * CT];
#pragma unroll
    for (int c = 0; c < 2 * CT; ++c) {                        // tiles past the last one, ranks past the adapter's: others once more
        const int u = min(c0 + c / 2, units - 1), s = u / per, row = min((u - s * per) * 16 + (c & 1) * 8 + r8, rank - 1);
        ar[c] = (int64_t)(s * A.rank + row) * A.k;
    }
    f32x4 acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int u_end = min((cut + 1) * A.cut_units, (A.k + 63) >> 6);
    u32x4 in[2 * (RT + CT)];
    auto load = [&](int u) {
        const int k = u * 64 + 8 * p8, at = min(k, A.k - 8);
#pragma unroll
        for (int c = 0; c < 2 * CT; ++c) in[2 * RT + c] = *(const u32x4*)(a0 + ar[c] + at);
#pragma unroll
        for (int r = 0; r < 2 * RT; ++r) in[r] = *(const u32x4*)(xr[r] + at);
        if (k != at)                                          // behind the row's end: nothing
#pragma unroll
            for (int r = 0; r < 2 * RT; ++r) in[r] = (u32x4){0, 0, 0, 0};
    };
    u32x4* mine = stage[w];
    int u = cut * A.cut_units + w;
    if (u < u_end) load(u);
    for (; u < u_end; u += AD_WAVES) {
        sort_fence();                                         // (a wave's LDS operations take place in order)
#pragma unroll
        for (int i = 0; i < 2 * (RT + CT); ++i) mine[(i * 8 + r8) * 8 + (p8 ^ r8)] = in[i];
        sort_fence();
        if (u + AD_WAVES < u_end) load(u + AD_WAVES);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4 xv[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) xv[r] = mine[(r * 16 + i16) * 8 + ((4 * half + q) ^ (i16 & 7))];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const u32x4 av = mine[((RT + c) * 16 + i16) * 8 + ((4 * half + q) ^ (i16 & 7))];
#pragma unroll
                for (int r = 0; r < RT; ++r)
                    acc[r * CT + c] = T::mfma16(bitcast<typename T::vec8>(av), bitcast<typename T::vec8>(xv[r]), acc[r * CT + c]);
            }
        }
    }
    __syncthreads();
    u32x4(*red)[ROWS * 8] = stage;                            // float32 from here on
    const int width = A.s.n * A.rank;
    auto store = [&](int t, const f32x4& v) {
        const int r = t / CT, c = t - r * CT, u = c0 + c;
        if (u >= units) return;
        const int s = u / per, j = (u - s * per) * 16 + 4 * q, row = r * 16 + i16;       // four ranks of a row a lane
        if (row < tile.count && j < A.rank) *(f32x4*)(A.h + ((int64_t)cut * A.tokens + tile.first + row) * width + s * A.rank + j) = v;
    };
    if constexpr (N % 4 == 0) {                               // halves exchanged with wave w ^ 2, halves of those with wave w ^ 1
        f32x4 half[N / 2], quarter[N / 4];
        // (branches, not selections: those would put the accumulators into memory)
        auto exchange = [&](auto n, bool up, const f32x4* v, f32x4* kept, int other) {
            constexpr int H = decltype(n)::value;
            if (up) {
#pragma unroll
                for (int i = 0; i < H; ++i) { red[w][i * 64 + lane] = bitcast<u32x4>(v[i]); kept[i] = v[H + i]; }
            } else {
#pragma unroll
                for (int i = 0; i < H; ++i) { red[w][i * 64 + lane] = bitcast<u32x4>(v[H + i]); kept[i] = v[i]; }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < H; ++i) kept[i] += bitcast<f32x4>(red[other][i * 64 + lane]);
            __syncthreads();
        };
        exchange(std::integral_constant<int, N / 2>{}, w & 2, acc, half, w ^ 2);
        exchange(std::integral_constant<int, N / 4>{}, w & 1, half, quarter, w ^ 1);
        const int t0 = (w & 2 ? N / 2 : 0) + (w & 1 ? N / 4 : 0);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) store(t0 + i, quarter[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) red[w][i * 64 + lane] = bitcast<u32x4>(acc[i]);
        __syncthreads();
        for (int t = w; t < N; t += AD_WAVES) {
            f32x4 v = bitcast<f32x4>(red[0][t * 64 + lane]);
#pragma unroll
            for (int o = 1; o < AD_WAVES; ++o) v += bitcast<f32x4>(red[o][t * 64 + lane]);
            store(t, v);
        }
    }
}

// A row of h, scaled, to the planes: sixteen lanes a row, v[i] the ranks 64 i + 4 (lane & 15) .. + 3 of it; what lies at or behind the
// adapter's rank becomes zero.  `factor` gets what the products of the row are to be multiplied with.
template <typename T>
__device__ __forceinline__ void row_to_planes(f32x4* v, float scale, int rank, int row, uint16_t* planes, int pitch, float* factor) {
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
        if (j >= (rank + 31) / 32 * 32) continue;
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float a = v[i][2 * e] * up, b = v[i][2 * e + 1] * up;
            hi[e] = pack2<T>(a, b);
            const float ra = a - T::to_float((uint16_t)hi[e]), rb = b - T::to_float((uint16_t)(hi[e] >> 16));
            lo[e] = pack2<T>(fabsf(ra) < INFINITY ? ra : 0.f, fabsf(rb) < INFINITY ? rb : 0.f);      // infinite: hi says it
        }
        *(u32x2*)(planes + row * pitch + j) = (u32x2){hi[0], hi[1]};
        *(u32x2*)(planes + (16 + row) * pitch + j) = (u32x2){lo[0], lo[1]};
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

// out = base + (B h): a workgroup adds up the cuts of 16 rows' h, puts them into LDS as hi and lo, and computes 4 x groups_each groups
// of 64 columns of one slice.  The product is taken with the columns as the matrix instruction's rows, 32 ranks at a time, once with hi
// and once with lo; its results go through LDS (of the wave's own) into rows of 128 bytes, eight lanes each, as base and out are moved.  A
// group's first 64 ranks of B and its base rows are loaded behind the products and the results of the group before it, the first one's
// in front of the sums of h (two groups ahead: no faster).  Workgroups go along the rows: over rows first, 2% slower, their pieces
// of 2 KB lying a row apart.  Of 8191 rows of three adapters of rank 32, 6144 and 4096 columns, it takes 48 and 35 us, a copy of base to out
// 39 and 27: every 16 rows load their columns' B anew, with 32 ranks as many bytes as base and out.
constexpr int AD_PITCH = AD_GROUP + 4;                        // floats of a row of results
template <typename T>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_expand_kernel(const AdapterArgs A) {
    constexpr int ROWS = 16, NV = AD_MAX_RANK / 64;
    extern __shared__ __align__(16) uint16_t planes[];        // [2][ROWS][pitch]
    __shared__ __align__(16) float turned[AD_WAVES][16 * AD_PITCH];
    __shared__ float factor[ROWS];                            // what a row's products are to be multiplied with
    int block = blockIdx.x % A.col_blocks;
    const int piece = blockIdx.x / A.col_blocks, sub = piece % A.subs;
    AdapterTile tile = A.tiles[piece / A.subs];
    tile.first += sub * ROWS;
    tile.count = min(tile.count - sub * ROWS, ROWS);
    if (tile.count <= 0) return;
    const int rank = tile.adapter < 0 ? 0 : adapter_rank(A, tile.adapter);
    if (rank == 0 && A.out == A.base) return;
    const int block_cols = AD_GROUP * AD_WAVES * A.groups_each;
    const int s = slice_of(A, block, block_cols);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
    const int r8 = lane >> 3, p8 = lane & 7;
    const int per = (rank + 31) >> 5, width = A.s.n * A.rank, first = A.s.first[s], cols = A.s.width[s];
    const int start = block * block_cols + w * AD_GROUP;
    const int end = min((block + 1) * block_cols, cols);
    int rows[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) rows[r] = A.order[tile.first + min(r * 8 + r8, tile.count - 1)];
    u32x4 bv[2][4], raw[2];
    const uint16_t* b0 = A.b + ((int64_t)max(tile.adapter, 0) * A.s.total + first) * A.rank;
    auto load_b = [&](int c0, int b, int t) {                 // 32 ranks of the group's columns
        const int k = min(t * 32 + 8 * q, A.rank - 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) bv[b][j] = *(const u32x4*)(b0 + (int64_t)min(c0 + 16 * j + i16, cols - 1) * A.rank + k);
    };
    auto whole = [&](int c0) { return A.vec_io && (first & 7) == 0 && c0 + 8 * p8 + 8 <= cols; };
    auto load_first_b = [&](int c0) {
        if (rank) load_b(c0, 0, 0);
        if (per > 1) load_b(c0, 1, 1);
    };
    auto load_base = [&](int c0) {
        if (whole(c0))
#pragma unroll
            for (int r = 0; r < 2; ++r) raw[r] = *(const u32x4*)(A.base + (int64_t)rows[r] * A.base_stride + first + c0 + 8 * p8);
    };
    if (start < end) {
        load_first_b(start);
        load_base(start);
    }
    if (rank) {
        const float scale = A.scales ? A.scales[tile.adapter] : 1.f;
        f32x4 v[NV];
        const int64_t cut = (int64_t)A.tokens * width;
#pragma unroll
        for (int i = 0; i < NV; ++i) {                        // sixteen lanes a row, four ranks a lane
            const int j = 64 * i + 4 * i16;
            v[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (j >= rank) continue;
            const float* h = A.h + (int64_t)(tile.first + min(w * 4 + q, tile.count - 1)) * width + s * A.rank + j;
            for (int c = 0; c < A.cuts; c += 4) {
                f32x4 part[4];
#pragma unroll
                for (int o = 0; o < 4; ++o) part[o] = *(const f32x4*)(h + min(c + o, A.cuts - 1) * cut);
#pragma unroll
                for (int o = 0; o < 4; ++o)
                    if (c + o < A.cuts) v[i] += part[o];
            }
        }
        row_to_planes<T>(v, scale, rank, w * 4 + q, planes, A.pitch, factor);
    }
    __syncthreads();
    const uint16_t* hi = planes + i16 * A.pitch + 8 * q;
    const uint16_t* lo = hi + ROWS * A.pitch;
    float* mine = turned[w];
    float f[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) f[r] = rank ? factor[r * 8 + r8] : 0.f;
    for (int c0 = start; c0 < end; c0 += AD_GROUP * AD_WAVES) {
        f32x4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        auto product = [&](int b, int t) {
            if (t == per - 1 && (rank & 31)) {                // behind the adapter's rank, whatever lies there
                const int left = rank - (t * 32 + 8 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) bv[b][j][e] &= left >= 2 * e + 2 ? 0xffffffffu : left == 2 * e + 1 ? 0xffffu : 0u;
            }
            const u32x4 h = *(const u32x4*)(hi + t * 32), l = *(const u32x4*)(lo + t * 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = T::mfma16(bitcast<typename T::vec8>(bv[b][j]), bitcast<typename T::vec8>(h), acc[j]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = T::mfma16(bitcast<typename T::vec8>(bv[b][j]), bitcast<typename T::vec8>(l), acc[j]);
        };
        for (int t = 0; t < per; t += 2) {
            product(0, t);
            if (t + 2 < per) load_b(c0, 0, t + 2);
            if (t + 1 < per) {
                product(1, t + 1);
                if (t + 3 < per) load_b(c0, 1, t + 3);
            }
        }
        const int next = c0 + AD_GROUP * AD_WAVES;
        if (next < end) load_first_b(next);
        const bool vec = whole(c0);
        const int col = c0 + 8 * p8;
        sort_fence();
#pragma unroll
        for (int j = 0; j < 4; ++j) *(f32x4*)(mine + i16 * AD_PITCH + 16 * j + 4 * q) = acc[j];
        sort_fence();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float* at = mine + (8 * h + r8) * AD_PITCH + 8 * p8;
            const f32x4 d0 = *(const f32x4*)at, d1 = *(const f32x4*)(at + 4);
            if (8 * h + r8 >= tile.count) continue;
            uint16_t* out = A.out + (int64_t)rows[h] * A.out_stride + first + col;
            if (vec) {
                float x[8];
                unpack8<T>(raw[h], x);
                u32x4 o = raw[h];
                if (rank)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f32x4& d = e < 2 ? d0 : d1;
                        o[e] = pack2<T>(fmaf(d[2 * (e & 1)], f[h], x[2 * e]), fmaf(d[2 * (e & 1) + 1], f[h], x[2 * e + 1]));
                    }
                *(u32x4*)out = o;
            } else {
                const uint16_t* base = A.base + (int64_t)rows[h] * A.base_stride + first + col;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < cols) out[e] = rank ? T::from_float(fmaf(e < 4 ? d0[e & 3] : d1[e & 3], f[h], T::to_float(base[e]))) : base[e];
            }
        }
        if (next < end) load_base(next);
    }
}

// Both products of a single row in one launch: a workgroup computes its slice's h for itself, in vector instructions, and then a column a
// thread.  A wave computes RB ranks at a time, sixteen waves all of them, with eight steps' loads of 1 KB on their way, B's first
// ranks and base in front of them; h stays in float32.  A's matrix is read by every workgroup, at about 90 KB a microsecond, so it is taken up to 2^17
// elements.  (us with the gap behind it, of the two launches in brackets: K 4096, 4096 columns, ranks 8, 16 and 32: 4.5, 5.3, 7.3 (7.8, 7.7,
// 8.1); 2 x 14336 columns 4.7, 5.6, 9.1 (8.2, 8.2, 8.2); K 14336, rank 16: 11.3 (8.6).  A call of one launch takes the host 3 us less.)
constexpr int64_t AF_MOST = 1 << 17;
constexpr int AF_WAVES = 16, AF_COLS = AF_WAVES * 64, AF_LOADS = 8;
template <typename T, int RB>
__global__ __launch_bounds__(AF_WAVES * 64) void adapter_row_kernel(const AdapterArgs A) {
    constexpr int STEPS = AF_LOADS / RB;
    __shared__ __align__(16) float h[AD_MAX_RANK];
    const AdapterTile tile = A.tiles[0];
    const int rank = tile.adapter < 0 ? 0 : adapter_rank(A, tile.adapter);
    if (rank == 0 && A.out == A.base) return;
    int block = blockIdx.x;
    const int s = slice_of(A, block, AF_COLS);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cols = A.s.width[s], col = block * AF_COLS + threadIdx.x, at = A.s.first[s] + min(col, cols - 1);
    const uint16_t base = A.base[at];
    u32x4 bv[2];
    const uint16_t* b = A.b + ((int64_t)max(tile.adapter, 0) * A.s.total + at) * A.rank;
    if (rank) {
        bv[0] = *(const u32x4*)b;
        bv[1] = *(const u32x4*)(b + min(8, A.rank - 8));
        const uint16_t* a0 = A.a + ((int64_t)tile.adapter * A.s.n + s) * A.rank * A.k;
        const float scale = A.scales ? A.scales[tile.adapter] : 1.f;
        for (int j0 = w * RB; j0 < rank; j0 += AF_WAVES * RB) {
            float acc[RB];
#pragma unroll
            for (int j = 0; j < RB; ++j) acc[j] = 0.f;
            for (int k1 = 0; k1 < A.k; k1 += STEPS * 512) {
                const int k0 = k1 + 8 * lane;
                u32x4 av[STEPS][RB], xv[STEPS];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int k = min(k0 + 512 * i, A.k - 8);
#pragma unroll
                    for (int j = 0; j < RB; ++j) av[i][j] = *(const u32x4*)(a0 + (int64_t)min(j0 + j, rank - 1) * A.k + k);
                    xv[i] = *(const u32x4*)(A.x + k);
                }
                __builtin_amdgcn_sched_barrier(0);            // all of them before the first use
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    if (k0 + 512 * i >= A.k) break;           // behind the row's end
                    float x[8];
                    unpack8<T>(xv[i], x);
#pragma unroll
                    for (int j = 0; j < RB; ++j) {
                        float f[8];
                        unpack8<T>(av[i][j], f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[j] = fmaf(f[e], x[e], acc[j]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < RB; ++j) {
                const float sum = wave_sum(acc[j]) * scale;
                if (lane == 0 && j0 + j < rank) h[j0 + j] = sum;
            }
        }
    }
    __syncthreads();
    if (col >= cols) return;
    float sum = 0.f;
    for (int j0 = 0; j0 < rank; j0 += 16) {
        if (j0) {
            bv[0] = *(const u32x4*)(b + min(j0, A.rank - 8));
            bv[1] = *(const u32x4*)(b + min(j0 + 8, A.rank - 8));
        }
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            float f[8];
            unpack8<T>(bv[o], f);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (j0 + 8 * o + e < rank) sum = fmaf(f[e], h[j0 + 8 * o + e], sum);      // (behind the adapter's rank: whatever lies there)
        }
    }
    A.out[at] = rank ? T::from_float(T::to_float(base) + sum) : base;
}

// How the products are cut.  Two tiles of ranks a workgroup (three of 64 rows: x is read by fewer).  Cuts of K: 1024 workgroups where there
// is that much, four units a wave and cut at least (eight where there are 128 tiles), 8 cuts at most: a cut is another float32 copy
// of h.  Groups of columns a wave: up to four behind one sum of h, while 512 workgroups are left.  (us, of both kernels.  8191 rows, K 4096,
// 4096 + 2 x 1024 columns, rank 32: 72 in one cut, 68 in two, 78 in four; four tiles a workgroup 75; one group a wave 88.  64 rows of 24
// adapters of up to 64 ranks, K 14336: 21 in two cuts, 16.5 in four, 15.3 in eight; K 4096, 2 x 14336 columns: one group a wave
// 27, two 25.)
struct AdapterPlan {
    int cuts, cut_units, blocks, ct, groups_each;
};
AdapterPlan adapter_plan(int tokens, int adapters, int tile, int k, int slices, int rank, const int32_t* widths) {
    AdapterPlan p;
    const int units = slices * ((rank + 15) / 16), most = tile == 16 ? 2 : 3;
    p.blocks = (units + most - 1) / most;
    p.ct = (units + p.blocks - 1) / p.blocks;
    const int k_units = (k + 63) / 64;
    const int64_t tiles = std::min<int64_t>(adapter_max_tiles(tokens, adapters, tile), tokens);
    const int64_t want = (1024 + tiles * p.blocks - 1) / (tiles * p.blocks);
    const int cuts = (int)std::min<int64_t>(std::min<int64_t>(want, 8), std::max(1, k_units / ((tiles < 128 ? 4 : 8) * AD_WAVES)));
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
    // 16 waves where their counts fit 64 KB of LDS
#define AD_ROWS(WAVES)                                                                                                              \
    hipLaunchKernelGGL(adapter_rows_kernel<WAVES>, dim3(1), dim3(WAVES * 64), sizeof(int) * (size_t)((WAVES + 2) * (adapters + 1) + 2), \
                       (hipStream_t)stream, plan, (AdapterTile*)(plan + adapter_order_ints(tokens)), adapter_ids, tokens, adapters, tile, \
                       adapter_max_tiles(tokens, adapters, tile), 32 - __builtin_clz((unsigned)adapters | 1u))
    if (adapters <= 512) AD_ROWS(16);
    else AD_ROWS(8);
#undef AD_ROWS
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
    const int block_cols = AD_GROUP * AD_WAVES * p.groups_each;
    int64_t col_blocks = 0;
    for (int i = 0; i < slices; ++i) col_blocks += (A.s.width[i] + block_cols - 1) / block_cols;
    A.max_tiles = tiles, A.blocks = p.blocks, A.pitch = (rank + 31) / 32 * 32 + 8;
    if (tokens == 1 && (int64_t)rank * k <= AF_MOST) {
        int blocks = 0;
        for (int i = 0; i < slices; ++i) blocks += (A.s.width[i] + AF_COLS - 1) / AF_COLS;
#define AD_ROW(T, RB) hipLaunchKernelGGL((adapter_row_kernel<T, RB>), dim3(blocks), dim3(AF_WAVES * 64), 0, st, A)
        if (dtype == MF_BF16) {
            if (rank <= AF_WAVES) AD_ROW(BF16, 1);
            else AD_ROW(BF16, 2);
        } else {
            if (rank <= AF_WAVES) AD_ROW(FP16, 1);
            else AD_ROW(FP16, 2);
        }
#undef AD_ROW
        return MF_LAUNCH_CHECK();
    }
    const int64_t shrinks = ((int64_t)tiles * p.cuts + 7) / 8 * 8 * p.blocks;
    A.subs = tile / 16, A.col_blocks = (int)col_blocks;
    MF_REQUIRE(shrinks < (1 << 24) && tiles * A.subs * col_blocks < (1 << 24), "adapter_linear: %d rows of %lld columns", tokens,
               (long long)columns);
    const dim3 g1((unsigned)shrinks);
#define AD_SHRINK(T, RT, CT) hipLaunchKernelGGL((adapter_shrink_kernel<T, RT, CT>), g1, dim3(AD_WAVES * 64), 0, st, A)
#define AD_SHRINK_T(T)                                \
    do {                                              \
        if (tile == 16) {                             \
            if (p.ct == 1) AD_SHRINK(T, 1, 1);        \
            else AD_SHRINK(T, 1, 2);                  \
        } else {                                      \
            if (p.ct == 1) AD_SHRINK(T, 4, 1);        \
            else if (p.ct == 2) AD_SHRINK(T, 4, 2);   \
            else AD_SHRINK(T, 4, 3);                  \
        }                                             \
    } while (0)
    if (dtype == MF_BF16) AD_SHRINK_T(BF16);
    else AD_SHRINK_T(FP16);
#undef AD_SHRINK_T
#undef AD_SHRINK
    const int rc = MF_LAUNCH_CHECK();
    if (rc) return rc;
    const dim3 g2((unsigned)(tiles * A.subs * col_blocks));
    const size_t lds = (size_t)2 * 16 * A.pitch * 2;
    if (dtype == MF_BF16) hipLaunchKernelGGL(adapter_expand_kernel<BF16>, g2, dim3(AD_WAVES * 64), lds, st, A);
    else hipLaunchKernelGGL(adapter_expand_kernel<FP16>, g2, dim3(AD_WAVES * 64), lds, st, A);
    return MF_LAUNCH_CHECK();
}
