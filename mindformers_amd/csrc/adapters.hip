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

// Counting sort in one workgroup, in the rows' order within an adapter: every wave counts, then places, a piece of the rows of its own.
// Bound by latency: ids, two scans and the placing one behind the other.
__global__ __launch_bounds__(AD_SORT_THREADS) void adapter_rows_kernel(int* __restrict__ order, AdapterTile* __restrict__ tiles,
                                                                       const int* __restrict__ ids, int tokens, int adapters, int tile,
                                                                       int max_tiles) {
    extern __shared__ int lds[];
    const int n = adapters + 1;                               // the last: rows without an adapter
    int* hist = lds;                                          // [waves][n]
    int* start = hist + AD_SORT_WAVES * n;                    // [n + 1]
    int* tstart = start + n + 1;
    __shared__ int w_rows[AD_SORT_WAVES], w_tiles[AD_SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    for (int i = tid; i < AD_SORT_WAVES * n; i += AD_SORT_THREADS) hist[i] = 0;
    __syncthreads();
    const int piece = ((tokens + AD_SORT_WAVES - 1) / AD_SORT_WAVES + 63) / 64 * 64;
    const int r0 = min(w * piece, tokens), r1 = min(r0 + piece, tokens);
    auto key = [&](int r) {
        const int a = ids[r];
        return a >= 0 && a < adapters ? a : adapters;
    };
    for (int r = r0 + lane; r < r1; r += 64) atomicAdd(&hist[w * n + key(r)], 1);
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
    for (int rb = r0; rb < r1; rb += 64) {                    // rows of one adapter among 64 are found by their ballots
        const int r = rb + lane, a = r < r1 ? key(r) : -1;
        uint64_t todo = __ballot(a >= 0);
        while (todo) {
            const int b = __builtin_amdgcn_readlane(a, (int)__builtin_ctzll(todo));
            const uint64_t m = __ballot(a == b);
            sort_fence();
            const int at = hist[w * n + b];
            if (a == b) order[start[b] + at + __popcll(m & ((1ull << lane) - 1ull))] = r;
            sort_fence();
            if (lane == 0) hist[w * n + b] = at + __popcll(m);
            todo &= ~m;
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
    int groups_each;                                          // column groups of a wave
    int vec_io;                                               // base and out rows on 16-byte borders
    AdapterSlices s;
};

__device__ __forceinline__ int adapter_rank(const AdapterArgs& A, int a) { return A.ranks ? min(max(A.ranks[a], 0), A.rank) : A.rank; }

// h of RT x 16 rows and up to CT tiles of 16 ranks (of whatever slices), over one cut of K.  Lane l of a fragment holds rank or row
// l & 15 and 8 values from 8 (l >> 4) on, as both operands lie in memory.  The waves take units of 64 columns in turn and meet in LDS.
template <typename T, int RT, int CT>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_shrink_kernel(const AdapterArgs A) {
    __shared__ f32x4 red[AD_WAVES][RT * CT][64];
    const AdapterTile tile = A.tiles[blockIdx.x];
    if (tile.count <= 0 || tile.adapter < 0) return;
    const int rank = adapter_rank(A, tile.adapter);
    const int per = (rank + 15) >> 4, units = per * A.s.n, c0 = blockIdx.z * CT;
    if (c0 >= units) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
    const uint16_t* xr[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) xr[r] = A.x + (int64_t)A.order[tile.first + min(r * 16 + i16, tile.count - 1)] * A.x_stride + 8 * q;
    const uint16_t* ar[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {                            // tiles past the last one, ranks past the bank's: others once more
        const int u = min(c0 + c, units - 1), s = u / per, row = min((u - s * per) * 16 + i16, A.rank - 1);
        ar[c] = A.a + ((int64_t)(tile.adapter * A.s.n + s) * A.rank + row) * A.k + 8 * q;
    }
    f32x4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int u_end = min((int)(blockIdx.y + 1) * A.cut_units, (A.k + 63) >> 6);
    const int last = A.k - 8 - 8 * q;                         // where this lane's last whole piece starts
    for (int u = blockIdx.y * A.cut_units + w; u < u_end; u += AD_WAVES) {
        u32x4 xv[2][RT], av[2][CT];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = u * 64 + half * 32, at = min(k, last);      // last may be negative: then this lane's piece starts in front
#pragma unroll
            for (int r = 0; r < RT; ++r) xv[half][r] = *(const u32x4*)(xr[r] + at);
#pragma unroll
            for (int c = 0; c < CT; ++c) av[half][c] = *(const u32x4*)(ar[c] + at);
            if (k > last)                                     // behind the row's end: nothing
#pragma unroll
                for (int r = 0; r < RT; ++r) xv[half][r] = (u32x4){0, 0, 0, 0};
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int c = 0; c < CT; ++c)
                    acc[r][c] = T::mfma16(bitcast<typename T::vec8>(av[half][c]), bitcast<typename T::vec8>(xv[half][r]), acc[r][c]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) red[w][r * CT + c][lane] = acc[r][c];
    __syncthreads();
    const int width = A.s.n * A.rank;
    for (int t = w; t < RT * CT; t += AD_WAVES) {
        const int r = t / CT, c = t - r * CT, u = c0 + c;
        if (u >= units) continue;
        const int s = u / per, j = (u - s * per) * 16 + 4 * q, row = r * 16 + i16;       // four ranks of a row a lane
        f32x4 v = red[0][t][lane];
#pragma unroll
        for (int o = 1; o < AD_WAVES; ++o) v += red[o][t][lane];
        if (row < tile.count && j < A.rank) *(f32x4*)(A.h + ((int64_t)blockIdx.y * A.tokens + tile.first + row) * width + s * A.rank + j) = v;
    }
}

// out = base + (B h): a workgroup computes 4 x groups_each groups of 64 columns of one slice for RT x 16 rows.  The product is taken
// with the columns as the matrix instruction's rows, in an order that leaves a lane 16 columns side by side of one row: base and
// out move in 32 bytes a lane, 128 a row.
template <typename T, int RT>
__global__ __launch_bounds__(AD_WAVES * 64) void adapter_expand_kernel(const AdapterArgs A) {
    constexpr int ROWS = RT * 16, PITCH = AD_MAX_RANK + 8;
    __shared__ __align__(16) uint16_t planes[2][ROWS][PITCH]; // h as hi and lo
    __shared__ float factor[ROWS];                            // what a row of the planes is to be multiplied with
    __shared__ int rows[ROWS];
    const AdapterTile tile = A.tiles[blockIdx.x];
    if (tile.count <= 0) return;
    const int rank = tile.adapter < 0 ? 0 : adapter_rank(A, tile.adapter);
    if (rank == 0 && A.out == A.base) return;
    int block = blockIdx.y, s = 0;
    const int block_cols = AD_GROUP * AD_WAVES * A.groups_each;
    for (;; ++s) {                                            // the slice of this block
        const int n = (A.s.width[s] + block_cols - 1) / block_cols;
        if (block < n) break;
        block -= n;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
    if (threadIdx.x < ROWS) rows[threadIdx.x] = A.order[tile.first + min((int)threadIdx.x, tile.count - 1)];
    const int per = (rank + 15) >> 4, width = A.s.n * A.rank;
    const float scale = rank && A.scales ? A.scales[tile.adapter] : 1.f;
    for (int row = w * 4 + q; rank && row < ROWS; row += AD_WAVES * 4) {      // sixteen lanes a row, four ranks a lane at a time
        f32x4 v[AD_MAX_RANK / 64];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < AD_MAX_RANK / 64; ++i) {
            const int j = 64 * i + 4 * i16;
            v[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (j < rank && row < tile.count) {
                const float* h = A.h + (int64_t)(tile.first + row) * width + s * A.rank + j;
                for (int c = 0; c < A.cuts; ++c) v[i] += *(const f32x4*)(h + (int64_t)c * A.tokens * width);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[i][e] = j + e < rank ? v[i][e] * scale : 0.f;
                    most = fmaxf(most, fabsf(v[i][e]));
                }
            }
        }
        float up = 1.f, down = 1.f;
        if constexpr (std::is_same_v<T, FP16>) {              // h may pass the range of fp16: rows go in with a power of two
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
        for (int i = 0; i < AD_MAX_RANK / 64; ++i) {
            const int j = 64 * i + 4 * i16;
            if (j >= per * 16) continue;
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float a = v[i][2 * e] * up, b = v[i][2 * e + 1] * up;
                hi[e] = pack2<T>(a, b);
                const float ra = a - T::to_float((uint16_t)hi[e]), rb = b - T::to_float((uint16_t)(hi[e] >> 16));
                lo[e] = pack2<T>(fabsf(ra) < INFINITY ? ra : 0.f, fabsf(rb) < INFINITY ? rb : 0.f);      // infinite: hi says it
            }
            *(u32x2*)&planes[0][row][j] = (u32x2){hi[0], hi[1]};
            *(u32x2*)&planes[1][row][j] = (u32x2){lo[0], lo[1]};
        }
    }
    __syncthreads();
    const int first = A.s.first[s], cols = A.s.width[s];
    for (int g = 0; g < A.groups_each; ++g) {
        const int c0 = ((block * A.groups_each + g) * AD_WAVES + w) * AD_GROUP;
        if (c0 >= cols) break;
        const bool whole = A.vec_io && c0 + AD_GROUP <= cols && (first & 7) == 0;
        const int mine = c0 + 16 * q;                         // this lane's sixteen columns
        u32x4 raw[RT][2];
        if (whole) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    raw[r][p] = *(const u32x4*)(A.base + (int64_t)rows[r * 16 + i16] * A.base_stride + first + mine + 8 * p);
        }
        f32x4 acc[RT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (rank) {
            const uint16_t* br[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = min(c0 + (i16 >> 2) * 16 + 4 * j + (i16 & 3), cols - 1);
                br[j] = A.b + ((int64_t)tile.adapter * A.s.total + first + n) * A.rank;
            }
            for (int t = 0; t < per; ++t) {
                const int k = t * 16 + 8 * (q & 1), left = rank - k;
                u32x4 bv[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) bv[j] = *(const u32x4*)(br[j] + min(k, A.rank - 8));
                if (left < 8) {                               // behind the adapter's rank, whatever lies there
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) bv[j][e] &= left >= 2 * e + 2 ? 0xffffffffu : left == 2 * e + 1 ? 0xffffu : 0u;
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const u32x4 hv = *(const u32x4*)&planes[lane >> 5][r * 16 + i16][k];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[r][j] = T::mfma16(bitcast<typename T::vec8>(bv[j]), bitcast<typename T::vec8>(hv), acc[r][j]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const int row = r * 16 + i16;
            if (row >= tile.count) continue;
            const float f = rank ? factor[row] : 0.f;
            uint16_t* out = A.out + (int64_t)rows[row] * A.out_stride + first + mine;
            if (whole) {
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[8];
                    unpack8<T>(raw[r][p], v);
                    u32x4 o = raw[r][p];
                    if (rank)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[e] = pack2<T>(fmaf(acc[r][2 * p + (e >> 1)][2 * (e & 1)], f, v[2 * e]),
                                            fmaf(acc[r][2 * p + (e >> 1)][2 * (e & 1) + 1], f, v[2 * e + 1]));
                    *(u32x4*)(out + 8 * p) = o;
                }
            } else {
                const uint16_t* base = A.base + (int64_t)rows[row] * A.base_stride + first + mine;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (mine + e < cols) out[e] = rank ? T::from_float(fmaf(acc[r][e >> 2][e & 3], f, T::to_float(base[e]))) : base[e];
            }
        }
    }
}

struct AdapterPlan {
    int cuts, cut_units, blocks, ct, groups_each;
};
AdapterPlan adapter_plan(int tokens, int adapters, int tile, int k, int slices, int rank, int64_t columns) {
    AdapterPlan p;
    const int units = slices * ((rank + 15) / 16);
    p.ct = units >= 4 ? 4 : units >= 2 ? 2 : 1;
    p.blocks = (units + p.ct - 1) / p.ct;
    const int k_units = (k + 63) / 64;
    const int64_t tiles = std::max<int64_t>(1, std::min<int64_t>(adapter_max_tiles(tokens, adapters, tile), tokens));
    const int64_t want = std::max<int64_t>(1, 512 / (tiles * p.blocks));
    int cuts = (int)std::min<int64_t>(want, std::max(1, k_units / 4));       // a unit a wave at least
    cuts = std::min(cuts, 8);
    p.cut_units = (k_units + cuts - 1) / cuts;
    p.cuts = (k_units + p.cut_units - 1) / p.cut_units;
    p.groups_each = columns * tiles >= (int64_t)4096 * AD_GROUP * AD_WAVES ? 2 : 1;
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
                       adapter_max_tiles(tokens, adapters, tile));
    return MF_LAUNCH_CHECK();
}

extern "C" size_t mf_adapter_workspace_bytes(int tokens, int adapters, int tile, int k, int slices, int rank) {
    if (tokens <= 0 || adapters <= 0 || (tile != 16 && tile != 64) || k <= 0 || slices <= 0 || slices > AD_MAX_SLICES || rank <= 0 ||
        rank > AD_MAX_RANK)
        return 0;
    return sizeof(float) * (size_t)adapter_plan(tokens, adapters, tile, k, slices, rank, 0).cuts * tokens * slices * rank;
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
    const AdapterPlan p = adapter_plan(tokens, adapters, tile, k, slices, rank, columns);
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
    const dim3 g1((unsigned)tiles, (unsigned)p.cuts, (unsigned)p.blocks);
#define AD_SHRINK(T, RT)                                                                                                   \
    do {                                                                                                                   \
        if (p.ct == 4) hipLaunchKernelGGL((adapter_shrink_kernel<T, RT, 4>), g1, dim3(AD_WAVES * 64), 0, st, A);           \
        else if (p.ct == 2) hipLaunchKernelGGL((adapter_shrink_kernel<T, RT, 2>), g1, dim3(AD_WAVES * 64), 0, st, A);      \
        else hipLaunchKernelGGL((adapter_shrink_kernel<T, RT, 1>), g1, dim3(AD_WAVES * 64), 0, st, A);                     \
    } while (0)
    if (dtype == MF_BF16) {
        if (tile == 16) AD_SHRINK(BF16, 1);
        else AD_SHRINK(BF16, 4);
    } else {
        if (tile == 16) AD_SHRINK(FP16, 1);
        else AD_SHRINK(FP16, 4);
    }
#undef AD_SHRINK
    const int rc = MF_LAUNCH_CHECK();
    if (rc) return rc;
    int64_t col_blocks = 0;
    const int block_cols = AD_GROUP * AD_WAVES * p.groups_each;
    for (int i = 0; i < slices; ++i) col_blocks += (A.s.width[i] + block_cols - 1) / block_cols;
    MF_REQUIRE(col_blocks <= 65535, "adapter_linear: %lld columns", (long long)columns);
    const dim3 g2((unsigned)tiles, (unsigned)col_blocks);
    if (dtype == MF_BF16) {
        if (tile == 16) hipLaunchKernelGGL((adapter_expand_kernel<BF16, 1>), g2, dim3(AD_WAVES * 64), 0, st, A);
        else hipLaunchKernelGGL((adapter_expand_kernel<BF16, 4>), g2, dim3(AD_WAVES * 64), 0, st, A);
    } else {
        if (tile == 16) hipLaunchKernelGGL((adapter_expand_kernel<FP16, 1>), g2, dim3(AD_WAVES * 64), 0, st, A);
        else hipLaunchKernelGGL((adapter_expand_kernel<FP16, 4>), g2, dim3(AD_WAVES * 64), 0, st, A);
    }
    return MF_LAUNCH_CHECK();
}
