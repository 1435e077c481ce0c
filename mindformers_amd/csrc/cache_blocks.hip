// Blocks of a paged cache that several sequences share: forking block tables (and giving blocks back), closing up a
// pool, and the copies that either asks for.  Block tables are int32 [rows, width], -1 = no block; a block is in use if
// an entry of a table names it, so that the tables are the only state and a step is a function of them.
//
// What bounds the two planning operators is launch latency and one workgroup's walk over the tables: their answer hangs
// on a ranking of all free blocks, which one workgroup forms from a bitmap in LDS (one bit a block, 128 KB for a million).  Under the
// profiler 16 rows of 32 blocks in 1024 take 8 us in one launch, 512 rows of 256 in 131072 5.9 + 10.6 in two, closing up 64 rows of
// 32 in 1024 9.0 + 4.5.
#include <algorithm>

#include "common.h"

namespace {

constexpr int CB_THREADS = 1024;
constexpr int CB_WAVES = CB_THREADS / 64;
constexpr int CB_MAX_BLOCKS = 1 << 20;                        // bits of the bitmap: 128 KB of LDS
constexpr int FORK_FILL = 16;                                 // more new tokens than this a row are placed by a kernel of their own
constexpr int CB_MAX_ROWS = 4096;                             // rows of a fork: 16 KB of LDS beside it
constexpr int FORK_MARKERS = 16;                              // most workgroups that mark the blocks of large tables

struct ForkArgs {
    int32_t *tables_out, *lens_out, *slots, *copies, *missing;
    const int32_t *tables, *lens, *parents;
    const uint8_t* held;
    int32_t *fresh, *ranks;                                   // workspace: the blocks that are handed out; with FORK_FILL, [1 + rows]:
                                                              // how many, and the place of each row's first block behind its open one
    uint32_t* marks;                                          // workspace: the markers' bitmaps, fork_words() each
    int markers;                                              // workgroups of fork_mark_kernel, 0: none
    int rows, width, num_blocks, block_size, new_tokens, window, sinks;
};

// Row s of a fork: its parent's row, its length and the number of blocks in use there.
struct ForkRow {
    int parent, len, used;                                    // parent -1: the row is empty
};
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int s) {
    ForkRow r;
    r.parent = a.parents ? a.parents[s] : s;
    if (r.parent < 0 || r.parent >= a.rows) return {-1, 0, 0};
    r.len = min(max(a.lens[r.parent], 0), a.width * a.block_size);
    r.used = (r.len + a.block_size - 1) / a.block_size;
    return r;
}
// Whether entry j of a row of `len` tokens stays: not where all its tokens lie in front of the window of the next query
// (position len, which sees tokens > len - window) and none of them is a sink.
__device__ __forceinline__ bool fork_keeps(const ForkArgs& a, int j, int len) {
    if (a.window == 0) return true;
    return (int64_t)(j + 1) * a.block_size > (int64_t)len - a.window + 1 || (int64_t)j * a.block_size < a.sinks;
}

// One row of the new tables without the blocks that are still to be found, by one wave.  The open block (the last one, where
// it is not full) is every child's here.
__device__ __forceinline__ void fork_gather_row(const ForkArgs& a, int s) {
    const ForkRow r = fork_row(a, s);
    const int32_t* from = a.tables + (int64_t)max(r.parent, 0) * a.width;
    int32_t* to = a.tables_out + (int64_t)s * a.width;
    for (int j = threadIdx.x & 63; j < a.width; j += 64) {
        int page = -1;
        if (j < r.used && fork_keeps(a, j, r.len)) {
            page = from[j];
            if (page >= a.num_blocks) page = -1;
        }
        to[j] = max(page, -1);
    }
}

__global__ __launch_bounds__(256) void fork_gather_kernel(ForkArgs a) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s < a.rows) fork_gather_row(a, s);
}

// words of a bitmap with a bit for every block, as 16-byte pieces
__host__ __device__ __forceinline__ int fork_words(int num_blocks) { return (num_blocks + 127) / 128 * 4; }

// The rows gathered and their blocks marked, each workgroup in a bitmap of its own that the assigning one joins.  512 rows of 256
// entries: 5.9 us and 10.6 for the assigning workgroup; 3.4 and 16.0 where that one marks all entries (an LDS operation each).
__global__ __launch_bounds__(CB_THREADS) void fork_mark_kernel(ForkArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t bits[];
    const int words = fork_words(a.num_blocks), lane = threadIdx.x & 63;
    for (int w = threadIdx.x; w < words; w += CB_THREADS) bits[w] = 0;
    __syncthreads();
    for (int s = blockIdx.x * CB_WAVES + (threadIdx.x >> 6); s < a.rows; s += gridDim.x * CB_WAVES) {
        const ForkRow r = fork_row(a, s);
        const int32_t* from = a.tables + (int64_t)max(r.parent, 0) * a.width;
        int32_t* to = a.tables_out + (int64_t)s * a.width;
        for (int j0 = 0; j0 < a.width; j0 += 256) {
            int page[4];                                      // four reads on their way at a time
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + 64 * k + lane;
                page[k] = j < r.used && j < a.width && fork_keeps(a, j, r.len) ? from[j] : -1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + 64 * k + lane;
                if (j >= a.width) continue;
                const bool on = page[k] >= 0 && page[k] < a.num_blocks;
                to[j] = on ? page[k] : -1;
                if (on) atomicOr(&bits[page[k] >> 5], 1u << (page[k] & 31));
            }
        }
    }
    __syncthreads();
    u32x4* mine = (u32x4*)(a.marks + (int64_t)blockIdx.x * words);
    for (int i = threadIdx.x; i < words / 4; i += CB_THREADS) mine[i] = ((const u32x4*)bits)[i];
}

// Exclusive prefix sum over the workgroup's threads; `total` is the sum.  red: CB_WAVES ints of LDS.
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(incl, o, 64);
        if (lane >= o) incl += t;
    }
    __syncthreads();                                          // red may still be read from the scan before
    if (lane == 63) red[w] = incl;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < CB_WAVES; ++i) {
        const int t = red[i];
        before += i < w ? t : 0;
        sum += t;
    }
    total = sum;
    return before + incl - v;
}

__device__ __forceinline__ void mark(uint32_t* bits, int page, int num_blocks) {
    if (page < 0 || page >= num_blocks) return;
    atomicOr(&bits[page >> 5], 1u << (page & 31));            // nothing waits for it; looking first took half as long again
}
// the bits of all entries of a table
__device__ __forceinline__ void mark_table(uint32_t* bits, const int32_t* t, int64_t n, int num_blocks) {
    const int64_t n4 = ((uintptr_t)t & 15) == 0 ? n / 4 : 0;
    for (int64_t i0 = threadIdx.x; i0 < n4; i0 += 8 * CB_THREADS) {
        i32x4 v[8];                                           // eight reads on their way at a time: one workgroup waits for each
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = i0 + k * CB_THREADS;
            v[k] = i < n4 ? ((const i32x4*)t)[i] : (i32x4){-1, -1, -1, -1};
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) mark(bits, v[k][e], num_blocks);
    }
    for (int64_t i = 4 * n4 + threadIdx.x; i < n; i += CB_THREADS) mark(bits, t[i], num_blocks);
}
// word w of the blocks that belong to others (a byte a block, null: none)
__device__ __forceinline__ uint32_t held_word(const uint8_t* __restrict__ held, int w, int num_blocks) {
    if (!held) return 0;
    uint32_t m = 0;
    for (int i = 0; i < 32 && 32 * w + i < num_blocks; ++i) m |= (uint32_t)(held[32 * w + i] != 0) << i;
    return m;
}
__device__ __forceinline__ uint32_t in_range(int w, int num_blocks) {
    const int left = num_blocks - 32 * w;
    return left >= 32 ? ~0u : (left <= 0 ? 0u : (1u << left) - 1u);
}

// The blocks that a fork's rows ask for: rows ascending, in a row the copy of its open block first, then the blocks of its
// new tokens; request i gets the i-th lowest free block.  GATHER: the rows are gathered here too (small tables: one launch).
struct ForkRequest {
    ForkRow r;
    int open, wanted, over;                                   // block to copy (-1: none), blocks behind it, more for which the table has no place
};
template <bool GATHER>
__global__ __launch_bounds__(CB_THREADS) void fork_assign_kernel(ForkArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t bits[];
    __shared__ int red[CB_WAVES];
    const int tid = threadIdx.x;
    const int words = fork_words(a.num_blocks);
    int* eldest = (int*)(bits + words);                       // lowest child of every row
    if (!GATHER && a.markers) {
        for (int i = tid; i < words / 4; i += CB_THREADS) {
            u32x4 m = {0u, 0u, 0u, 0u}, v[FORK_MARKERS];
#pragma unroll
            for (int g = 0; g < FORK_MARKERS; ++g) v[g] = ((const u32x4*)(a.marks + (int64_t)min(g, a.markers - 1) * words))[i];
#pragma unroll
            for (int g = 0; g < FORK_MARKERS; ++g) m |= v[g];
            if (a.held)
#pragma unroll
                for (int e = 0; e < 4; ++e) m[e] |= held_word(a.held, 4 * i + e, a.num_blocks);
            ((u32x4*)bits)[i] = m;
        }
    } else {
        for (int w = tid; w < words; w += CB_THREADS) bits[w] = held_word(a.held, w, a.num_blocks);
    }
    for (int s = tid; s < a.rows; s += CB_THREADS) eldest[s] = a.rows;
    if constexpr (GATHER) {
        for (int s = tid >> 6; s < a.rows; s += CB_WAVES) fork_gather_row(a, s);
        __threadfence_block();
    }
    __syncthreads();
    for (int s = tid; s < a.rows; s += CB_THREADS) {
        const int p = a.parents ? a.parents[s] : s;
        if (p >= 0 && p < a.rows) atomicMin(&eldest[p], s);
    }
    if (GATHER || !a.markers) mark_table(bits, a.tables_out, (int64_t)a.rows * a.width, a.num_blocks);
    __syncthreads();

    auto request = [&](int s) -> ForkRequest {
        ForkRequest q = {{-1, 0, 0}, -1, 0, 0};
        if (s >= a.rows) return q;
        q.r = fork_row(a, s);
        if (q.r.parent < 0) return q;
        const int all = (int)(((int64_t)q.r.len + a.new_tokens + a.block_size - 1) / a.block_size) - q.r.used;
        q.wanted = min(all, a.width - q.r.used);
        q.over = all - q.wanted;
        if (q.r.len % a.block_size != 0 && eldest[q.r.parent] != s) q.open = a.tables_out[(int64_t)s * a.width + q.r.used - 1];
        return q;
    };
    // how many blocks are asked for
    const ForkRequest first = request(tid);
    int asked = (first.open >= 0) + first.wanted;
    for (int s = tid + CB_THREADS; s < a.rows; s += CB_THREADS) {
        const ForkRequest q = request(s);
        asked += (q.open >= 0) + q.wanted;
    }
    int total;
    (void)block_scan(asked, red, total);

    // the lowest free blocks, 32 * CB_THREADS at a time until there are enough
    int found = 0;
    for (int w0 = 0; w0 < words && found < total; w0 += CB_THREADS) {
        const int w = w0 + tid;
        uint32_t free_bits = w < words ? ~bits[w] & in_range(w, a.num_blocks) : 0u;
        int here;
        int rank = found + block_scan((int)__popc(free_bits), red, here);
        while (free_bits && rank < total) {
            a.fresh[rank++] = 32 * w + __ffs(free_bits) - 1;
            free_bits &= free_bits - 1;
        }
        found += here;
    }
    found = min(found, total);
    __threadfence_block();
    __syncthreads();

    // hand them out
    int base = 0, base_copy = 0, given = 0;
    for (int s0 = 0; s0 < a.rows; s0 += CB_THREADS) {
        const int s = s0 + tid;
        const ForkRequest q = s0 == 0 ? first : request(s);
        const ForkRow r = q.r;
        const bool split = q.open >= 0;
        int all, copies;
        const int begin = base + block_scan(split + q.wanted, red, all);
        const bool copied = split && begin < found;
        const int at = base_copy + block_scan(copied, red, copies);
        if (s < a.rows) {
            int32_t* row = a.tables_out + (int64_t)s * a.width;
            int last = -1;                                    // block of the first new token, where the open one takes it
            if (split) {
                last = copied ? a.fresh[begin] : -1;
                row[r.used - 1] = last;
                if (copied) {
                    a.copies[3 * at] = q.open;
                    a.copies[3 * at + 1] = last;
                    a.copies[3 * at + 2] = r.len % a.block_size;
                    ++given;
                }
            }
            const int got = max(min(q.wanted, found - begin - split), 0);
            given += got - q.over;
            const int cap = a.width * a.block_size;
            a.lens_out[s] = r.parent >= 0 ? (int)min((int64_t)r.len + a.new_tokens, (int64_t)cap) : 0;
            if (a.new_tokens > FORK_FILL) a.ranks[1 + s] = begin + split;
            const bool here = a.new_tokens <= FORK_FILL;
            for (int i = 0; here && i < got; ++i) row[r.used + i] = a.fresh[begin + split + i];
            for (int i = 0; here && i < a.new_tokens; ++i) {
                const int64_t pos = (int64_t)r.len + i;
                int slot = -1;
                if (r.parent >= 0 && pos < cap) {
                    const int page = split && pos / a.block_size == r.used - 1 ? last : row[pos / a.block_size];
                    if (page >= 0) slot = page * a.block_size + (int)(pos % a.block_size);
                }
                a.slots[(int64_t)s * a.new_tokens + i] = slot;
            }
        }
        base += all;
        base_copy += copies;
    }
    for (int i = base_copy + tid; i < a.rows; i += CB_THREADS) {
        a.copies[3 * i] = -1;
        a.copies[3 * i + 1] = -1;
        a.copies[3 * i + 2] = 0;
    }
    int got;
    (void)block_scan(given, red, got);
    if (tid == 0) {
        *a.missing = total - got;
        if (a.new_tokens > FORK_FILL) a.ranks[0] = found;
    }
}
// Blocks and slots of many new tokens (a prompt's): a workgroup a row.
__global__ __launch_bounds__(256) void fork_fill_kernel(ForkArgs a) {
    const int s = blockIdx.x, tid = threadIdx.x;
    const ForkRow r = fork_row(a, s);
    int32_t* row = a.tables_out + (int64_t)s * a.width;
    const int64_t last = (int64_t)r.len + a.new_tokens;
    const int rank = a.ranks[1 + s], wanted = (int)((last + a.block_size - 1) / a.block_size) - r.used;
    const int got = r.parent < 0 ? 0 : max(min(min(wanted, a.width - r.used), a.ranks[0] - rank), 0);
    for (int i = tid; i < got; i += 256) row[r.used + i] = a.fresh[rank + i];
    for (int i = tid; i < a.new_tokens; i += 256) {           // a slot's block by its rank: the row may still be on its way
        const int64_t pos = (int64_t)r.len + i;
        const int j = (int)(pos / a.block_size), b = j - r.used;
        int page = -1;
        if (r.parent >= 0 && j < a.width) page = b < 0 ? row[j] : (b < got ? a.fresh[rank + b] : -1);
        a.slots[(int64_t)s * a.new_tokens + i] = page >= 0 ? page * a.block_size + (int)(pos % a.block_size) : -1;
    }
}

// Closing up a pool: the n live blocks that may move go to the n lowest blocks that are not held; one that is there
// already stays, the others go, ascending, to the holes, ascending.
struct CompactArgs {
    int32_t *copies, *live, *to, *holes;                      // to, holes: workspace [num_blocks]
    const int32_t* tables;
    const uint8_t* held;
    int64_t entries;
    int num_blocks, block_size;
};
__global__ __launch_bounds__(CB_THREADS) void compact_plan_kernel(CompactArgs a) {
    extern __shared__ uint32_t bits[];
    __shared__ int red[CB_WAVES];
    const int tid = threadIdx.x;
    const int words = (a.num_blocks + 31) / 32, most = a.num_blocks / 2;
    for (int w = tid; w < words; w += CB_THREADS) bits[w] = 0;
    for (int i = tid; i < a.num_blocks; i += CB_THREADS) a.to[i] = i;
    __syncthreads();
    mark_table(bits, a.tables, a.entries, a.num_blocks);
    __syncthreads();
    int mine = 0;
    for (int w = tid; w < words; w += CB_THREADS) {
        bits[w] &= ~held_word(a.held, w, a.num_blocks);       // blocks of others stay where they are
        mine += __popc(bits[w]);
    }
    int n;
    (void)block_scan(mine, red, n);
    int places = 0, moves = 0, holes = 0;                     // in the words before this round's
    for (int w0 = 0; w0 < words; w0 += CB_THREADS) {
        const int w = w0 + tid;
        const uint32_t may = w < words ? in_range(w, a.num_blocks) & ~held_word(a.held, w, a.num_blocks) : 0u;
        const uint32_t live = w < words ? bits[w] : 0u;
        int here;
        int left = n - (places + block_scan(__popc(may), red, here));
        places += here;
        uint32_t target = 0, rest = may;
        if (left >= (int)__popc(may)) target = may;
        else
            for (; left > 0; --left) {
                target |= rest & (0u - rest);
                rest &= rest - 1;
            }
        uint32_t go = live & ~target, hole = target & ~live;
        int at = moves + block_scan(__popc(go), red, here);
        moves += here;
        for (; go; go &= go - 1, ++at)
            if (at < most) a.copies[3 * at] = 32 * w + __ffs(go) - 1;
        at = holes + block_scan(__popc(hole), red, here);
        holes += here;
        for (; hole; hole &= hole - 1, ++at)
            if (at < most) a.holes[at] = 32 * w + __ffs(hole) - 1;
    }
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < most; i += CB_THREADS) {
        const bool used = i < moves;                          // as many holes as moves
        const int dst = used ? a.holes[i] : -1;
        if (used) a.to[a.copies[3 * i]] = dst;
        else a.copies[3 * i] = -1;
        a.copies[3 * i + 1] = dst;
        a.copies[3 * i + 2] = used ? a.block_size : 0;
    }
    if (tid == 0) *a.live = n;
}
__global__ __launch_bounds__(256) void compact_remap_kernel(int32_t* __restrict__ out, const int32_t* __restrict__ tables,
                                                            const int32_t* __restrict__ to, int64_t entries, int num_blocks) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= entries) return;
    const int page = tables[i];
    out[i] = page >= 0 && page < num_blocks ? to[page] : -1;
}

// Block copies within the cache tensors of all layers in one launch.  The list is on the device and may be longer than
// what is used of it (it ends at the first negative source, whatever lies behind that).  The workgroups take (copy, tensor, piece) in
// turn, stop at a negative source of their own, and store nothing before they have seen that none lies in front of their entry; those
// reads go beside the block's.  Bound: memory.
constexpr int COPY_TENSORS = 128;
constexpr int COPY_PIECE = 16384;                             // bytes of a block that a workgroup copies at a time
constexpr int COPY_THREADS = 256;
// Lists of up to this many entries go to as many as 32768 workgroups, longer ones, of which every workgroup reads the entries in front of its
// own, to 2048.  us on 2048 | 16384 | 32768 | 65536, used of listed copies: 24 of 512 in 64 caches, blocks of 256 KB 152 | 143 | 144 | 161, 192 of
// 512 in 16 caches 312 | 296 | 288 (5.6 TB/s; the library's copy of 200 MiB reaches 5.4) | 297, 3000 of 4096 in 8 2513 | 2472 | 2397 | 2443; on
// 2048 | 16384 | 65536 30000 of 60000 in 2, blocks of 32 KB 809 | 797 | 1222, of 2 KB 116 | 247 | 437, 250000 of 500000 of these 926 | 2245 | 7080.
constexpr int COPY_SHORT = 4096;
struct CopyTensors {
    uint8_t* base[COPY_TENSORS];
    uint32_t row_bytes[COPY_TENSORS];
};
// Whether one of the entries [from, to), from < to, has a negative source.  Up to COPY_ALONE of them are read by every wave for itself,
// without a barrier; more by the workgroup, a wave every fourth 64.  from and to are the workgroup's.
constexpr int COPY_WAVES = COPY_THREADS / 64;
constexpr int COPY_ALONE = 512;
__device__ __forceinline__ bool copies_end(const int32_t* __restrict__ copies, int from, int to) {
    const int lane = threadIdx.x & 63;
    const bool alone = to - from <= COPY_ALONE;
    const int64_t step = alone ? 64 : 64 * COPY_WAVES;
    int any = 0;
    for (int64_t n0 = from + lane + (alone ? 0 : 64 * (threadIdx.x >> 6)); n0 - lane < to; n0 += 2 * step) {
        int src[2];                                           // two reads on their way at a time: most entries have few in front
#pragma unroll
        for (int k = 0; k < 2; ++k) src[k] = copies[3 * min(n0 + k * step, (int64_t)to - 1)];
        any |= src[0] | src[1];
    }
    return alone ? __ballot(any < 0) != 0 : __syncthreads_or(any < 0);
}
__global__ __launch_bounds__(COPY_THREADS) void copy_blocks_kernel(CopyTensors t, const int32_t* __restrict__ copies, int most,
                                                                   int tensors, int pieces, int num_blocks, int block_size) {
    int seen = 0;                                             // no negative source in front of this entry
    const int64_t items = (int64_t)most * tensors * pieces;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int piece = (int)(it % pieces);
        const int64_t ct = it / pieces;
        const int x = (int)(ct % tensors);
        const int c = (int)(ct / tensors);
        const int32_t* e = copies + 3 * (int64_t)c;
        const int src = e[0], dst = e[1];
        if (src < 0) return;                                  // the end, or behind it: this workgroup's later entries are too
        const int rows = min(max(e[2], 0), block_size);
        if (src >= num_blocks || dst < 0 || dst >= num_blocks || src == dst) continue;
        const int64_t block_bytes = (int64_t)block_size * t.row_bytes[x];
        const int64_t from = (int64_t)piece * COPY_PIECE;
        const int64_t to = min((int64_t)rows * t.row_bytes[x], from + COPY_PIECE);
        const uint8_t* s = t.base[x] + src * block_bytes;
        uint8_t* d = t.base[x] + dst * block_bytes;
        const bool wide = (((uintptr_t)s | (uintptr_t)d) & 15) == 0;
        const int64_t end = wide ? max(to & ~(int64_t)15, from) : from;        // 16 bytes at a time as far as there
        constexpr int STEP = COPY_THREADS * 16;
        int64_t i = from + threadIdx.x * 16;
        u32x4 v[4];                                           // past the caches: neither side is read again soon
        const bool ahead = i + 3 * STEP < end;
        if (ahead) {                                          // on their way while the list is looked through
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = __builtin_nontemporal_load((const u32x4*)(s + i + k * STEP));
        }
        if (c > seen) {
            if (copies_end(copies, seen, c)) return;
            seen = c;
        }
        if (ahead) {
#pragma unroll
            for (int k = 0; k < 4; ++k) __builtin_nontemporal_store(v[k], (u32x4*)(d + i + k * STEP));
            i += 4 * STEP;
        }
        for (; i < end; i += STEP) *(u32x4*)(d + i) = *(const u32x4*)(s + i);
        for (i = end + threadIdx.x; i < to; i += COPY_THREADS) d[i] = s[i];
    }
}
static_assert(COPY_PIECE == 4 * 16 * COPY_THREADS, "a piece is what the workgroup reads at once");

template <typename K>
int set_lds(K kern, size_t bytes, bool (&done)[MF_MAX_DEVICES]) {
    if (bytes <= 64 * 1024) return 0;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    if (dev >= 0 && dev < MF_MAX_DEVICES && done[dev]) return 0;
    e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, CB_MAX_BLOCKS / 8 + 4 * CB_MAX_ROWS);
    if (e == hipSuccess && dev >= 0 && dev < MF_MAX_DEVICES) done[dev] = true;
    return (int)e;
}

}  // namespace

// Markers of a fork: one for every 8192 entries from two on, as long as the assigning workgroup has no more than 256 KB of bitmaps
// to read.
static int fork_markers(int rows, int width, int num_blocks) {
    const int64_t n = std::min<int64_t>((int64_t)rows * width / 8192, 65536 / fork_words(num_blocks));
    return n < 2 ? 0 : (int)std::min<int64_t>(n, FORK_MARKERS);
}
// `ranks`; at most a copied block and the blocks of the new tokens for every row
static size_t fork_list_words(int rows, int block_size, int new_tokens) {
    return (1 + (size_t)rows * (2 + ((size_t)new_tokens + block_size - 1) / block_size) + 3) / 4 * 4;
}
extern "C" size_t mf_fork_blocks_workspace_bytes(int rows, int width, int num_blocks, int block_size, int new_tokens) {
    if (rows <= 0 || width <= 0 || num_blocks <= 0 || num_blocks > CB_MAX_BLOCKS || block_size <= 0 || new_tokens < 0) return 0;
    return sizeof(int32_t) * (fork_list_words(rows, block_size, new_tokens) +
                              (size_t)fork_markers(rows, width, num_blocks) * fork_words(num_blocks));
}

extern "C" int mf_fork_blocks(int32_t* tables_out, int32_t* lens_out, int32_t* slots, int32_t* copies, int32_t* missing,
                              const int32_t* tables, const int32_t* lens, const int32_t* parents, const uint8_t* held, int rows,
                              int width, int num_blocks, int block_size, int new_tokens, int window, int sinks, void* workspace,
                              size_t workspace_bytes, void* stream) {
    MF_REQUIRE(rows > 0 && width > 0 && block_size > 0 && new_tokens >= 0 && window >= 0 && sinks >= 0, "fork_blocks: bad sizes");
    MF_REQUIRE(num_blocks > 0 && num_blocks <= CB_MAX_BLOCKS, "fork_blocks: %d blocks, 1 to %d are served", num_blocks, CB_MAX_BLOCKS);
    MF_REQUIRE(rows <= CB_MAX_ROWS, "fork_blocks: %d rows, up to %d are served", rows, CB_MAX_ROWS);
    MF_REQUIRE((int64_t)width * block_size + new_tokens <= 0x7fffffffLL && (int64_t)num_blocks * block_size <= 0x7fffffffLL &&
                   (int64_t)rows * (2 + ((int64_t)new_tokens + block_size - 1) / block_size) <= 0x7fffffffLL,
               "fork_blocks: positions or slots overflow 32 bits");
    MF_REQUIRE(window > 0 || sinks == 0, "fork_blocks: sinks go with a window");
    MF_REQUIRE(tables_out && lens_out && copies && missing && tables && lens && (slots || new_tokens == 0), "fork_blocks: null argument");
    MF_REQUIRE(tables_out != tables && lens_out != lens, "fork_blocks: a row is read by all its children: the outputs need tensors of their own");
    const size_t need = mf_fork_blocks_workspace_bytes(rows, width, num_blocks, block_size, new_tokens);
    MF_REQUIRE(workspace && workspace_bytes >= need, "fork_blocks: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    MF_REQUIRE(((uintptr_t)workspace & 15) == 0, "fork_blocks: workspace must be 16-byte aligned");
    int32_t* ws = (int32_t*)workspace;
    const int markers = fork_markers(rows, width, num_blocks);
    const ForkArgs a = {tables_out, lens_out, slots, copies, missing, tables, lens, parents, held, ws + 1 + rows, ws,
                        (uint32_t*)ws + fork_list_words(rows, block_size, new_tokens), markers, rows, width, num_blocks, block_size, new_tokens, window, sinks};
    hipStream_t st = (hipStream_t)stream;
    const size_t bitmap = (size_t)fork_words(num_blocks) * 4, lds = bitmap + 4 * (size_t)rows;
    const bool small = (int64_t)rows * width <= 8192;
    static bool set[3][MF_MAX_DEVICES] = {};
    int rc;
    if (small) {
        if ((rc = set_lds(fork_assign_kernel<true>, lds, set[1]))) return rc;
        hipLaunchKernelGGL(fork_assign_kernel<true>, dim3(1), dim3(CB_THREADS), lds, st, a);
    } else {
        if (markers) {
            if ((rc = set_lds(fork_mark_kernel, bitmap, set[2]))) return rc;
            hipLaunchKernelGGL(fork_mark_kernel, dim3(markers), dim3(CB_THREADS), bitmap, st, a);
        } else {
            hipLaunchKernelGGL(fork_gather_kernel, dim3((rows + 3) / 4), dim3(256), 0, st, a);
        }
        if ((rc = MF_LAUNCH_CHECK())) return rc;
        if ((rc = set_lds(fork_assign_kernel<false>, lds, set[0]))) return rc;
        hipLaunchKernelGGL(fork_assign_kernel<false>, dim3(1), dim3(CB_THREADS), lds, st, a);
    }
    if ((rc = MF_LAUNCH_CHECK())) return rc;
    if (new_tokens > FORK_FILL) hipLaunchKernelGGL(fork_fill_kernel, dim3(rows), dim3(256), 0, st, a);
    return MF_LAUNCH_CHECK();
}

extern "C" size_t mf_compact_blocks_workspace_bytes(int num_blocks) {
    return num_blocks > 0 ? 2 * (size_t)num_blocks * sizeof(int32_t) : 0;
}

extern "C" int mf_compact_blocks(int32_t* tables_out, int32_t* copies, int32_t* live, const int32_t* tables, const uint8_t* held,
                                 int rows, int width, int num_blocks, int block_size, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    MF_REQUIRE(rows > 0 && width > 0 && block_size > 0, "compact_blocks: bad sizes");
    MF_REQUIRE(num_blocks > 0 && num_blocks <= CB_MAX_BLOCKS, "compact_blocks: %d blocks, 1 to %d are served", num_blocks, CB_MAX_BLOCKS);
    MF_REQUIRE(tables_out && live && tables && (copies || num_blocks < 2), "compact_blocks: null argument");
    const size_t need = mf_compact_blocks_workspace_bytes(num_blocks);
    MF_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0,
               "compact_blocks: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    const int64_t entries = (int64_t)rows * width;
    MF_REQUIRE(entries <= 0x7fffffffLL, "compact_blocks: the table overflows 32 bits");
    int32_t* ws = (int32_t*)workspace;
    const CompactArgs a = {copies, live, ws, ws + num_blocks, tables, held, entries, num_blocks, block_size};
    hipStream_t st = (hipStream_t)stream;
    const size_t lds = ((size_t)num_blocks + 31) / 32 * 4;
    static bool set[MF_MAX_DEVICES] = {};
    int rc;
    if ((rc = set_lds(compact_plan_kernel, lds, set))) return rc;
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(CB_THREADS), lds, st, a);
    if ((rc = MF_LAUNCH_CHECK())) return rc;
    hipLaunchKernelGGL(compact_remap_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, st, tables_out, tables, ws,
                       entries, num_blocks);
    return MF_LAUNCH_CHECK();
}

extern "C" int mf_copy_blocks(void* const* host_caches, const int32_t* host_row_bytes, int n_caches, const int32_t* copies,
                              int n_copies, int num_blocks, int block_size, void* stream) {
    MF_REQUIRE(n_caches >= 0 && n_copies >= 0 && num_blocks > 0 && block_size > 0, "copy_blocks: bad sizes");
    if (n_caches == 0 || n_copies == 0) return 0;
    MF_REQUIRE(host_caches && host_row_bytes && copies, "copy_blocks: null argument");
    for (int i = 0; i < n_caches; ++i) {
        MF_REQUIRE(host_caches[i] && host_row_bytes[i] > 0, "copy_blocks: null cache or empty row");
        MF_REQUIRE((int64_t)host_row_bytes[i] * block_size <= 0x7fffffffLL, "copy_blocks: a block of %lld bytes",
                   (long long)host_row_bytes[i] * block_size);
    }
    hipStream_t st = (hipStream_t)stream;
    for (int c0 = 0; c0 < n_caches; c0 += COPY_TENSORS) {
        CopyTensors t = {};
        const int n = std::min(COPY_TENSORS, n_caches - c0);
        int64_t block = 0;
        for (int i = 0; i < n; ++i) {
            t.base[i] = (uint8_t*)host_caches[c0 + i];
            t.row_bytes[i] = (uint32_t)host_row_bytes[c0 + i];
            block = std::max(block, (int64_t)block_size * host_row_bytes[c0 + i]);
        }
        const int pieces = (int)((block + COPY_PIECE - 1) / COPY_PIECE);
        const int64_t items = (int64_t)n_copies * n * pieces;
        const int64_t grid = std::min<int64_t>(items, n_copies <= COPY_SHORT ? 32768 : 2048);
        hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)grid), dim3(COPY_THREADS), 0, st, t, copies, n_copies, n, pieces,
                           num_blocks, block_size);
        const int rc = MF_LAUNCH_CHECK();
        if (rc) return rc;
    }
    return 0;
}
