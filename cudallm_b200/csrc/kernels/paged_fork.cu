// Bookkeeping of a paged cache's sequences: forking (sharing, copy on write, freeing, new pages) and compaction.
//
// A plan decides who gets which page (all of it integer prefix sums, so the result does not depend on any order of
// threads); then the tokens of every layer move and tables and references are written. The moves read and write each
// byte once and HBM bounds them; with few of them the plan's chain of dependent loads (parent, length, entry,
// references) does.
//
// One launch where plan and moves are small: every block makes the whole plan for itself, in shared memory, which costs no
// more time than one block making it, and moves its share (four beams: 13.7 us a call instead of 16). Otherwise two: a plan kernel into
// the workspace and a move kernel over the GPU, in place when the plan is done.
//
// Measured (B200, graph replay): 128 rows, 64 tails of 16 layers (69 MB copied) 31.2 us, of which the move is 21.3 (6.5 TB/s); 750 pages
// of 16 layers compacted (393 MB) 131 us (6.0 TB/s); four beams 5.1 us.
#include <algorithm>
#include <atomic>
#include <climits>

#include "common/check.h"
#include "kernels/kernels.h"
#include "kernels/launch.cuh"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"
#include "kernels/ptx.cuh"

namespace cudallm {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kEach = 16;  // pages of a thread in one pass over the references
constexpr int kMoveThreads = 256;
// Plans of up to 16384 pages (and 1024 rows) are made by 256 threads, whose barriers cost less (four beams: 5.0 us on the GPU instead of 8.1).
constexpr int kOneThreads = 256;
constexpr int kOnePages = 16384;
constexpr int kOneBlocks = 3;  // of the kernels that plan and move, on an SM
constexpr int kSharedRows = 4096;  // rows whose counters fit the plan's shared memory
constexpr unsigned kAll = 0xffffffffu;

// Exclusive prefix sum of one value per thread over a block; `total` gets the sum. Barriers on both sides.
template <int THREADS>
__device__ int block_scan(int v, int* sm, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(kAll, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = s;
    __syncthreads();
    int w = lane < THREADS / 32 ? sm[lane] : 0;  // every warp sums the warps' totals for itself
#pragma unroll
    for (int o = 1; o < THREADS / 32; o <<= 1) {
        const int t = __shfl_up_sync(kAll, w, o);
        if (lane >= o) w += t;
    }
    total = __shfl_sync(kAll, w, THREADS / 32 - 1);
    const int before = __shfl_sync(kAll, w, (warp + 31) & 31);
    return s - v + (warp > 0 ? before : 0);
}

__device__ __forceinline__ bool is_page(int p, int n_pages) { return p >= 0 && p < n_pages; }

// This thread's kEach references from p on (p a multiple of kEach); pages past the end read as `none`.
__device__ __forceinline__ void load_refs(const int* refs, int p, int n, int none, bool wide, int (&r)[kEach]) {
    if (wide && p + kEach <= n) {
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            const int4 v = *reinterpret_cast<const int4*>(refs + p + i);
            r[i] = v.x, r[i + 1] = v.y, r[i + 2] = v.z, r[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) r[i] = p + i < n ? refs[p + i] : none;
    }
}

// One warp copies `tokens` tokens of one head of one page of one layer, of k and of v.
template <int AT_ONCE>
__device__ __forceinline__ void copy_head(const cudallm_pages& pg, FastDiv by_row, int layer, int head, int src, int dst, int tokens) {
    const int per_row = pg.head_dim / 8, n = tokens * per_row, lane = threadIdx.x & 31;  // 16-byte words
    const long long base = layer * pg.layer_stride + head * pg.head_stride;
    const uint16_t *ks = static_cast<const uint16_t*>(pg.k) + base + src * pg.page_stride, *vs = static_cast<const uint16_t*>(pg.v) + base + src * pg.page_stride;
    uint16_t *kd = static_cast<uint16_t*>(pg.k) + base + dst * pg.page_stride, *vd = static_cast<uint16_t*>(pg.v) + base + dst * pg.page_stride;
    for (int c0 = lane; c0 < n; c0 += 32 * AT_ONCE) {
        uint4 k[AT_ONCE], v[AT_ONCE];
        long long at[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int c = c0 + 32 * i;
            if (c >= n) break;
            const int t = div_by(c, by_row);
            at[i] = t * pg.token_stride + (c - t * per_row) * 8;
            k[i] = *reinterpret_cast<const uint4*>(ks + at[i]);
            v[i] = *reinterpret_cast<const uint4*>(vs + at[i]);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (c0 + 32 * i >= n) break;
            *reinterpret_cast<uint4*>(kd + at[i]) = k[i];
            *reinterpret_cast<uint4*>(vd + at[i]) = v[i];
        }
    }
}

// ---- fork ----------------------------------------------------------------------------------------

struct OutRow {
    int parent, len, from, start;  // the parent (-1: empty), its length, its entries that are taken over, rank of the first new page
};
struct OldRow {
    int full, held, children, kept;  // full pages, entries held, children, whether a child takes over what follows the full pages
    int open;                        // the page after the full ones, or -1
};
struct Copy {
    int src, dst, tokens, pad;
};
struct ForkPlan {
    int* totals;  // new pages found, copies, pages missing
    OutRow* out;
    Copy* copies;
    OldRow* old;
    int *fresh, *counters, *found;
};
constexpr int kOneRows = 512, kOneFound = 2048;  // what a plan in shared memory has room for
constexpr int kOneEntries = 16384;               // and of the tables, which one block writes then
// Heads of pages that may move in one launch. With more, the plan repeated by each block costs more than a second launch:
// 64 tails of 16 layers take 31.0 us in two and 33.9 in one (compacting 3001 pages: 131.2 and 130.5).
constexpr long long kOneHeads = 8192;

// Bytes of a plan for that many rows and new pages, and its parts in 16-byte aligned memory.
__host__ __device__ inline size_t fork_plan_bytes(int rows, int found) { return 16 + (2 * 16 + 20 + 3 * 4) * static_cast<size_t>(rows) + 4 * static_cast<size_t>(found); }
__host__ __device__ inline ForkPlan fork_plan(void* memory, int rows, int found) {
    char* p = static_cast<char*>(memory);
    ForkPlan s;
    s.totals = reinterpret_cast<int*>(p);
    s.out = reinterpret_cast<OutRow*>(p + 16);
    s.copies = reinterpret_cast<Copy*>(s.out + rows);
    s.found = reinterpret_cast<int*>(s.copies + rows);
    s.old = reinterpret_cast<OldRow*>(s.found + found);
    s.fresh = reinterpret_cast<int*>(s.old + rows);
    s.counters = s.fresh + rows;
    return s;
}

__device__ __forceinline__ int row_len(const cudallm_pages& pg, const cudallm_fork_args& a, int r) {
    const long long cap = static_cast<long long>(a.table_width) * pg.page_size;
    return static_cast<int>(min(static_cast<long long>(max(a.lens[r], 0)), cap));
}

// The plan of a fork, by all threads of a block. `counters`: room for two ints for each of n_rows. Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void plan_fork(const cudallm_pages& pg, const cudallm_fork_args& a, const ForkPlan& s, int* counters, bool wide) {
    __shared__ int sm[32];
    __shared__ unsigned long long over;
    int refs[kEach];  // of the first pass, under way while the rows are looked at
    load_refs(a.refs, threadIdx.x * kEach, pg.n_pages, 1, wide, refs);
    int *children = counters, *first = counters + a.n_rows;
    for (int r = threadIdx.x; r < a.n_rows; r += THREADS) {
        children[r] = 0;
        first[r] = INT_MAX;
    }
    if (threadIdx.x == 0) over = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_out; i += THREADS) {
        const int p = a.parents[i];
        if (p >= 0 && p < a.n_rows) {
            atomicAdd(&children[p], 1);
            atomicMin(&first[p], i);
        }
    }
    for (int r = threadIdx.x; r < a.n_rows; r += THREADS) {
        const int full = row_len(pg, a, r) / pg.page_size;
        const int* row = a.tables + r * a.table_stride;
        int held = full, open = -1;
        for (; held < a.table_width; ++held) {
            const int e = row[held];
            if (!is_page(e, pg.n_pages)) break;
            if (held == full) open = e;
        }
        s.old[r] = {full, held, 0, open >= 0 && a.refs[open] == 1, open};
    }
    __syncthreads();
    for (int r = threadIdx.x; r < a.n_rows; r += THREADS) {  // a thread's own rows
        s.old[r].children = children[r];
        if (children[r] == 0) s.old[r].kept = 0;
    }
    __syncthreads();
    int base = 0;
    for (int i0 = 0; i0 < a.n_out; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        int fresh = 0;
        OutRow o{-1, 0, 0, 0};
        if (i < a.n_out) {
            const int p = a.parents[i];
            if (p >= 0 && p < a.n_rows) {
                const OldRow old = s.old[p];
                o.parent = p;
                o.len = row_len(pg, a, p);
                o.from = old.kept && first[p] == i ? old.held : old.full;
                const long long want = (static_cast<long long>(o.len) + a.room + pg.page_size - 1) / pg.page_size;
                fresh = static_cast<int>(max(0LL, min(want, static_cast<long long>(a.table_width)) - o.from));
                if (want > a.table_width) atomicAdd(&over, static_cast<unsigned long long>(want - a.table_width));
            }
        }
        int total;
        o.start = base + block_scan<THREADS>(fresh, sm, total);
        if (i < a.n_out) {
            s.out[i] = o;
            s.fresh[i] = fresh;
        }
        base += total;
    }
    int found = 0;
    for (int p0 = 0; p0 < pg.n_pages && found < base; p0 += (THREADS * kEach)) {
        const int p = p0 + threadIdx.x * kEach;
        if (p0 > 0) load_refs(a.refs, p, pg.n_pages, 1, wide, refs);
        int n = 0, total;
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += refs[i] == 0;
        int at = found + block_scan<THREADS>(n, sm, total);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (refs[i] == 0 && at < base) s.found[at] = p + i;
            at += refs[i] == 0;
        }
        found += total;
    }
    found = min(found, base);
    __syncthreads();
    int copies = 0;
    for (int i0 = 0; i0 < a.n_out; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        Copy c{0, 0, 0, 0};
        if (i < a.n_out) {
            const OutRow o = s.out[i];
            if (o.parent >= 0) {
                const OldRow old = s.old[o.parent];
                const int tail = o.len - old.full * pg.page_size;
                const bool keeps = old.kept && first[o.parent] == i;
                if (!keeps && tail > 0 && old.open >= 0 && s.fresh[i] > 0 && o.start < found) c = {old.open, s.found[o.start], tail, 0};
            }
        }
        int total;
        const int at = copies + block_scan<THREADS>(c.tokens > 0, sm, total);
        if (c.tokens > 0) s.copies[at] = c;
        copies += total;
    }
    if (threadIdx.x == 0) {
        s.totals[0] = found;
        s.totals[1] = copies;
        const unsigned long long missing = over + static_cast<unsigned long long>(base - found);
        s.totals[2] = static_cast<int>(min(missing, static_cast<unsigned long long>(INT_MAX)));
    }
    __syncthreads();
}

// Rows of the outputs, and the references that the parents' pages lose or gain: thread `me` of `threads` takes entries.
__device__ __forceinline__ void fork_rows(const cudallm_pages& pg, const cudallm_fork_args& a, const ForkPlan& s, int rows, long long me, long long threads) {
    const int n_found = s.totals[0];
    const long long entries = static_cast<long long>(rows) * a.table_width;
    for (long long x = me; x < entries; x += threads) {
        const int i = static_cast<int>(x / a.table_width), j = static_cast<int>(x % a.table_width);
        if (i < a.n_rows) {
            const OldRow old = s.old[i];
            const int gain = j < old.full ? old.children - 1 : old.kept ? 0 : -1;
            if (j < old.held && gain != 0) {
                const int p = a.tables[i * a.table_stride + j];
                if (is_page(p, pg.n_pages)) atomicAdd(&a.refs_out[p], gain);
            }
        }
        if (i < a.n_out) {
            const OutRow o = s.out[i];
            int e = -1;
            if (o.parent >= 0 && j < o.from) {
                e = a.tables[o.parent * a.table_stride + j];
                if (!is_page(e, pg.n_pages)) e = -1;
            } else if (j < o.from + s.fresh[i] && o.start + j - o.from < n_found) {
                e = s.found[o.start + j - o.from];
                atomicAdd(&a.refs_out[e], 1);
            }
            a.tables_out[i * a.table_out_stride + j] = e;
        }
    }
    for (long long i = me; i < a.n_out; i += threads) a.lens_out[i] = s.out[i].len;
}

// Copies: warp `warp` of `warps` takes every so manieth head of a page.
template <int AT_ONCE>
__device__ __forceinline__ void fork_copies(const cudallm_pages& pg, const ForkPlan& s, FastDiv by_row, long long warp, long long warps) {
    const long long units = static_cast<long long>(s.totals[1]) * pg.n_layers * pg.n_kv_heads;
    for (long long u = warp; u < units; u += warps) {
        const int head = static_cast<int>(u % pg.n_kv_heads), layer = static_cast<int>(u / pg.n_kv_heads % pg.n_layers);
        const Copy c = s.copies[u / pg.n_kv_heads / pg.n_layers];
        copy_head<AT_ONCE>(pg, by_row, layer, head, c.src, c.dst, c.tokens);
    }
}

// Block 0 plans; the others copy the references, which the move kernel then changes.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) fork_plan_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_fork_args a, ForkPlan s,
                                                            bool wide) {
    extern __shared__ int shared_counters[];
    grid_dep_wait();
    grid_dep_launch();
    if (blockIdx.x > 0) {
        for (int p = (blockIdx.x - 1) * THREADS + threadIdx.x; p < pg.n_pages; p += (gridDim.x - 1) * THREADS) a.refs_out[p] = a.refs[p];
        return;
    }
    plan_fork<THREADS>(pg, a, s, a.n_rows <= kSharedRows ? shared_counters : s.counters, wide);
    if (threadIdx.x == 0) *a.missing = s.totals[2];
}

// The first `writers` blocks write rows; the others' warps copy.
__global__ void __launch_bounds__(kMoveThreads) fork_move_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_fork_args a, ForkPlan s,
                                                                 int rows, int writers, FastDiv by_row) {
    grid_dep_wait();
    if (static_cast<int>(blockIdx.x) < writers) {
        fork_rows(pg, a, s, rows, static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x, static_cast<long long>(writers) * kMoveThreads);
    } else {
        constexpr int kWarps = kMoveThreads / 32;
        fork_copies<4>(pg, s, by_row, static_cast<long long>(blockIdx.x - writers) * kWarps + threadIdx.x / 32, static_cast<long long>(gridDim.x - writers) * kWarps);
    }
}

// The whole fork: block 0 writes the rows, the other blocks copy.
__global__ void __launch_bounds__(kOneThreads) fork_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_fork_args a, int rows, FastDiv by_row,
                                                           bool wide) {
    extern __shared__ __align__(16) char room[];
    const ForkPlan s = fork_plan(room, rows, kOneFound);
    grid_dep_wait();
    grid_dep_launch();
    if (blockIdx.x == 0) {
        for (int p = threadIdx.x; p < pg.n_pages; p += kOneThreads) a.refs_out[p] = a.refs[p];
    }
    plan_fork<kOneThreads>(pg, a, s, s.counters, wide);
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) *a.missing = s.totals[2];
        fork_rows(pg, a, s, rows, threadIdx.x, kOneThreads);
    } else {
        constexpr int kWarps = kOneThreads / 32;
        fork_copies<4>(pg, s, by_row, static_cast<long long>(blockIdx.x - 1) * kWarps + threadIdx.x / 32, static_cast<long long>(gridDim.x - 1) * kWarps);
    }
}

// ---- compact ---------------------------------------------------------------------------------------

struct CompactPlan {
    int* totals;          // pages in use, moves
    int *to, *src, *dst;  // new place of a page that moves; the moves (at most half of the pages: none moves onto one that stays)
};
__host__ __device__ inline size_t compact_plan_bytes(int n_pages) { return 16 + 8 * static_cast<size_t>(n_pages); }
__host__ __device__ inline CompactPlan compact_plan(void* memory, int n_pages) {
    int* p = static_cast<int*>(memory);
    return {p, p + 4, p + 4 + n_pages, p + 4 + n_pages + n_pages / 2};
}

// The plan of a compaction, by all threads of a block. Ends with a barrier.
template <int THREADS>
__device__ __forceinline__ void plan_compact(const cudallm_pages& pg, const cudallm_compact_args& a, const CompactPlan& s, bool wide) {
    __shared__ int sm[32];
    int refs[kEach], live = 0;
    for (int p0 = 0; p0 < pg.n_pages; p0 += (THREADS * kEach)) {
        load_refs(a.refs, p0 + threadIdx.x * kEach, pg.n_pages, 0, wide, refs);
        int n = 0, total;
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += refs[i] > 0;
        block_scan<THREADS>(n, sm, total);
        live += total;
    }
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < pg.n_pages; p0 += (THREADS * kEach)) {
        const int p = p0 + threadIdx.x * kEach;
        if (pg.n_pages > (THREADS * kEach)) load_refs(a.refs, p, pg.n_pages, 0, wide, refs);
        int n = 0, total;  // holes in the low half, movers in the high one: a pass has at most 16384 of each
        static_assert(THREADS * kEach < 1 << 15, "two counts in one int");
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += refs[i] > 0 ? (p + i >= live) << 16 : p + i < live;
        const int at = block_scan<THREADS>(n, sm, total);
        int h = holes + (at & 0xffff), m = movers + (at >> 16);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (refs[i] > 0 && p + i >= live) s.src[m++] = p + i;
            if (refs[i] <= 0 && p + i < live) s.dst[h++] = p + i;
        }
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += THREADS) s.to[s.src[k]] = s.dst[k];
    if (threadIdx.x == 0) {
        s.totals[0] = live;
        s.totals[1] = movers;
    }
    __syncthreads();
}

// Carries a plan out: thread `me` of `threads`.
template <int AT_ONCE>
__device__ __forceinline__ void move_compact(const cudallm_pages& pg, const cudallm_compact_args& a, const CompactPlan& s, FastDiv by_row, long long me, long long threads) {
    const int live = s.totals[0];
    if (me == 0) *a.live = live;
    const long long units = static_cast<long long>(s.totals[1]) * pg.n_layers * pg.n_kv_heads;
    for (long long u = me / 32; u < units; u += threads / 32) {
        const int head = static_cast<int>(u % pg.n_kv_heads), layer = static_cast<int>(u / pg.n_kv_heads % pg.n_layers);
        const int k = static_cast<int>(u / pg.n_kv_heads / pg.n_layers);
        copy_head<AT_ONCE>(pg, by_row, layer, head, s.src[k], s.dst[k], pg.page_size);
    }
    for (long long p = me; p < pg.n_pages; p += threads) {
        const int r = a.refs[p];
        if (p >= live) a.refs_out[p] = 0;
        if (r > 0) a.refs_out[p < live ? p : s.to[p]] = r;
    }
    const long long entries = static_cast<long long>(a.n_rows) * a.table_width;
    for (long long e = me; e < entries; e += threads) {
        const long long r = e / a.table_width, j = e % a.table_width;
        const int p = a.tables[r * a.table_stride + j];
        a.tables_out[r * a.table_out_stride + j] = !is_page(p, pg.n_pages) ? -1 : p >= live && a.refs[p] > 0 ? s.to[p] : p;
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) compact_plan_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_compact_args a, CompactPlan s,
                                                               bool wide) {
    grid_dep_wait();
    grid_dep_launch();
    plan_compact<THREADS>(pg, a, s, wide);
}

__global__ void __launch_bounds__(kMoveThreads) compact_move_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_compact_args a, CompactPlan s,
                                                                    FastDiv by_row) {
    grid_dep_wait();
    move_compact<4>(pg, a, s, by_row, static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x, static_cast<long long>(gridDim.x) * kMoveThreads);
}

__global__ void __launch_bounds__(kOneThreads) compact_kernel(const __grid_constant__ cudallm_pages pg, const __grid_constant__ cudallm_compact_args a, FastDiv by_row,
                                                              bool wide) {
    extern __shared__ __align__(16) char room[];
    const CompactPlan s = compact_plan(room, pg.n_pages);
    grid_dep_wait();
    grid_dep_launch();
    plan_compact<kOneThreads>(pg, a, s, wide);
    move_compact<4>(pg, a, s, by_row, static_cast<long long>(blockIdx.x) * kOneThreads + threadIdx.x, static_cast<long long>(gridDim.x) * kOneThreads);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

size_t pages_workspace_bytes(int n_pages, int rows) {
    if (n_pages < 1 || rows < 0 || rows > kMaxPageRows) return 0;
    return std::max(fork_plan_bytes(rows, n_pages), compact_plan_bytes(n_pages));
}

void launch_paged_fork(const cudallm_pages& pg, const cudallm_fork_args& a, cudaStream_t stream) {
    const int rows = std::max(a.n_rows, a.n_out), sms = num_sms();
    const FastDiv by_row = fast_div(pg.head_dim / 8);
    const bool wide = aligned16(a.refs);
    const long long heads = static_cast<long long>(a.n_out) * pg.n_layers * pg.n_kv_heads;  // most that are copied
    const long long most_new = a.n_out * (2LL + a.room / pg.page_size);
    if (pg.n_pages <= kOnePages && rows <= kOneRows && most_new <= kOneFound && static_cast<long long>(rows) * a.table_width <= kOneEntries &&
        heads <= kOneHeads) {
        constexpr int kWarps = kOneThreads / 32;
        const int blocks = 1 + static_cast<int>(std::min<long long>(kOneBlocks * sms - 1, std::max<long long>(1, (heads + kWarps - 1) / kWarps)));
        launch_kernel(fork_kernel, dim3(blocks), dim3(kOneThreads), fork_plan_bytes(rows, kOneFound), stream, true, pg, a, rows, by_row, wide);
        return;
    }
    const ForkPlan s = fork_plan(a.workspace, rows, pg.n_pages);
    const bool small = pg.n_pages <= kOnePages && rows <= kPlanThreads;
    const int threads = small ? kOneThreads : kPlanThreads, copiers = std::min(sms, (pg.n_pages + threads - 1) / threads);  // of the references
    const size_t smem = a.n_rows <= kSharedRows ? 8 * static_cast<size_t>(a.n_rows) : 0;
    launch_kernel(small ? fork_plan_kernel<kOneThreads> : fork_plan_kernel<kPlanThreads>, dim3(1 + copiers), dim3(threads), smem, stream, true, pg, a, s, wide);
    if (rows == 0) return;
    const int movers = static_cast<int>(std::min<long long>(8LL * sms, (heads + kMoveThreads / 32 - 1) / (kMoveThreads / 32)));
    const long long entries = static_cast<long long>(rows) * a.table_width;
    const int writers = static_cast<int>(std::min<long long>(sms, 1 + entries / (4 * kMoveThreads)));
    launch_kernel(fork_move_kernel, dim3(writers + movers), dim3(kMoveThreads), 0, stream, true, pg, a, s, rows, writers, by_row);
}

void launch_paged_compact(const cudallm_pages& pg, const cudallm_compact_args& a, cudaStream_t stream) {
    const FastDiv by_row = fast_div(pg.head_dim / 8);
    const bool wide = aligned16(a.refs);
    const long long heads = static_cast<long long>(pg.n_pages / 2) * pg.n_layers * pg.n_kv_heads;  // most that move
    if (pg.n_pages <= kOnePages && heads <= kOneHeads) {
        const size_t smem = compact_plan_bytes(pg.n_pages);
        static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use its shared memory
        allow_shared(compact_kernel, static_cast<int>(compact_plan_bytes(kOnePages)), allowed);
        const long long most = 1 + (heads + kOneThreads / 32 - 1) / (kOneThreads / 32);
        launch_kernel(compact_kernel, dim3(static_cast<int>(std::min<long long>(kOneBlocks * num_sms(), most))), dim3(kOneThreads), smem, stream, true, pg, a, by_row, wide);
        return;
    }
    const CompactPlan s = compact_plan(a.workspace, pg.n_pages);
    const bool small = pg.n_pages <= kOnePages;
    launch_kernel(small ? compact_plan_kernel<kOneThreads> : compact_plan_kernel<kPlanThreads>, dim3(1), dim3(small ? kOneThreads : kPlanThreads), 0, stream, true,
                  pg, a, s, wide);
    const int blocks = static_cast<int>(std::min<long long>(8LL * num_sms(), 1 + (heads + kMoveThreads / 32 - 1) / (kMoveThreads / 32)));
    launch_kernel(compact_move_kernel, dim3(blocks), dim3(kMoveThreads), 0, stream, true, pg, a, s, by_row);
}

}  // namespace cudallm
