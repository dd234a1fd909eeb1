// Bookkeeping of a paged cache's sequences: forking (sharing, copy on write, freeing, new pages) and compaction.
//
// Both run as a plan kernel of one block, which decides who gets which page (all of it integer prefix sums, so the
// result does not depend on any order of threads), and a kernel over the whole GPU that moves the tokens of every
// layer and writes tables and references.
#include <climits>

#include "common/check.h"
#include "kernels/paged.h"

namespace cudallm {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;

// Exclusive prefix sum of one value per thread over the block; `total` gets the sum. Barriers on both sides.
__device__ int block_scan(int v, int* sm, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) sm[warp] = s;
    __syncthreads();
    if (warp == 0) {
        int w = sm[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += t;
        }
        sm[lane] = w;
    }
    __syncthreads();
    total = sm[31];
    return s - v + (warp > 0 ? sm[warp - 1] : 0);
}

// Scratch of a fork: per parent row the number of children, the first child, the entries held and whether the pages
// from the first not full one on are its own; per new row the first rank among the new pages; the new pages by rank.
struct ForkScratch {
    int *children, *first, *held, *alone, *start, *fresh, *found;
    int* n_found;
};

__host__ __device__ inline ForkScratch fork_scratch(void* workspace, int rows) {
    int* p = static_cast<int*>(workspace);
    ForkScratch s;
    s.n_found = p;
    p += 64;
    s.children = p;
    s.first = p + rows;
    s.held = p + 2 * rows;
    s.alone = p + 3 * rows;
    s.start = p + 4 * rows;
    s.fresh = p + 5 * rows;
    s.found = p + 6 * rows;
    return s;
}

__device__ __forceinline__ bool is_page(int p, int n_pages) { return p >= 0 && p < n_pages; }

__device__ __forceinline__ int row_len(const cudallm_pages& pg, const cudallm_fork_args& a, int r) {
    const long long cap = static_cast<long long>(a.table_width) * pg.page_size;
    return static_cast<int>(min(static_cast<long long>(max(a.lens[r], 0)), cap));
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(cudallm_pages pg, cudallm_fork_args a, ForkScratch s) {
    __shared__ int sm[32];
    __shared__ unsigned long long sm_over;
    for (int r = threadIdx.x; r < a.n_rows; r += kPlanThreads) {
        s.children[r] = 0;
        s.first[r] = INT_MAX;
    }
    if (threadIdx.x == 0) sm_over = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_out; i += kPlanThreads) {
        const int p = a.parents[i];
        if (p >= 0 && p < a.n_rows) {
            atomicAdd(&s.children[p], 1);
            atomicMin(&s.first[p], i);
        }
    }
    for (int r = threadIdx.x; r < a.n_rows; r += kPlanThreads) {
        const int full = row_len(pg, a, r) / pg.page_size;
        const int* row = a.tables + r * a.table_stride;
        int held = full;
        while (held < a.table_width && is_page(row[held], pg.n_pages)) ++held;
        s.held[r] = held;
        s.alone[r] = held > full && a.refs[row[full]] == 1;
    }
    __syncthreads();
    int base = 0;
    for (int i0 = 0; i0 < a.n_out; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        int fresh = 0;
        if (i < a.n_out) {
            const int p = a.parents[i];
            if (p >= 0 && p < a.n_rows) {
                const long long len = row_len(pg, a, p);
                const long long want = (len + a.room + pg.page_size - 1) / pg.page_size;
                const bool keeps = s.alone[p] && s.first[p] == i;
                const int from = keeps ? s.held[p] : static_cast<int>(len / pg.page_size);
                fresh = static_cast<int>(max(0LL, min(want, static_cast<long long>(a.table_width)) - from));
                if (want > a.table_width) atomicAdd(&sm_over, static_cast<unsigned long long>(want - a.table_width));
            }
        }
        int total;
        const int at = block_scan(fresh, sm, total);
        if (i < a.n_out) {
            s.start[i] = base + at;
            s.fresh[i] = fresh;
        }
        base += total;
    }
    int found = 0;
    for (int p0 = 0; p0 < pg.n_pages && found < base; p0 += kPlanThreads) {
        const int p = p0 + threadIdx.x;
        const int free = p < pg.n_pages && a.refs[p] == 0;
        int total;
        const int at = block_scan(free, sm, total);
        if (free && found + at < base) s.found[found + at] = p;
        found += total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        found = min(found, base);
        *s.n_found = found;
        const unsigned long long missing = sm_over + static_cast<unsigned long long>(base - found);
        *a.missing = static_cast<int>(min(missing, static_cast<unsigned long long>(INT_MAX)));
    }
}

// Copies `tokens` tokens of one page of one layer, all heads, of k and v.
template <typename Vec>
__device__ void copy_page(const cudallm_pages& pg, int layer, int src, int dst, int tokens) {
    constexpr int kElems = sizeof(Vec) / 2;
    const int per_row = pg.head_dim / kElems;
    const int total = tokens * pg.n_kv_heads * per_row;
    const long long l = layer * pg.layer_stride;
    for (int u = threadIdx.x; u < total; u += blockDim.x) {
        const int c = u % per_row, t = u / per_row % tokens, h = u / per_row / tokens;
        const long long at = l + h * pg.head_stride + t * pg.token_stride + c * kElems;
        const long long from = at + src * pg.page_stride, to = at + dst * pg.page_stride;
        *reinterpret_cast<Vec*>(static_cast<uint16_t*>(pg.k) + to) = *reinterpret_cast<const Vec*>(static_cast<const uint16_t*>(pg.k) + from);
        *reinterpret_cast<Vec*>(static_cast<uint16_t*>(pg.v) + to) = *reinterpret_cast<const Vec*>(static_cast<const uint16_t*>(pg.v) + from);
    }
}

// Block (i, y): y == 0 writes row i of the outputs and, for parent row i, the references its pages lose or gain;
// the blocks of a row share its copy's layers.
__global__ void __launch_bounds__(kMoveThreads) fork_move_kernel(cudallm_pages pg, cudallm_fork_args a, ForkScratch s) {
    const int i = blockIdx.x;
    const int n_found = *s.n_found;
    if (blockIdx.y == 0 && i < a.n_rows) {
        const int full = row_len(pg, a, i) / pg.page_size, held = s.held[i], kids = s.children[i];
        const bool kept = s.alone[i] && kids > 0;
        for (int j = threadIdx.x; j < held; j += kMoveThreads) {
            const int p = a.tables[i * a.table_stride + j];
            const int gain = j < full ? kids - 1 : kept ? 0 : -1;
            if (gain != 0 && is_page(p, pg.n_pages)) atomicAdd(&a.refs_out[p], gain);
        }
    }
    if (i >= a.n_out) return;
    const int parent = a.parents[i];
    const bool alive = parent >= 0 && parent < a.n_rows;
    const int len = alive ? row_len(pg, a, parent) : 0, full = len / pg.page_size;
    const bool keeps = alive && s.alone[parent] && s.first[parent] == i;
    const int from = keeps ? s.held[parent] : full, start = s.start[i], fresh = s.fresh[i];
    const int* old = a.tables + static_cast<long long>(alive ? parent : 0) * a.table_stride;
    if (blockIdx.y == 0) {
        for (int j = threadIdx.x; j < a.table_width; j += kMoveThreads) {
            int e = -1;
            if (alive && j < from) {
                e = is_page(old[j], pg.n_pages) ? old[j] : -1;
            } else if (alive && j < from + fresh && start + j - from < n_found) {
                e = s.found[start + j - from];
                atomicAdd(&a.refs_out[e], 1);
            }
            a.tables_out[i * a.table_out_stride + j] = e;
        }
        if (threadIdx.x == 0) a.lens_out[i] = len;
    }
    const int tail = len - full * pg.page_size;
    if (alive && !keeps && tail > 0 && s.held[parent] > full && fresh > 0 && start < n_found) {
        for (int l = blockIdx.y; l < pg.n_layers; l += gridDim.y) copy_page<uint4>(pg, l, old[full], s.found[start], tail);
    }
}

struct CompactScratch {
    int *to, *src, *dst;
    int* n_moves;
};

__host__ __device__ inline CompactScratch compact_scratch(void* workspace, int n_pages) {
    int* p = static_cast<int*>(workspace);
    CompactScratch s;
    s.n_moves = p;
    p += 64;
    s.to = p;
    s.src = p + n_pages;
    s.dst = p + 2 * static_cast<size_t>(n_pages);
    return s;
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(cudallm_pages pg, cudallm_compact_args a, CompactScratch s) {
    __shared__ int sm[32];
    int live = 0;
    for (int p0 = 0; p0 < pg.n_pages; p0 += kPlanThreads) {
        const int p = p0 + threadIdx.x;
        int total;
        block_scan(p < pg.n_pages && a.refs[p] > 0, sm, total);
        live += total;
    }
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < pg.n_pages; p0 += kPlanThreads) {
        const int p = p0 + threadIdx.x;
        const bool in = p < pg.n_pages, used = in && a.refs[p] > 0;
        const bool hole = in && !used && p < live, mover = used && p >= live;
        int total;
        const int h = block_scan(hole, sm, total) + holes;
        holes += total;
        const int m = block_scan(mover, sm, total) + movers;
        movers += total;
        if (hole) s.dst[h] = p;
        if (mover) s.src[m] = p;
        if (in) {
            s.to[p] = p;
            a.refs_out[p] = used && p < live ? a.refs[p] : 0;
        }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += kPlanThreads) {
        s.to[s.src[k]] = s.dst[k];
        a.refs_out[s.dst[k]] = a.refs[s.src[k]];
    }
    if (threadIdx.x == 0) {
        *s.n_moves = movers;
        *a.live = live;
    }
}

__global__ void __launch_bounds__(kMoveThreads) compact_move_kernel(cudallm_pages pg, cudallm_compact_args a, CompactScratch s) {
    const long long moves = static_cast<long long>(*s.n_moves) * pg.n_layers;
    for (long long u = blockIdx.x; u < moves; u += gridDim.x) {
        copy_page<uint4>(pg, static_cast<int>(u % pg.n_layers), s.src[u / pg.n_layers], s.dst[u / pg.n_layers], pg.page_size);
    }
    const long long entries = static_cast<long long>(a.n_rows) * a.table_width;
    for (long long e = static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x; e < entries;
         e += static_cast<long long>(gridDim.x) * kMoveThreads) {
        const long long r = e / a.table_width, j = e % a.table_width;
        const int p = a.tables[r * a.table_stride + j];
        a.tables_out[r * a.table_out_stride + j] = is_page(p, pg.n_pages) ? s.to[p] : -1;
    }
}

}  // namespace

size_t pages_workspace_bytes(int n_pages, int rows) {
    if (n_pages < 1 || rows < 0 || rows > kMaxPageRows) return 0;
    const size_t fork = 6 * static_cast<size_t>(rows) + n_pages, compact = 3 * static_cast<size_t>(n_pages);
    return 4 * (64 + (fork > compact ? fork : compact));
}

void launch_paged_fork(const cudallm_pages& pg, const cudallm_fork_args& a, cudaStream_t stream) {
    const int rows = a.n_rows > a.n_out ? a.n_rows : a.n_out;
    CLLM_CUDA(cudaMemcpyAsync(a.refs_out, a.refs, sizeof(int) * static_cast<size_t>(pg.n_pages), cudaMemcpyDeviceToDevice, stream));
    const ForkScratch s = fork_scratch(a.workspace, rows);
    fork_plan_kernel<<<1, kPlanThreads, 0, stream>>>(pg, a, s);
    CLLM_CUDA(cudaGetLastError());
    if (rows == 0) return;
    fork_move_kernel<<<dim3(rows, pg.n_layers < 64 ? pg.n_layers : 64), kMoveThreads, 0, stream>>>(pg, a, s);
    CLLM_CUDA(cudaGetLastError());
}

void launch_paged_compact(const cudallm_pages& pg, const cudallm_compact_args& a, cudaStream_t stream) {
    const CompactScratch s = compact_scratch(a.workspace, pg.n_pages);
    compact_plan_kernel<<<1, kPlanThreads, 0, stream>>>(pg, a, s);
    CLLM_CUDA(cudaGetLastError());
    compact_move_kernel<<<8 * 148, kMoveThreads, 0, stream>>>(pg, a, s);
    CLLM_CUDA(cudaGetLastError());
}

}  // namespace cudallm
