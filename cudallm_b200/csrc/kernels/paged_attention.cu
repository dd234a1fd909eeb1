// Attention of one new token per sequence over a paged key-value cache.
//
//   out[b][h] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q.k_t,  m = max_t s_t,
//   lse[b][h] = m + ln sum_t exp(s_t - m)
//
// What bounds it: a key and a value are read (2 tokens kv_heads head_dim 2 B) for 4 flops per query head of their group and element, so HBM
// does for groups of up to 16 heads. They are read once for groups of up to 16 heads of up to 128 dims and of up to 8 above; each
// further 16 (8) heads of a group are an item of their own, which reads them again (64 sequences of 4000 tokens, one key head x 128, 8 / 16 / 32 / 48
// heads: 32 / 43 / 65 / 88 us; x 256, 8 / 16: 75 / 131 us), since two groups of 8 at 256 dims do not fit the registers.
//
// Split. The positions of all (sequence, key head) items are cut into tiles of kTile tokens and counted through from
// first to last; CTA c takes tiles [c Q, (c + 1) Q), so ragged lengths spread evenly and one long sequence covers the
// GPU. A CTA's part of an item is a segment; the warps of the CTA take its tiles in turn, each with its own running (m,
// sum, out), which are joined in warp order. Segments that are not a whole item are left in the workspace, and a second
// kernel, whose blocks are already in place when the last of them is written, joins them in the order of the CTAs.
//
// Tiles. A warp copies its tiles with 16-byte asynchronous copies into a ring of its own (no block barrier between
// tiles), two or three deep; each lane looks up the page of one token, so pages of any size may end inside a tile. Rows are
// swizzled (chunk ^ row % 8) so that ldmatrix reads them without bank conflicts. Tokens without a page, outside the
// window or past the length are filled with zeros instead of being read, and masked by one bit each.
//
// Arithmetic. m16n8k16 matrix instructions with fp32 accumulators, 8 query heads a group: the second 8 rows of the
// 16-row operand are free, so they carry a second plane of it. Scores: q as one plane of the cache's type when it has
// that type, else as its rounding and the rounding of the rest (fp16: 22 bits; bf16: a third plane makes 24 bits for
// fp32 queries). Weights: p likewise in two planes (fp16: 22 bits of weights brought up to 2^15; bf16: 16 bits, a third plane
// makes 24 for fp32 results: see Shape). Each tile's product starts from zero and is added to the running fp32 output outside of the
// tensor core, whose additions truncate. The matrix work is below a fifth of the tensor pipe's time, so the legacy instruction is fast
// enough here, and its operands stay in registers between the two products; tcgen05 tiles of 64 or 128 rows would be padding for 8 heads.
//
// Measured (B200, graph replay): 32 heads on 8 key heads x 64, fp32 on bf16: 64 sequences of 512..767 tokens 25.6 us (3.3 TB/s), of 2048
// 51.4 us (5.2 TB/s); one of 32768 19.5 us (3.4 TB/s); 32 on 4 x 128, 37 ragged sequences of up to 8111 60.4 us (5.1 TB/s). About 9 us of
// each are the chain length - entry - page at the start, the last CTA and the join.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "common/check.h"
#include "kernels/kernels.h"
#include "kernels/launch.cuh"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"
#include "kernels/ptx.cuh"

namespace cudallm {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCtas = 512;
constexpr int kMaxRows = 2048;          // sequences of one launch (their tile counts are summed in shared memory)
constexpr int kSlotFloats = 16 * 2 + 16 * 128;  // a partial: m, sum and out of 16 heads x 128 dims or 8 x 256
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr size_t kEndingBytes = 32 * kMaxCtas;
constexpr int kUnit = 8;  // tiles of a CTA where there are few

// What a CTA's first segment is the last part of: the partials of CTAs c0 .. c0 + n - 1 make up `heads` rows of the output (n = 0: nothing).
struct __align__(16) Ending {
    int n, c0, heads, pad;
    long long row0;
};

struct Params {
    const void* q;
    const char* k;  // the layer's pages
    const char* v;
    void* out;
    float* lse;
    const int* tables;
    const int* lens;
    float* parts;  // [CTA][2] partials
    Ending* endings;  // [CTA]
    long long q_seq_stride, q_head_stride, table_stride, page_stride, head_stride, token_stride;  // elements
    float scale2;                                                                                  // scale * log2(e)
    float lse_unit;                                                                                // 2^-kLift
    int n_seq, n_heads, n_pages, page_size, table_width, head_dim, window;
    int group;      // query heads per key head
    int per_head;   // items per key head (groups of 8 HG query heads)
    int items;      // items per sequence
    FastDiv page_div;
    bool long_runs;      // page_size % 16 == 0: 16 tokens from a multiple of 16 on lie in one page
    bool dense;          // a head's tokens are HD dims apart and have as many
    long long row_step;  // bytes between the rows of one copy instruction and the next
};

template <typename KV>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                   uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same product with nothing to add to.
template <typename KV>
__device__ __forceinline__ void mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<KV, __nv_bfloat16>) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// 16 bytes global -> shared, or 16 zero bytes where `bytes` is 0.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// (a, b) rounded to the cache's type and packed, a in the low half; a and b keep what the rounding left.
template <typename KV>
__device__ __forceinline__ uint32_t take_plane(float& a, float& b) {
    uint32_t bits;
    if constexpr (std::is_same_v<KV, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        memcpy(&bits, &h, 4);
        a -= __uint_as_float(bits << 16);
        b -= __uint_as_float(bits & 0xffff0000u);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        memcpy(&bits, &h, 4);
        a -= __low2float(h);
        b -= __high2float(h);
    }
    return bits;
}

// 2^x to 22 bits; results below the normal range are 0.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// HD: head dims rounded up to 64, 128 or 256; HG: groups of 8 query heads of an item.
template <typename X, typename KV, int HD, int HG>
struct Shape {
    static constexpr bool kBf16 = std::is_same_v<KV, __nv_bfloat16>, kF32 = std::is_same_v<X, float>;
    static constexpr int kQPlanes = std::is_same_v<X, KV> ? 1 : kBf16 && kF32 ? 3 : 2;
    // For bf16 results over bf16 two planes do: of the outputs of 32768 tokens 2.6 in 1000 are not the bf16 number nearest to the exact one, 0.5 with a
    // third plane or with fp32 products, and a third costs up to 11 % (us with two and three: 64 x 512..767 23.4 and 24.1, 37 ragged 59.4 and 63.3,
    // groups of 16 x 128 100 and 111).
    static constexpr int kPPlanes = kBf16 && kF32 ? 3 : 2;
    static constexpr bool kScaleQ = !kBf16 && kQPlanes > 1;
    // Weights are exp2(x - max + kLift). fp16's grid ends at 2^-24: planes of weights up to 1 would lose all that is 17 nats below the maximum, and
    // digits from 10 nats on; with the largest at 2^15 what is lost is 2^-40 of it (output error under one token 17 nats above 32767 others:
    // 0.19 without, 5e-8 with the lift). Sums and outputs carry the factor until the one is divided by the other.
    static constexpr float kLift = kBf16 ? 0.f : 15.f;
    static constexpr int kTile = HD == 64 ? 32 : 16;  // tokens
    static constexpr int kStages = HD == 256 || HG == 2 ? 3 : 2;
    static constexpr int kCtas = HD == 256 ? 1 : HG == 2 ? 2 : 3;  // resident on an SM, by shared memory and registers
    static constexpr int kRowBytes = HD * 2;
    static constexpr int kPlaneBytes = kTile * kRowBytes;  // keys or values of a tile
    static constexpr int kStageBytes = 2 * kPlaneBytes;
    static constexpr int kHeads = 8 * HG;
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kQWords = HG * (HD / 16) * kQPlanes * 2 * 32;  // an item's query as matrix operands
    static constexpr int kJoin = (kWarps - 1) * (8 * 64 + 16) * 4;      // all but one warp's out, m and sum of 8 heads x 64 dims
    static constexpr int kFixed = kRing + kJoin + kQWords * 4 + kWarps * (kStages + 8 * HG) * 4 + 64;
};

struct Segment {
    int b, item;        // sequence, item of it
    int t0, t1, tiles;  // [t0, t1) of the item's tiles
    unsigned at;        // flat number of the item's first tile
    int len, first;     // the sequence's positions are [first, len)
    int first_tile;     // the tile of `first`
};

// One CTA's walk over its flat range of tiles.
struct Walk {
    const unsigned* before;  // [n_seq + 1] flat tiles of one item before sequence b (shared memory)
    int n_seq, items, pad;   // items per sequence; tiles of an item are rounded up to `pad` in the flat count
    unsigned f1;             // end of this CTA's range
};

template <int TILE>
__device__ __forceinline__ void tiles_of(const Params& p, int b, int& len, int& first, int& first_tile, int& tiles) {
    const int cap = p.table_width * p.page_size;  // below 2^31 (checked on the host)
    len = min(max(p.lens[b], 0), cap);
    first = p.window > 0 ? max(0, len - p.window) : 0;
    first_tile = first / TILE;
    tiles = len > 0 ? (len + TILE - 1) / TILE - first_tile : 0;
}

// The segment of sequence b, item `item` from flat tile f on.
template <int TILE>
__device__ __forceinline__ void open_segment(const Params& p, const Walk& w, Segment& s, int b, int item, unsigned f) {
    s.b = b;
    s.item = item;
    tiles_of<TILE>(p, b, s.len, s.first, s.first_tile, s.tiles);
    const unsigned padded = w.before[b + 1] - w.before[b];
    s.at = w.before[b] * w.items + item * padded;
    s.t0 = static_cast<int>(f - s.at);
    s.t1 = static_cast<int>(min(static_cast<unsigned>(s.tiles), w.f1 - s.at));
}

// The next segment; false when the range is done.
template <int TILE>
__device__ __forceinline__ bool next_segment(const Params& p, const Walk& w, Segment& s) {
    const unsigned padded = w.before[s.b + 1] - w.before[s.b];
    const unsigned f = s.at + padded;  // where the next item starts
    if (f >= w.f1) return false;
    int b = s.b, item = s.item + 1;
    if (item == w.items) {
        item = 0;
        do ++b;
        while (w.before[b + 1] == w.before[b]);
    }
    open_segment<TILE>(p, w, s, b, item, f);
    return true;
}

template <typename X, typename KV, int HD, int HG>
__global__ void __launch_bounds__(kThreads, Shape<X, KV, HD, HG>::kCtas) attend_kernel(const __grid_constant__ Params p) {
    using S = Shape<X, KV, HD, HG>;
    constexpr int kStages = S::kStages;
    constexpr int TILE = S::kTile, NT = TILE / 8, KS = HD / 16, JS = TILE / 16;
    extern __shared__ __align__(128) char smem[];
    char* ring = smem;
    float* join_o = reinterpret_cast<float*>(smem + S::kRing);                       // [kWarps - 1][16 floats a lane, 4 at a time]
    float* join_m = join_o + (kWarps - 1) * 512;                                     // [kWarps - 1][8]
    float* join_l = join_m + (kWarps - 1) * 8;                                       // [kWarps - 1][8]
    uint32_t* q_words = reinterpret_cast<uint32_t*>(join_l + (kWarps - 1) * 8);      // [hg][ks][plane][2][lane]
    unsigned* masks = q_words + S::kQWords;                                          // [warp][stage]
    float* q_tops = reinterpret_cast<float*>(masks + kWarps * kStages);              // [warp][head]
    unsigned* shared_word = reinterpret_cast<unsigned*>(q_tops + kWarps * 8 * HG);   // [16]
    unsigned* before = reinterpret_cast<unsigned*>(smem + S::kFixed);                // [n_seq + 1]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t4 = lane & 3, hd = p.head_dim;
    grid_dep_wait();
    if (threadIdx.x == 0) p.endings[blockIdx.x].n = 0;
    grid_dep_launch();  // the join's blocks may take the places that this kernel's leave

    // Tiles of one item before each sequence, as they are and in units of kUnit; empty rows are answered here.
    unsigned total = 0, total_pad = 0;
    for (int b0 = 0; b0 < p.n_seq; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int len, first, first_tile, tiles = 0;
        if (b < p.n_seq) tiles_of<TILE>(p, b, len, first, first_tile, tiles);
        unsigned s = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned t = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += t;
        }
        const unsigned pads = __reduce_add_sync(0xffffffffu, (tiles + kUnit - 1) / kUnit);
        if (lane == 31) {
            shared_word[warp] = s;
            shared_word[kWarps + warp] = pads;
        }
        __syncthreads();
        unsigned base = total;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) base += shared_word[w];
            total += shared_word[w];
            total_pad += shared_word[kWarps + w];
        }
        if (b < p.n_seq) before[b] = base + s - tiles;
        __syncthreads();
    }
    if (threadIdx.x == 0) before[p.n_seq] = total;
    for (int b = blockIdx.x; b < p.n_seq; b += gridDim.x) {
        if (p.lens[b] > 0 && p.table_width > 0) continue;
        for (int i = threadIdx.x; i < p.n_heads * hd; i += kThreads) {
            static_cast<X*>(p.out)[static_cast<long long>(b) * p.n_heads * hd + i] = from_float<X>(0.f);
        }
        if (p.lse != nullptr) {
            for (int h = threadIdx.x; h < p.n_heads; h += kThreads) p.lse[static_cast<long long>(b) * p.n_heads + h] = -INFINITY;
        }
    }
    // Few tiles: an item's tiles are cut every kUnit. Otherwise every CTA takes an equal share.
    const bool few = total_pad * p.items <= gridDim.x;
    const unsigned share = few ? kUnit : (total * p.items + gridDim.x - 1) / gridDim.x;
    const unsigned all = few ? total_pad * kUnit * p.items : total * p.items;
    __syncthreads();
    if (few) {  // the same sums of rounded tile counts
        unsigned run = 0;
        for (int b0 = 0; b0 < p.n_seq; b0 += kThreads) {
            const int b = b0 + threadIdx.x;
            const unsigned mine = b < p.n_seq ? (before[b + 1] - before[b] + kUnit - 1) / kUnit * kUnit : 0;
            unsigned s = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned t = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += t;
            }
            if (lane == 31) shared_word[warp] = s;
            __syncthreads();
            unsigned base = run;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) base += shared_word[w];
                run += shared_word[w];
            }
            if (b < p.n_seq) before[b] = base + s - mine;
            __syncthreads();
        }
        if (threadIdx.x == 0) before[p.n_seq] = run;
        __syncthreads();
    }
    const unsigned f0 = min(all, blockIdx.x * share);
    Walk walk{before, p.n_seq, p.items, few ? kUnit : 1, min(all, f0 + share)};
    if (f0 >= walk.f1) return;

    // The first segment: the last sequence that starts at or before f0.
    Segment seg;
    {
        int lo = 0, hi = p.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (before[mid] * p.items <= f0) lo = mid;
            else hi = mid;
        }
        const unsigned padded = before[lo + 1] - before[lo];
        open_segment<TILE>(p, walk, seg, lo, static_cast<int>((f0 - before[lo] * p.items) / padded), f0);
    }

    // ---- the query, as operands in shared memory: warp w turns k-steps w, w + kWarps, ... of the next segment ----
    constexpr int QS = (KS + kWarps - 1) / kWarps;
    float raw[HG][QS][4];
    auto fetch_q = [&](const Segment& s) {
        const int kvh = s.item / p.per_head, h_first = (s.item % p.per_head) * S::kHeads;
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
            const int h = h_first + hg * 8 + g;
            const X* q = static_cast<const X*>(p.q) + s.b * p.q_seq_stride + (kvh * p.group + h) * p.q_head_stride;
#pragma unroll
            for (int i = 0; i < QS; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = (i * kWarps + warp) * 16 + 2 * t4 + (e & 1) + (e >> 1) * 8;
                    raw[hg][i][e] = h < p.group && d < hd ? as_float(q[d]) : 0.f;
                }
            }
        }
    };
    auto put_tops = [&] {  // largest |q| of this warp's dims
        if constexpr (S::kScaleQ) {
#pragma unroll
            for (int hg = 0; hg < HG; ++hg) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < QS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(raw[hg][i][e]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (t4 == 0) q_tops[warp * 8 * HG + hg * 8 + g] = top;
            }
        }
    };
    float q_scale[HG];
    auto put_q = [&] {  // after a barrier behind put_tops
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
            float shrink = 1.f;
            q_scale[hg] = p.scale2;
            if constexpr (S::kScaleQ) {
                // fp16 planes: the head is brought to 2^14 <= max|q| < 2^15 by a power of two, which the scale gives back; what fp16's grid
                // of 2^-24 takes from the smallest dims is then below 2^-39 of the largest one.
                float top = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, q_tops[w * 8 * HG + hg * 8 + g]);
                const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 15), 254) - 127 - 14;  // -126 .. 113: both powers are normal
                shrink = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                q_scale[hg] *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            }
#pragma unroll
            for (int i = 0; i < QS; ++i) {
                const int ks = i * kWarps + warp;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = raw[hg][i][e] * shrink;
#pragma unroll
                for (int pl = 0; pl < S::kQPlanes; ++pl) {
                    uint32_t* w = q_words + ((hg * KS + ks) * S::kQPlanes + pl) * 64 + lane;
                    w[0] = take_plane<KV>(v[0], v[1]);
                    w[32] = take_plane<KV>(v[2], v[3]);
                }
            }
        }
    };
    static_assert(KS % kWarps == 0, "every warp turns as many k-steps");
    fetch_q(seg);  // on its way while the first tiles are looked up

    // ---- the warp's stream of tiles ----
    Segment ls = seg;                  // of the next tile to load
    int lt = ls.t0 + warp;             // that tile
    bool more = true;                  // there is one
    int l_slot = 0, l_token = 0;       // this lane's token of it, and its slot in its page
    int l_page = -1;
    bool l_valid = false;
    const uint32_t my_ring = smem_addr(ring) + warp * (kStages * S::kStageBytes);
    // One copy instruction of the warp covers kRowsAtOnce rows; this lane takes 16-byte chunk lane % kChunks of row lane / kChunks.
    constexpr int kChunks = HD / 8, kRowsAtOnce = 32 / kChunks;
    const int inside = lane % kChunks * 8 < hd ? 16 : 0;
    const uint32_t my_dst = lane / kChunks * S::kRowBytes + ((lane % kChunks ^ lane / kChunks) << 4);
    const long long my_src = inside ? lane / kChunks * p.token_stride * 2 + lane % kChunks * 16 : 0;
    auto look_up = [&] {  // moves to the next tile of this warp and reads its lane's page number
        while (more && lt >= ls.t1) {
            more = next_segment<TILE>(p, walk, ls);
            lt = ls.t0 + warp;
        }
        if (!more) return;
        l_token = (ls.first_tile + lt) * TILE + (lane % TILE);
        l_valid = l_token >= ls.first && l_token < ls.len;
        const int entry = div_by(l_token, p.page_div);
        l_slot = l_token - entry * p.page_size;
        l_page = l_valid ? p.tables[ls.b * p.table_stride + entry] : -1;
    };
    auto load_tile = [&](int stage) {
        if (more) {
            const bool valid = l_page >= 0 && l_page < p.n_pages;
            const long long off = valid ? (l_page * p.page_stride + l_slot * p.token_stride + ls.item / p.per_head * p.head_stride) * 2 : -1;
            const unsigned mask = __ballot_sync(0xffffffffu, valid);
            if (lane == 0) masks[warp * kStages + stage] = mask;
            const uint32_t dst = my_ring + stage * S::kStageBytes + my_dst;
            if (mask == 0xffffffffu && p.long_runs) {  // 16 tokens at a time lie in one page, evenly spaced
#pragma unroll
                for (int r16 = 0; r16 < TILE; r16 += 16) {
                    const long long o = __shfl_sync(0xffffffffu, off, r16) + my_src;
                    const char *k = p.k + o, *v = p.v + o;
#pragma unroll
                    for (int r0 = r16; r0 < r16 + 16; r0 += kRowsAtOnce) {
                        const uint32_t d = (dst ^ ((r0 & 7) << 4)) + r0 * S::kRowBytes;
                        if (p.dense) {
                            copy16(d, k + (r0 - r16) * S::kRowBytes, 16);
                            copy16(d + S::kPlaneBytes, v + (r0 - r16) * S::kRowBytes, 16);
                        } else {
                            copy16(d, k, inside);
                            copy16(d + S::kPlaneBytes, v, inside);
                            k += p.row_step;
                            v += p.row_step;
                        }
                    }
                }
            } else {
#pragma unroll
                for (int r0 = 0; r0 < TILE; r0 += kRowsAtOnce) {
                    const long long o = __shfl_sync(0xffffffffu, off, r0 + lane / kChunks);
                    const int bytes = o >= 0 ? inside : 0;
                    const long long at = bytes ? o + lane % kChunks * 16 : 0;
                    const uint32_t d = (dst ^ ((r0 & 7) << 4)) + r0 * S::kRowBytes;
                    copy16(d, p.k + at, bytes);
                    copy16(d + S::kPlaneBytes, p.v + at, bytes);
                }
            }
            lt += kWarps;
        }
        copy_commit();
    };
    look_up();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        load_tile(s);
        look_up();
    }

    put_tops();
    __syncthreads();
    put_q();
    __syncthreads();

    int stage = 0, joiner = 0;
    for (;;) {
        // ---- one segment ----
        const int kvh = seg.item / p.per_head, h_first = (seg.item % p.per_head) * S::kHeads;
        const int heads = min(S::kHeads, p.group - h_first);  // query heads of this item
        const long long row0 = static_cast<long long>(seg.b) * p.n_heads + kvh * p.group + h_first;

        uint32_t qf[HG][KS][S::kQPlanes][2];  // planes of q: dims 16 ks + 2 t4 + {0, 1} and + 8
#pragma unroll
        for (int i = 0; i < HG * KS * S::kQPlanes * 2; ++i) (&qf[0][0][0][0])[i] = q_words[i * 32 + lane];
        Segment following = seg;
        const bool goes_on = next_segment<TILE>(p, walk, following);
        if (goes_on) fetch_q(following);

        float o[HG][HD / 8][2], m[HG], l[HG];
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
            m[hg] = -INFINITY;
            l[hg] = 0.f;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) o[hg][n][0] = o[hg][n][1] = 0.f;
        }

        for (int t = seg.t0 + warp; t < seg.t1; t += kWarps) {
            load_tile(stage == 0 ? kStages - 1 : stage - 1);
            look_up();
            copy_wait<kStages - 1>();
            __syncwarp();
            const uint32_t kb = my_ring + stage * S::kStageBytes, vb = kb + S::kPlaneBytes;
            const unsigned mask = masks[warp * kStages + stage];

            // scores
            float s[HG][NT][4];
            const int k_row = (lane >> 4) * 8 + (lane & 7), k_chunk = (lane >> 3) & 1;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks * 16 >= hd) break;
#pragma unroll
                for (int n2 = 0; n2 < NT / 2; ++n2) {
                    const int r = n2 * 16 + k_row;
                    uint32_t b[4];
                    ldmatrix4(b, kb + r * S::kRowBytes + (((2 * ks + k_chunk) ^ (r & 7)) << 4));
#pragma unroll
                    for (int hg = 0; hg < HG; ++hg) {
                        const uint32_t lo0 = S::kQPlanes > 1 ? qf[hg][ks][S::kQPlanes > 1][0] : 0u;
                        const uint32_t lo1 = S::kQPlanes > 1 ? qf[hg][ks][S::kQPlanes > 1][1] : 0u;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float(&c)[4] = s[hg][2 * n2 + i];
                            if (ks == 0) mma_first<KV>(c, qf[hg][ks][0][0], lo0, qf[hg][ks][0][1], lo1, b[2 * i], b[2 * i + 1]);
                            else mma<KV>(c, qf[hg][ks][0][0], lo0, qf[hg][ks][0][1], lo1, b[2 * i], b[2 * i + 1]);
                        }
                        if constexpr (S::kQPlanes > 2) {
                            mma<KV>(s[hg][2 * n2], qf[hg][ks][2][0], 0u, qf[hg][ks][2][1], 0u, b[0], b[1]);
                            mma<KV>(s[hg][2 * n2 + 1], qf[hg][ks][2][0], 0u, qf[hg][ks][2][1], 0u, b[2], b[3]);
                        }
                    }
                }
            }

            // weights: this thread has tokens 8 n + 2 t4 + {0, 1} of head g
            constexpr unsigned kAll = TILE == 32 ? 0xffffffffu : 0xffffu;
            const bool whole = (mask & kAll) == kAll;
            uint32_t pf[HG][JS][S::kPPlanes][2];
            float fade[HG];
#pragma unroll
            for (int hg = 0; hg < HG; ++hg) {
                float x[NT][2], top = -INFINITY;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[n][e] = (s[hg][n][e] + s[hg][n][2 + e]) * q_scale[hg];
                        if (!whole && !((mask >> (8 * n + 2 * t4 + e)) & 1u)) x[n][e] = -INFINITY;
                        top = fmaxf(top, x[n][e]);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m_new = fmaxf(m[hg], top), ref = m_new == -INFINITY ? 0.f : m_new;
                fade[hg] = exp2_fast(m[hg] - ref);
                m[hg] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[n][e] -= ref;  // exact near the maximum, which ref - kLift would not be
                        if constexpr (S::kLift != 0.f) x[n][e] += S::kLift;
                        x[n][e] = exp2_fast(x[n][e]);
                        sum += x[n][e];
                    }
                }
                l[hg] = l[hg] * fade[hg] + sum;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int pl = 0; pl < S::kPPlanes; ++pl) pf[hg][n / 2][pl][n & 1] = take_plane<KV>(x[n][0], x[n][1]);
            }

            // out = out * fade + weights x values
            const int v_row = lane & 15, v_chunk = lane >> 4;
#pragma unroll
            for (int n2 = 0; n2 < HD / 16; ++n2) {
                if (n2 * 16 >= hd) break;
                float acc[HG][2][4];
#pragma unroll
                for (int j = 0; j < JS; ++j) {
                    const int r = j * 16 + v_row;
                    uint32_t b[4];
                    ldmatrix4_trans(b, vb + r * S::kRowBytes + (((2 * n2 + v_chunk) ^ (r & 7)) << 4));
#pragma unroll
                    for (int hg = 0; hg < HG; ++hg) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (j == 0) mma_first<KV>(acc[hg][i], pf[hg][j][0][0], pf[hg][j][1][0], pf[hg][j][0][1], pf[hg][j][1][1], b[2 * i], b[2 * i + 1]);
                            else mma<KV>(acc[hg][i], pf[hg][j][0][0], pf[hg][j][1][0], pf[hg][j][0][1], pf[hg][j][1][1], b[2 * i], b[2 * i + 1]);
                            if constexpr (S::kPPlanes > 2) {
                                mma<KV>(acc[hg][i], pf[hg][j][S::kPPlanes - 1][0], 0u, pf[hg][j][S::kPPlanes - 1][1], 0u, b[2 * i], b[2 * i + 1]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int hg = 0; hg < HG; ++hg)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            o[hg][2 * n2 + i][e] = fmaf(o[hg][2 * n2 + i][e], fade[hg], acc[hg][i][e] + acc[hg][i][2 + e]);
            }
            __syncwarp();
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }

        // ---- join the warps: one of them, in turn, adds the others' 8 heads x 64 dims to its own ----
        const bool whole_item = seg.t0 == 0 && seg.t1 == seg.tiles;
        float* part = p.parts + (static_cast<size_t>(blockIdx.x) * 2 + (seg.t0 == 0)) * kSlotFloats;
        const int others = (warp - joiner - 1) & (kWarps - 1);  // place of this warp's values; the joiner has none
        if (goes_on) put_tops();
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
            l[hg] += __shfl_xor_sync(0xffffffffu, l[hg], 1);
            l[hg] += __shfl_xor_sync(0xffffffffu, l[hg], 2);
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += 64) {
                __syncthreads();  // the values before have been read, and every warp has this segment's query
                if (hg + d0 == 0 && goes_on) put_q();
                if (warp != joiner) {
                    if (t4 == 0) {
                        join_m[others * 8 + g] = m[hg];
                        join_l[others * 8 + g] = l[hg];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        reinterpret_cast<float4*>(join_o)[(others * 4 + i) * 32 + lane] =
                            make_float4(o[hg][d0 / 8 + 2 * i][0], o[hg][d0 / 8 + 2 * i][1], o[hg][d0 / 8 + 2 * i + 1][0], o[hg][d0 / 8 + 2 * i + 1][1]);
                    }
                }
                __syncthreads();
                if (warp == joiner) {
                    float mm = m[hg], f[kWarps];
#pragma unroll
                    for (int w = 0; w < kWarps - 1; ++w) mm = fmaxf(mm, join_m[w * 8 + g]);
                    const float ref = mm == -INFINITY ? 0.f : mm;
                    f[kWarps - 1] = exp2_fast(m[hg] - ref);
                    float ll = l[hg] * f[kWarps - 1];
#pragma unroll
                    for (int w = 0; w < kWarps - 1; ++w) {
                        f[w] = exp2_fast(join_m[w * 8 + g] - ref);
                        ll = fmaf(f[w], join_l[w * 8 + g], ll);
                    }
                    const int row = hg * 8 + g;
                    const float norm = !whole_item ? 1.f : ll == 0.f ? 0.f : 1.f / ll;  // scores that are not numbers make ll one, too
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = o[hg][d0 / 8 + 2 * i + (e >> 1)][e & 1] * f[kWarps - 1];
#pragma unroll
                        for (int w = 0; w < kWarps - 1; ++w) {
                            const float4 x = reinterpret_cast<const float4*>(join_o)[(w * 4 + i) * 32 + lane];
                            v[0] = fmaf(f[w], x.x, v[0]);
                            v[1] = fmaf(f[w], x.y, v[1]);
                            v[2] = fmaf(f[w], x.z, v[2]);
                            v[3] = fmaf(f[w], x.w, v[3]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int d = d0 + (2 * i + (e >> 1)) * 8 + 2 * t4 + (e & 1);
                            if (row >= heads) continue;
                            if (!whole_item) part[32 + row * HD + d] = v[e];
                            else if (d < hd) static_cast<X*>(p.out)[(row0 + row) * hd + d] = from_float<X>(v[e] * norm);
                        }
                    }
                    if (d0 == 0 && t4 == 0 && row < heads) {
                        if (!whole_item) {
                            part[row] = mm;
                            part[16 + row] = ll;
                        } else if (p.lse != nullptr) {
                            p.lse[row0 + row] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll * p.lse_unit));
                        }
                    }
                }
            }
        }
        if (seg.t0 != 0 && seg.t1 == seg.tiles && threadIdx.x == 0) {  // the item's CTAs are those of its flat tiles
            const int c0 = static_cast<int>(seg.at / share);
            p.endings[blockIdx.x] = {static_cast<int>(blockIdx.x) + 1 - c0, c0, heads, 0, row0};
        }
        joiner = (joiner + 1) & (kWarps - 1);
        if (!goes_on) break;
        seg = following;
    }
    copy_wait<0>();
}

// Joins the partials of items that were cut, in the order of their CTAs: block (c, h) those of head h of the item that ends in CTA
// c's first segment. The block's WARPS warps take the partials in turn; the loads of each are independent of each other.
template <typename X, int HD, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) join_kernel(const __grid_constant__ Params p) {
    constexpr int V = HD / 32;  // dims of a lane
    __shared__ float warp_m[WARPS], warp_l[WARPS], warp_o[WARPS][HD];
    grid_dep_wait();
    const int4 head = __ldcg(reinterpret_cast<const int4*>(p.endings + blockIdx.x));
    const int parts = head.x, c0 = head.y, h = blockIdx.y;
    if (parts == 0 || h >= head.z) return;
    const long long row = __ldcg(&p.endings[blockIdx.x].row0) + h;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
    auto part = [&](int c) { return p.parts + (static_cast<size_t>(c0 + c) * 2 + (c == 0)) * kSlotFloats; };
    constexpr int kAtOnce = 8;
    for (int from = warp; from < parts; from += kAtOnce * WARPS) {
        float pm[kAtOnce], pl[kAtOnce], po[kAtOnce][V];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int c = from + k * WARPS;
            pm[k] = -INFINITY;
            if (c >= parts) continue;
            const float* src = part(c);
            pm[k] = __ldcg(src + h);
            pl[k] = __ldcg(src + 16 + h);
            src += 32 + h * HD + lane * V;
            if constexpr (V == 2) {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
                po[k][0] = v.x, po[k][1] = v.y;
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(src + i));
                    po[k][i] = v.x, po[k][i + 1] = v.y, po[k][i + 2] = v.z, po[k][i + 3] = v.w;
                }
            }
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) top = fmaxf(top, pm[k]);
        const float ref = top == -INFINITY ? 0.f : top, old = exp2_fast(m - ref);
        m = top;
        l *= old;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] *= old;
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (from + k * WARPS >= parts) break;
            const float f = exp2_fast(pm[k] - ref);
            l = fmaf(f, pl[k], l);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(f, po[k][i], o[i]);
        }
    }
    if (lane == 0) {
        warp_m[warp] = m;
        warp_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) warp_o[warp][lane * V + i] = o[i];
    __syncthreads();
    for (int d = threadIdx.x; d < p.head_dim; d += 32 * WARPS) {
        float mm = -INFINITY, ll = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, warp_m[w]);
        const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2_fast(warp_m[w] - ref);
            ll = fmaf(f, warp_l[w], ll);
            v = fmaf(f, warp_o[w][d], v);
        }
        static_cast<X*>(p.out)[row * p.head_dim + d] = from_float<X>(ll == 0.f ? 0.f : v / ll);
        if (d == 0 && p.lse != nullptr) p.lse[row] = ll == 0.f ? -INFINITY : fmaf(mm, kLn2, logf(ll * p.lse_unit));
    }
}

template <typename X, typename KV, int HD, int HG>
void launch_shape(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream) {
    using S = Shape<X, KV, HD, HG>;
    Params p;
    p.q = a.q;
    p.k = static_cast<const char*>(pg.k) + 2 * a.layer * pg.layer_stride;
    p.v = static_cast<const char*>(pg.v) + 2 * a.layer * pg.layer_stride;
    p.endings = static_cast<Ending*>(a.workspace);
    p.parts = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kEndingBytes);
    p.q_seq_stride = a.q_seq_stride;
    p.q_head_stride = a.q_head_stride;
    p.table_stride = a.table_stride;
    p.page_stride = pg.page_stride;
    p.head_stride = pg.head_stride;
    p.token_stride = pg.token_stride;
    p.scale2 = a.scale * kLog2e;
    p.lse_unit = std::exp2(-S::kLift);
    p.n_heads = a.n_heads;
    p.n_pages = pg.n_pages;
    p.page_size = pg.page_size;
    p.table_width = a.table_width;
    p.head_dim = pg.head_dim;
    p.window = a.window;
    p.group = a.n_heads / pg.n_kv_heads;
    p.per_head = (p.group + S::kHeads - 1) / S::kHeads;
    p.items = p.per_head * pg.n_kv_heads;
    p.page_div = fast_div(pg.page_size);
    p.long_runs = pg.page_size % 16 == 0;
    p.dense = pg.token_stride == HD && pg.head_dim == HD;
    p.row_step = pg.token_stride * 2 * (32 / (HD / 8));
    auto kernel = attend_kernel<X, KV, HD, HG>;
    static std::atomic<uint64_t> allowed{0};  // devices on which this kernel may use its shared memory
    allow_shared(kernel, S::kFixed + 4 * (kMaxRows + 1), allowed);
    const long long cap = static_cast<long long>(a.table_width) * pg.page_size;
    const long long row_tiles = std::max(1LL, (cap + S::kTile - 1) / S::kTile * p.items);  // most tiles of a sequence
    CLLM_REQUIRE(row_tiles <= (1LL << 31), "cudallm_paged_attend: the tables are too wide");
    const int at_once = static_cast<int>(std::min<long long>(kMaxRows, std::max(1LL, (1LL << 31) / row_tiles)));
    for (int b0 = 0; b0 < a.n_seq; b0 += at_once) {
        p.n_seq = std::min(at_once, a.n_seq - b0);
        p.lens = a.lens + b0;
        p.tables = a.tables + b0 * a.table_stride;
        p.q = static_cast<const X*>(a.q) + b0 * a.q_seq_stride;
        p.out = static_cast<X*>(a.out) + static_cast<long long>(b0) * a.n_heads * pg.head_dim;
        p.lse = a.lse != nullptr ? a.lse + static_cast<long long>(b0) * a.n_heads : nullptr;
        const size_t smem = S::kFixed + 4 * (static_cast<size_t>(p.n_seq) + 1);
        const long long most = std::max<long long>(1, (row_tiles + kUnit - 1) / kUnit * p.n_seq + p.items * static_cast<long long>(p.n_seq));
        const int grid = static_cast<int>(std::min<long long>(std::min(kMaxCtas, num_sms() * std::min(S::kCtas, static_cast<int>(228 * 1024 / (smem + 1024)))), most));
        launch_kernel(kernel, dim3(grid), dim3(kThreads), smem, stream, true, p);
        // Items of up to kUnit tiles are cut only where equal shares cut them, which takes more tiles than there are CTAs x kUnit.
        const bool can_cut = (cap + S::kTile - 1) / S::kTile > kUnit || static_cast<long long>(p.n_seq) * p.items > grid;
        if (!can_cut) continue;
        // Up to 16 partials an item: blocks of 2 warps, of which an SM takes all that it gets at once (37 ragged sequences: 63.8 us with 8
        // warps, 60.6 with 2); more: 8 warps (one of 32768 tokens, 55 partials: 19.5 us with 8, 20.6 with 2).
        const bool few = grid <= 16LL * p.n_seq * p.items;
        launch_kernel(few ? join_kernel<X, HD, 2> : join_kernel<X, HD, 8>, dim3(grid, std::min(p.group, S::kHeads)), dim3(few ? 64 : 256), 0, stream, true, p);
    }
}

template <typename X, typename KV>
void launch_types(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream) {
    const bool two = a.n_heads / pg.n_kv_heads > 8;  // both groups of 8 heads share one read of the keys
    if (pg.head_dim <= 64) {
        two ? launch_shape<X, KV, 64, 2>(pg, a, stream) : launch_shape<X, KV, 64, 1>(pg, a, stream);
    } else if (pg.head_dim <= 128) {
        two ? launch_shape<X, KV, 128, 2>(pg, a, stream) : launch_shape<X, KV, 128, 1>(pg, a, stream);
    } else {
        launch_shape<X, KV, 256, 1>(pg, a, stream);  // a second group would not fit the registers
    }
}

}  // namespace

size_t attend_workspace_bytes() { return kEndingBytes + sizeof(float) * kSlotFloats * 2 * kMaxCtas; }

void launch_paged_attend(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream) {
    if (a.n_seq == 0) return;
    const bool bf16 = pg.kv_dtype == CUDALLM_KV_BF16;
    switch (a.x_dtype) {
        case CUDALLM_X_FP32: bf16 ? launch_types<float, __nv_bfloat16>(pg, a, stream) : launch_types<float, __half>(pg, a, stream); break;
        case CUDALLM_X_FP16: bf16 ? launch_types<__half, __nv_bfloat16>(pg, a, stream) : launch_types<__half, __half>(pg, a, stream); break;
        default: bf16 ? launch_types<__nv_bfloat16, __nv_bfloat16>(pg, a, stream) : launch_types<__nv_bfloat16, __half>(pg, a, stream); break;
    }
}

}  // namespace cudallm
