// Beam search's selection: the best continuations of each group of beams over beams and vocabulary.
//
//   candidate(w, t) = score[w] + (x[t] - lse(x)),  x = row w's logits,  lse(x) = m + ln sum_t exp(x[t] - m)
//
// Within a row candidates rank as (logit, then lower token), so the `keep` best by logit of each chunk of a row are the
// only ones that can be among the group's.
//
// chunk stage: one block per 8192 logits, which stay in registers (one read of the logits). It leaves their maximum, their sum of exponentials and the
//   sorted keys of their `keep` best. The maxima of 512 pieces give a lower bound of the keep-th best; the few logits above it are ranked by
//   counting. Where more than 256 are above it (ties, a masked vocabulary) the keep-th key itself is searched bit by bit over value and token.
// group stage: joins the rows' sums and ranks the lists' candidates in the same way. Up to 512 chunks the last block of a
//   group to finish does it; with more, a block for each group in a second launch, in place when the chunks are done (us a call with one
//   launch and with two, at 128256 tokens: 4 rows 12.8 and 15.4, 32 rows 13.0 and 15.3, 64 rows 17.4 and 15.3).
//
// Latency bounds it, not the read: a chunk is a chain of load, maximum, bound, list and rank. 64 rows x 128256 fp32 (8 x 8 beams, keep 8; ncu, cold
// caches): chunks 17 us at 1.9 TB/s, 1024 blocks in 1.7 waves of four an SM (64 registers), 40 % of the issue slots, a third of a warp's time
// waiting for its logits; groups 10 us on 8 blocks, of which half waits at barriers for keys from L2.
//
// Measured (B200, graph replay, other logits each time): 64 rows x 128256, fp32, 20.5 us (keep 8), 22.3 (16), 31.6 (64); bf16 the same; with 40 rows
// finished, keep 16, 15.6 us; 16 rows 12.3 us; 4 rows 12.0 us; 64 rows x 32000 12.4 us.
#include <cmath>

#include "common/check.h"
#include "kernels/launch.cuh"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"
#include "kernels/ptx.cuh"
#include "kernels/sampling.cuh"

namespace cudallm {

namespace {

constexpr int kThreads = 256;
constexpr int kEach = 32;  // logits of a thread
constexpr int kChunk = kThreads * kEach;
constexpr int kList = 256;  // candidates above the bound that are ranked by counting
constexpr int kGroupThreads = 512;
constexpr int kGroupList = 512;
constexpr int kOneLaunch = 512;  // chunks of a call with a single launch
constexpr unsigned kAll = 0xffffffffu;

// Rank bits of a logit: not a number counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t logit_bits(float x) { return float_order_key(isnan(x) ? -INFINITY : x + 0.f); }

// The r-th largest of the values a, b of a warp's lanes (0 = none, or fewer than r of them), or a lower bound of it: its first 16 bits where r
// is above 8.
__device__ __forceinline__ uint32_t warp_bound(uint32_t a, uint32_t b, int r) {
    uint32_t bound = 0;
    if (r <= 8) {  // one largest after the other
#pragma unroll 1
        for (int i = 0; i < r; ++i) {
            const uint32_t mine = max(a, b);
            bound = __reduce_max_sync(kAll, mine);
            const int owner = __ffs(__ballot_sync(kAll, mine == bound)) - 1;
            if (static_cast<int>(threadIdx.x & 31) == owner) {
                if (a == bound) a = 0;
                else b = 0;
            }
        }
        return bound;
    }
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t test = bound | 1u << bit;
        if (__popc(__ballot_sync(kAll, a >= test)) + __popc(__ballot_sync(kAll, b >= test)) >= r) bound = test;
    }
    return bound;
}

// A lower bound of the keep-th largest of a block's values, of which every thread brings two samples: where each of `warps` warps has r =
// keep / warps samples from its bound on, there are `keep` from the smallest of those bounds on. `sm` has a place for each warp;
// a barrier inside. At least 1, as values are.
template <int THREADS>
__device__ __forceinline__ uint32_t block_bound(uint32_t a, uint32_t b, int keep, int warps, uint32_t* sm) {
    warps = max(warps, 1);
    const uint32_t mine = warp_bound(a, b, (keep + warps - 1) / warps);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = static_cast<int>(threadIdx.x >> 5) < warps ? mine : kAll;
    __syncthreads();
    uint32_t bound = kAll;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) bound = min(bound, sm[w]);
    return max(bound, 1u);
}

// The first 16 bits of the keep-th largest of 512 values in shared memory (0 = none, or fewer than keep): a lower bound of it. One warp.
__device__ __forceinline__ uint32_t bound_of(const uint32_t* samples, int keep) {
    uint32_t v[16], bound = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = samples[(threadIdx.x & 31) + 32 * i];
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t test = bound | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) n += v[i] >= test;
        if (__reduce_add_sync(kAll, n) >= keep) bound = test;
    }
    return bound;
}

// Sum over the block of one count per thread; barriers on both sides.
template <int THREADS>
__device__ __forceinline__ int block_sum(int v, int* sm) {
    v = __reduce_add_sync(kAll, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) s += sm[w];
    return s;
}

struct Best {
    uint32_t bits;  // of the candidate
    int row;        // beam in the group
    uint64_t key;   // logit and token
};
__device__ __forceinline__ bool better(const Best& a, const Best& b) {
    return a.bits != b.bits ? a.bits > b.bits : a.row != b.row ? a.row < b.row : a.key > b.key;
}

constexpr int kSamples = 512;  // what bound_of takes
template <int THREADS>
struct GroupRoom {
    float lse[kMaxBeams], score[kMaxBeams];
    Best list[kGroupList], best[THREADS / 32];
    uint32_t samples[kSamples], bound;
    int count;
};

// The best of group g, from its rows' lists and sums, by all threads of a block.
template <int THREADS>
__device__ void select_group(const cudallm_beam_args& a, const uint64_t* lists, const float2* stats, int chunks, int g, GroupRoom<THREADS>& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sm.count = 0;
    for (int w = warp; w < a.beams; w += THREADS / 32) {
        const float2* st = stats + (static_cast<size_t>(g) * a.beams + w) * chunks;
        float m = -INFINITY, s = 0.f;
        for (int c = lane; c < chunks; c += 32) m = fmaxf(m, __ldcg(st + c).x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
        for (int c = lane; c < chunks; c += 32) {
            const float2 v = __ldcg(st + c);
            s += v.y * expf(v.x == -INFINITY ? (m == -INFINITY ? 0.f : -INFINITY) : v.x - m);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        if (lane == 0) {
            sm.lse[w] = m + logf(s);
            sm.score[w] = a.scores[static_cast<size_t>(g) * a.beams + w];
        }
    }
    __syncthreads();
    const int n_lists = a.beams * chunks;
    const uint64_t* keys = lists + static_cast<size_t>(g) * n_lists * a.keep;
    auto read = [&](int l, int k) {  // candidate k of list l
        Best b;
        b.key = __ldcg(keys + static_cast<size_t>(l) * a.keep + k);
        b.row = l / chunks;
        const float v = sm.score[b.row] + (candidate_value(b.key) - sm.lse[b.row]);
        b.bits = b.key == 0 ? 0u : float_order_key(isnan(v) ? -INFINITY : v + 0.f);
        return b;
    };
    // 512 walkers: with fewer lists, several take a list's candidates in turn. The first candidates of each are the samples.
    const int across = min(n_lists, kSamples), step = kSamples / across;
    for (int v = threadIdx.x; v < kSamples; v += THREADS) {
        const int k0 = v / across;
        uint32_t top = 0;
        if (k0 < step && k0 < a.keep) {
            for (int l = v % across; l < n_lists; l += across) top = max(top, read(l, k0).bits);
        }
        sm.samples[v] = top;
    }
    __syncthreads();
    if (warp == 0) {  // rows differ by their scores, so that no part of the lists says much about the others
        const uint32_t b = bound_of(sm.samples, a.keep);
        if (lane == 0) sm.bound = max(b, 1u);
    }
    __syncthreads();
    const uint32_t bound = sm.bound;
    auto each = [&](auto&& take) {  // every candidate from the bound on
        for (int v = threadIdx.x; v < kSamples; v += THREADS) {
            const int k0 = v / across;
            if (k0 >= step) break;
            for (int l = v % across; l < n_lists; l += across) {
                for (int k = k0; k < a.keep; k += step) {
                    const Best b = read(l, k);
                    if (b.bits < bound) break;  // lists descend
                    take(b);
                }
            }
        }
    };
    each([&](const Best& b) {
        const int p = atomicAdd(&sm.count, 1);
        if (p < kGroupList) sm.list[p] = b;
    });
    __syncthreads();
    auto write = [&](int k, const Best& b) {
        const size_t o = static_cast<size_t>(g) * a.keep + k;
        a.out_scores[o] = float_from_order_key(b.bits);
        a.out_parents[o] = g * a.beams + b.row;
        a.out_tokens[o] = candidate_index(b.key);
    };
    const int count = sm.count;
    if (count <= kGroupList) {
        for (int c = threadIdx.x; c < count; c += THREADS) {
            const Best b = sm.list[c];
            int rank = 0;
            for (int i = 0; i < count; ++i) rank += better(sm.list[i], b);
            if (rank < a.keep) write(rank, b);
        }
        return;
    }
    // Too many ties to count: one winner after the other.
    Best last{kAll, -1, ~0ull};
    for (int k = 0; k < a.keep; ++k) {
        Best best{0, kMaxBeams, 0};
        each([&](const Best& b) {
            if (better(last, b) && better(b, best)) best = b;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Best b{__shfl_xor_sync(kAll, best.bits, o), __shfl_xor_sync(kAll, best.row, o), __shfl_xor_sync(kAll, best.key, o)};
            if (better(b, best)) best = b;
        }
        __syncthreads();
        if (lane == 0) sm.best[warp] = best;
        __syncthreads();
        best = sm.best[0];
        for (int w = 1; w < THREADS / 32; ++w)
            if (better(sm.best[w], best)) best = sm.best[w];
        if (threadIdx.x == 0) write(k, best);
        last = best;
    }
}

// 2^x to 22 bits, which a sum of thousands of them averages out.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct ChunkRoom {
    uint64_t list[kList];
    float m[kThreads / 32], s[kThreads / 32];
    uint32_t bounds[kThreads / 32];
    int n[kThreads / 32], count;
};

// The sorted list and the sums of one chunk of a row that goes on.
template <typename X>
__device__ __forceinline__ void list_chunk(const cudallm_beam_args& a, int row, int chunk, bool wide, uint64_t* out, float2* stat, ChunkRoom& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const X* x = static_cast<const X*>(a.logits) + row * a.row_stride;
    constexpr int kVec = 16 / sizeof(X);
    const int c0 = chunk * kChunk, n = min(kChunk, a.vocab - c0);
    // Place in the chunk of this thread's logit j.
    auto at = [&](int j) {
        return wide ? (j / kVec * kThreads + static_cast<int>(threadIdx.x)) * kVec + j % kVec : j * kThreads + static_cast<int>(threadIdx.x);
    };
    float v[kEach];
    if (wide) {
#pragma unroll
        for (int j = 0; j < kEach; j += kVec) {
            const int i = at(j);
            if (i + kVec <= n) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + c0 + i));
                X part[kVec];
                memcpy(part, &raw, 16);
#pragma unroll
                for (int e = 0; e < kVec; ++e) v[j + e] = as_float(part[e]);
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) v[j + e] = i + e < n ? as_float(x[c0 + i + e]) : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[j] = at(j) < n ? as_float(x[c0 + at(j)]) : -INFINITY;
    }
    auto inside = [&](int j) { return n == kChunk || at(j) < n; };
    float top[2] = {-INFINITY, -INFINITY};  // what is not a number is left out, as -inf would be
#pragma unroll
    for (int j = 0; j < kEach; ++j) top[j & 1] = fmaxf(top[j & 1], v[j]);
    float m = fmaxf(top[0], top[1]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    const float ref = m == -INFINITY ? 0.f : m;
    constexpr float kLog2e = 1.4426950408889634f;
    float s = 0.f;  // x - m first: scaled apart, the two would differ by the rounding of m, which passes any exponent where all is masked by a large number
#pragma unroll
    for (int j = 0; j < kEach; ++j) s += exp2_fast((v[j] - ref) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    if (lane == 0) {
        sm.m[warp] = m;
        sm.s[warp] = s;
    }
    if (threadIdx.x == 0) sm.count = 0;
    // Threads with two logits or more have two samples.
    const int sampled = wide ? n / kVec : max(0, n - kThreads);
    const uint32_t low = block_bound<kThreads>(inside(0) ? logit_bits(top[0]) : 0u, inside(1) ? logit_bits(top[1]) : 0u, a.keep, min(sampled, kThreads) / 32, sm.bounds);
    const float bound = low > 1u ? float_from_order_key(low) : -INFINITY;
    if (warp == 1) {  // the warps' sums as one
        static_assert(kThreads / 32 == 8, "lanes 0 .. 7 have a warp's each");
        const float wm = sm.m[lane & 7];
        float mm = wm;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(kAll, mm, o));
        float ss = sm.s[lane & 7] * expf(wm == -INFINITY ? (mm == -INFINITY ? 0.f : -INFINITY) : wm - mm);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
        if (lane == 0) *stat = make_float2(mm, ss);
    }
    auto push = [&](int j, uint32_t bits) {
        const int p = atomicAdd(&sm.count, 1);
        if (p < kList) sm.list[p] = static_cast<uint64_t>(bits) << 32 | static_cast<uint32_t>(~(c0 + at(j)));
    };
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (!(v[j] < bound) && inside(j)) push(j, logit_bits(v[j]));
    __syncthreads();
    if (sm.count > kList) {
        // Too many ties to list: the keep-th value, then how far its ties go. 0 where there is no logit (every logit's bits are above).
        uint32_t bits[kEach], value = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) bits[j] = inside(j) ? logit_bits(v[j]) : 0u;
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t test = value | 1u << bit;
            int above = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) above += bits[j] >= test;
            if (block_sum<kThreads>(above, sm.n) >= a.keep) value = test;
        }
        int above = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) above += bits[j] > value;
        const int ties = a.keep - block_sum<kThreads>(above, sm.n);  // wanted: 1 or more
        static_assert(kChunk == 1 << 13, "places have 13 bits");
        uint32_t last = 0;  // the largest place with fewer ties before it
#pragma unroll 1
        for (int bit = 12; bit >= 0; --bit) {
            const uint32_t test = last | 1u << bit;
            above = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) above += bits[j] == value && at(j) < static_cast<int>(test);
            if (block_sum<kThreads>(above, sm.n) < ties) last = test;
        }
        if (threadIdx.x == 0) sm.count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (bits[j] > value || (bits[j] == value && static_cast<uint32_t>(at(j)) <= last)) push(j, bits[j]);
    }
    __syncthreads();
    const int count = min(sm.count, kList);
    if (threadIdx.x < count) {
        const uint64_t key = sm.list[threadIdx.x];
        int rank = 0;
        for (int i = 0; i < count; ++i) rank += sm.list[i] > key;
        if (rank < a.keep) out[rank] = key;
    }
    for (int k = count + threadIdx.x; k < a.keep; k += kThreads) out[k] = 0;
}

// Block = chunk of a row. With `counts` (one zero for each group), the last block of a group to finish selects its best.
template <typename X>
__global__ void __launch_bounds__(kThreads, 4) beam_chunk_kernel(const __grid_constant__ cudallm_beam_args a, uint64_t* lists, float2* stats, int chunks, bool wide,
                                                                 unsigned* counts) {
    __shared__ union {
        ChunkRoom chunk;
        GroupRoom<kThreads> group;
    } room;
    __shared__ bool last;
    grid_dep_wait();
    grid_dep_launch();
    const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    const size_t place = blockIdx.x;
    uint64_t* out = lists + place * a.keep;
    if (a.finished != nullptr && a.finished[row] != 0) {
        // 0 at eos, then -inf from the lowest token on; the other chunks of the row have nothing.
        for (int k = threadIdx.x; k < a.keep; k += kThreads) {
            const int t = k == 0 ? a.eos : k - 1 + (k - 1 >= a.eos ? 1 : 0);
            out[k] = chunk == 0 && t < a.vocab ? candidate_key(k == 0 ? 0.f : -INFINITY, t) : 0;
        }
        if (threadIdx.x == 0) stats[place] = chunk == 0 ? make_float2(0.f, 1.f) : make_float2(-INFINITY, 0.f);
    } else {
        list_chunk<X>(a, row, chunk, wide, out, stats + place, room.chunk);
    }
    if (counts == nullptr) return;
    __syncthreads();
    const int g = row / a.beams;
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(counts + g, 1u) == static_cast<unsigned>(a.beams * chunks - 1);
        if (last) counts[g] = 0u;
        __threadfence();
    }
    __syncthreads();
    if (last) select_group<kThreads>(a, lists, stats, chunks, g, room.group);
}

__global__ void __launch_bounds__(kGroupThreads) beam_group_kernel(const __grid_constant__ cudallm_beam_args a, const uint64_t* lists, const float2* stats,
                                                                   int chunks) {
    __shared__ GroupRoom<kGroupThreads> room;
    grid_dep_wait();
    select_group<kGroupThreads>(a, lists, stats, chunks, blockIdx.x, room);
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

size_t beam_workspace_bytes(int rows, int vocab, int keep) {
    if (rows < 0 || rows > kMaxPageRows || vocab < 1 || vocab > kMaxVocab || keep < 1 || keep > kMaxKeep) return 0;
    return CUDALLM_BEAM_COUNTER_BYTES + (sizeof(float2) + sizeof(uint64_t) * keep) * static_cast<size_t>(rows) * chunks_of(vocab);
}

void launch_beam_select(const cudallm_beam_args& a, cudaStream_t stream) {
    if (a.n_groups == 0) return;
    const int rows = a.n_groups * a.beams, chunks = chunks_of(a.vocab);
    const bool one = static_cast<long long>(rows) * chunks <= kOneLaunch && a.n_groups <= static_cast<int>(CUDALLM_BEAM_COUNTER_BYTES / 4);
    auto* counts = one ? static_cast<unsigned*>(a.workspace) : nullptr;
    auto* stats = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + CUDALLM_BEAM_COUNTER_BYTES);
    auto* lists = reinterpret_cast<uint64_t*>(stats + static_cast<size_t>(rows) * chunks);
    const size_t es = a.x_dtype == CUDALLM_X_FP32 ? 4 : 2;
    const bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (rows == 1 || a.row_stride * es % 16 == 0);
    auto* kernel = a.x_dtype == CUDALLM_X_FP32   ? beam_chunk_kernel<float>
                   : a.x_dtype == CUDALLM_X_FP16 ? beam_chunk_kernel<__half>
                                                 : beam_chunk_kernel<__nv_bfloat16>;
    launch_kernel(kernel, dim3(rows * chunks), dim3(kThreads), 0, stream, true, a, lists, stats, chunks, wide, counts);
    if (counts != nullptr) return;
    launch_kernel(beam_group_kernel, dim3(a.n_groups), dim3(kGroupThreads), 0, stream, true, a, static_cast<const uint64_t*>(lists),
                  static_cast<const float2*>(stats), chunks);
}

}  // namespace cudallm
