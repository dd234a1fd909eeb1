// Beam search's selection: the best continuations of each group of beams over beams and vocabulary.
//
//   candidate(w, t) = score[w] + (x[t] - lse(x)),  x = row w's logits,  lse(x) = m + ln sum_t exp(x[t] - m)
//
// Within a row candidates rank as (logit, then lower token), so the `keep` best by logit of each chunk of a row are the
// only ones that can be among the group's.
//
// chunk kernel: one block per 4096 logits, which stay in registers (one read of the logits, what bounds the operator at
//   many rows). It leaves their maximum, their sum of exponentials and the sorted keys of their `keep` best. A lower
//   bound of the keep-th best is the keep-th largest of the maxima of 512 pieces; the few logits above it are ranked by
//   counting. Where more than 256 are above it (ties, a masked vocabulary) the keep-th key itself is
//   searched bit by bit over value and token.
// group kernel: one block per group, in place when the chunks are done. It joins the rows' sums and ranks the chunks'
//   lists' candidates in the same way.
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
constexpr int kEach = 16;  // logits of a thread
constexpr int kChunk = kThreads * kEach;
constexpr int kList = 256;  // candidates above the bound that are ranked by counting
constexpr int kGroupThreads = 512;
constexpr int kGroupList = 512;
constexpr unsigned kAll = 0xffffffffu;

// Rank bits of a logit: not a number counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t logit_bits(float x) { return float_order_key(isnan(x) ? -INFINITY : x + 0.f); }

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

// 2^x to 22 bits, which a sum of thousands of them averages out; exp(x) = 2^(x log2(e)).
__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

template <typename X>
__global__ void __launch_bounds__(kThreads) beam_chunk_kernel(const __grid_constant__ cudallm_beam_args a, uint64_t* lists, float2* stats, int chunks,
                                                              bool wide) {
    __shared__ uint64_t list[kList];
    __shared__ float sm_m[kThreads / 32], sm_s[kThreads / 32];
    __shared__ uint32_t samples[2 * kThreads], sm_bound;
    __shared__ int sm_n[kThreads / 32], sm_count;
    static_assert(2 * kThreads == 512, "bound_of takes 512");
    grid_dep_launch();
    const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t place = blockIdx.x;
    uint64_t* out = lists + place * a.keep;
    if (a.finished != nullptr && a.finished[row] != 0) {
        // 0 at eos, then -inf from the lowest token on; the other chunks of the row have nothing.
        for (int k = threadIdx.x; k < a.keep; k += kThreads) {
            const int t = k == 0 ? a.eos : k - 1 + (k - 1 >= a.eos ? 1 : 0);
            out[k] = chunk == 0 && t < a.vocab ? candidate_key(k == 0 ? 0.f : -INFINITY, t) : 0;
        }
        if (threadIdx.x == 0) stats[place] = chunk == 0 ? make_float2(0.f, 1.f) : make_float2(-INFINITY, 0.f);
        return;
    }
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
    // Rank bits; 0 where there is no logit (every logit's are above 0).
    uint32_t bits[kEach], top[2] = {0, 0};
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        bits[j] = at(j) < n ? logit_bits(v[j]) : 0u;
        top[j & 1] = max(top[j & 1], bits[j]);
        m = fmaxf(m, v[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kEach; ++j) s += exp_fast(v[j] - ref);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    if (lane == 0) {
        sm_m[warp] = m;
        sm_s[warp] = s;
    }
    samples[threadIdx.x] = top[0];
    samples[kThreads + threadIdx.x] = top[1];
    __syncthreads();
    if (warp == 0) {
        const uint32_t b = bound_of(samples, a.keep);
        if (lane == 0) {
            sm_bound = max(b, 1u);  // places without a logit are never taken
            sm_count = 0;
        }
    }
    if (threadIdx.x == 32) {
        float mm = -INFINITY, ss = 0.f;
        for (int w = 0; w < kThreads / 32; ++w) mm = fmaxf(mm, sm_m[w]);
        for (int w = 0; w < kThreads / 32; ++w) ss += sm_s[w] * expf(sm_m[w] == -INFINITY ? (mm == -INFINITY ? 0.f : -INFINITY) : sm_m[w] - mm);
        stats[place] = make_float2(mm, ss);
    }
    __syncthreads();
    uint32_t bound = sm_bound;
    auto push = [&](int j) {
        const int p = atomicAdd(&sm_count, 1);
        if (p < kList) list[p] = static_cast<uint64_t>(bits[j]) << 32 | static_cast<uint32_t>(~(c0 + at(j)));
    };
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (bits[j] >= bound) push(j);
    __syncthreads();
    if (sm_count > kList) {
        // Too many ties to list: the keep-th value, then how far its ties go.
        bound = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t test = bound | 1u << bit;
            int above = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) above += bits[j] >= test;
            if (block_sum<kThreads>(above, sm_n) >= a.keep) bound = test;
        }
        int above = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) above += bits[j] > bound;
        const int ties = a.keep - block_sum<kThreads>(above, sm_n);  // wanted: 1 or more
        uint32_t last = 0;  // the largest place with fewer ties before it
#pragma unroll 1
        for (int bit = 11; bit >= 0; --bit) {
            const uint32_t test = last | 1u << bit;
            above = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) above += bits[j] == bound && at(j) < static_cast<int>(test);
            if (block_sum<kThreads>(above, sm_n) < ties) last = test;
        }
        if (threadIdx.x == 0) sm_count = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (bits[j] > bound || (bits[j] == bound && static_cast<uint32_t>(at(j)) <= last)) push(j);
    }
    __syncthreads();
    const int count = min(sm_count, kList);
    if (threadIdx.x < count) {
        const uint64_t key = list[threadIdx.x];
        int rank = 0;
        for (int i = 0; i < count; ++i) rank += list[i] > key;
        if (rank < a.keep) out[rank] = key;
    }
    for (int k = count + threadIdx.x; k < a.keep; k += kThreads) out[k] = 0;
}

struct Best {
    uint32_t bits;  // of the candidate
    int row;        // beam in the group
    uint64_t key;   // logit and token
};
__device__ __forceinline__ bool better(const Best& a, const Best& b) {
    return a.bits != b.bits ? a.bits > b.bits : a.row != b.row ? a.row < b.row : a.key > b.key;
}

__global__ void __launch_bounds__(kGroupThreads) beam_group_kernel(const __grid_constant__ cudallm_beam_args a, const uint64_t* lists, const float2* stats,
                                                                   int chunks) {
    __shared__ float lse[kMaxBeams], score[kMaxBeams];
    __shared__ Best list[kGroupList];
    __shared__ uint32_t samples[kGroupThreads], sm_bound;
    __shared__ int sm_count;
    const int g = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sm_count = 0;
    grid_dep_wait();
    for (int w = warp; w < a.beams; w += kGroupThreads / 32) {
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
            lse[w] = m + logf(s);
            score[w] = a.scores[static_cast<size_t>(g) * a.beams + w];
        }
    }
    __syncthreads();
    const int n_lists = a.beams * chunks;
    const uint64_t* keys = lists + static_cast<size_t>(g) * n_lists * a.keep;
    auto read = [&](int l, int k) {  // candidate k of list l
        Best b;
        b.key = __ldcg(keys + static_cast<size_t>(l) * a.keep + k);
        b.row = l / chunks;
        const float v = score[b.row] + (candidate_value(b.key) - lse[b.row]);
        b.bits = b.key == 0 ? 0u : float_order_key(isnan(v) ? -INFINITY : v + 0.f);
        return b;
    };
    // With fewer lists than threads, several threads take a list's candidates in turn; the first of each thread are the samples.
    const int across = min(n_lists, kGroupThreads), step = kGroupThreads / across;
    const int l0 = threadIdx.x % across, k0 = threadIdx.x / across;
    const bool works = k0 < step && k0 < a.keep;
    uint32_t top = 0;
    if (works) {
        for (int l = l0; l < n_lists; l += across) top = max(top, read(l, k0).bits);
    }
    samples[threadIdx.x] = top;
    __syncthreads();
    if (warp == 0) {
        const uint32_t b = bound_of(samples, a.keep);
        if (lane == 0) sm_bound = max(b, 1u);
    }
    __syncthreads();
    const uint32_t bound = sm_bound;
    if (works) {
        for (int l = l0; l < n_lists; l += across) {
            for (int k = k0; k < a.keep; k += step) {
                const Best b = read(l, k);
                if (b.bits < bound) break;  // lists descend
                const int p = atomicAdd(&sm_count, 1);
                if (p < kGroupList) list[p] = b;
            }
        }
    }
    __syncthreads();
    const int count = sm_count;
    auto write = [&](int k, const Best& b) {
        const size_t o = static_cast<size_t>(g) * a.keep + k;
        a.out_scores[o] = float_from_order_key(b.bits);
        a.out_parents[o] = g * a.beams + b.row;
        a.out_tokens[o] = candidate_index(b.key);
    };
    if (count <= kGroupList) {
        if (threadIdx.x < count) {
            const Best b = list[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < count; ++i) rank += better(list[i], b);
            if (rank < a.keep) write(rank, b);
        }
        return;
    }
    // Too many ties to count: one winner after the other.
    __shared__ Best sm_best[kGroupThreads / 32];
    Best last{kAll, -1, ~0ull};
    for (int k = 0; k < a.keep; ++k) {
        Best best{0, kMaxBeams, 0};
        if (works) {
            for (int l = l0; l < n_lists; l += across) {
                for (int i = k0; i < a.keep; i += step) {
                    const Best b = read(l, i);
                    if (b.bits < bound) break;
                    if (better(last, b) && better(b, best)) best = b;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Best b{__shfl_xor_sync(kAll, best.bits, o), __shfl_xor_sync(kAll, best.row, o), __shfl_xor_sync(kAll, best.key, o)};
            if (better(b, best)) best = b;
        }
        __syncthreads();
        if (lane == 0) sm_best[warp] = best;
        __syncthreads();
        best = sm_best[0];
        for (int w = 1; w < kGroupThreads / 32; ++w)
            if (better(sm_best[w], best)) best = sm_best[w];
        if (threadIdx.x == 0) write(k, best);
        last = best;
    }
}

int chunks_of(int vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace

size_t beam_workspace_bytes(int rows, int vocab, int keep) {
    if (rows < 0 || rows > kMaxPageRows || vocab < 1 || vocab > kMaxVocab || keep < 1 || keep > kMaxKeep) return 0;
    return 256 + (sizeof(float2) + sizeof(uint64_t) * keep) * static_cast<size_t>(rows) * chunks_of(vocab);
}

void launch_beam_select(const cudallm_beam_args& a, cudaStream_t stream) {
    if (a.n_groups == 0) return;
    const int rows = a.n_groups * a.beams, chunks = chunks_of(a.vocab);
    auto* stats = static_cast<float2*>(a.workspace);
    auto* lists = reinterpret_cast<uint64_t*>(stats + static_cast<size_t>(rows) * chunks);
    const size_t es = a.x_dtype == CUDALLM_X_FP32 ? 4 : 2;
    const bool wide = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (rows == 1 || a.row_stride * es % 16 == 0);
    auto* kernel = a.x_dtype == CUDALLM_X_FP32   ? beam_chunk_kernel<float>
                   : a.x_dtype == CUDALLM_X_FP16 ? beam_chunk_kernel<__half>
                                                 : beam_chunk_kernel<__nv_bfloat16>;
    launch_kernel(kernel, dim3(rows * chunks), dim3(kThreads), 0, stream, false, a, lists, stats, chunks, wide);
    launch_kernel(beam_group_kernel, dim3(a.n_groups), dim3(kGroupThreads), 0, stream, true, a, static_cast<const uint64_t*>(lists),
                  static_cast<const float2*>(stats), chunks);
}

}  // namespace cudallm
