// Beam search's selection: the best continuations of each group of beams over beams and vocabulary.
//
//   candidate(w, t) = score[w] + (x[t] - lse(x)),  x = row w's logits,  lse(x) = m + ln sum_t exp(x[t] - m)
//
// Within a row candidates rank as (logit, then lower token), so a row's `keep` best by logit are the only ones that can
// be among the group's. One block per row finds its lse and those, by `keep` passes over the row; one block per
// group then picks the best of its rows' lists.
#include <climits>
#include <cmath>

#include "common/check.h"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"
#include "kernels/sampling.cuh"

namespace cudallm {

namespace {

constexpr int kThreads = 512;

struct Candidate {
    float value;
    int token;
};

// Rank of a logit in its row: not a number counts as -inf, -0 as 0, lower tokens win ties.
__device__ __forceinline__ uint64_t row_key(float x, int token) { return candidate_key(isnan(x) ? -INFINITY : x + 0.f, token); }

__device__ __forceinline__ float block_reduce(float v, float* sm, bool is_max) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t = __shfl_xor_sync(0xffffffffu, v, o);
        v = is_max ? fmaxf(v, t) : v + t;
    }
    __syncthreads();
    if (lane == 0) sm[warp] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < kThreads / 32; ++w) v = is_max ? fmaxf(v, sm[w]) : v + sm[w];
    return v;
}

__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t t = __shfl_xor_sync(0xffffffffu, v, o);
        v = t > v ? t : v;
    }
    __syncthreads();
    if (lane == 0) sm[warp] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < kThreads / 32; ++w) v = sm[w] > v ? sm[w] : v;
    return v;
}

template <typename X>
__global__ void __launch_bounds__(kThreads) beam_row_kernel(cudallm_beam_args a, Candidate* lists) {
    __shared__ float sm_f[kThreads / 32];
    __shared__ uint64_t sm_k[kThreads / 32];
    const int row = blockIdx.x;
    const X* x = static_cast<const X*>(a.logits) + row * a.row_stride;
    const bool done = a.finished != nullptr && a.finished[row] != 0;
    auto at = [&](int t) { return done ? (t == a.eos ? 0.f : -INFINITY) : as_float(x[t]); };
    float m = -INFINITY, sum = 0.f;
    for (int t = threadIdx.x; t < a.vocab; t += kThreads) m = fmaxf(m, at(t));
    m = block_reduce(m, sm_f, true);
    for (int t = threadIdx.x; t < a.vocab; t += kThreads) sum += expf(at(t) - m);
    sum = block_reduce(sum, sm_f, false);
    const float lse = m + logf(sum), score = a.scores[row];
    uint64_t last = ~0ull;
    for (int k = 0; k < a.keep; ++k) {
        uint64_t best = 0;
        for (int t = threadIdx.x; t < a.vocab; t += kThreads) {
            const uint64_t key = row_key(at(t), t);
            if (key < last && key > best) best = key;
        }
        best = block_max(best, sm_k);
        if (threadIdx.x == 0) {
            Candidate c{-INFINITY, -1};
            if (best != 0) {
                const int t = candidate_index(best);
                const float v = score + (at(t) - lse);
                c = {isnan(v) ? -INFINITY : v, t};
            }
            lists[static_cast<size_t>(row) * a.keep + k] = c;
        }
        last = best;
    }
}

// Candidates of a group in the order (beam, rank in its row): the key (value, then lower place) ranks them.
__global__ void __launch_bounds__(kThreads) beam_group_kernel(cudallm_beam_args a, const Candidate* lists) {
    __shared__ uint64_t sm_k[kThreads / 32];
    const int g = blockIdx.x, n = a.beams * a.keep;
    const Candidate* list = lists + static_cast<size_t>(g) * n;
    uint64_t last = ~0ull;
    for (int k = 0; k < a.keep; ++k) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            if (list[i].token < 0) continue;
            const uint64_t key = candidate_key(list[i].value + 0.f, i);
            if (key < last && key > best) best = key;
        }
        best = block_max(best, sm_k);
        if (threadIdx.x == 0) {
            const int i = candidate_index(best);
            const size_t o = static_cast<size_t>(g) * a.keep + k;
            a.out_scores[o] = list[i].value;
            a.out_parents[o] = g * a.beams + i / a.keep;
            a.out_tokens[o] = list[i].token;
        }
        last = best;
    }
}

}  // namespace

size_t beam_workspace_bytes(int rows, int vocab, int keep) {
    if (rows < 0 || vocab < 1 || keep < 1 || keep > kMaxKeep) return 0;
    return kPagedCounterBytes + sizeof(Candidate) * static_cast<size_t>(rows) * keep;
}

void launch_beam_select(const cudallm_beam_args& a, cudaStream_t stream) {
    if (a.n_groups == 0) return;
    auto* lists = reinterpret_cast<Candidate*>(static_cast<char*>(a.workspace) + kPagedCounterBytes);
    const int rows = a.n_groups * a.beams;
    switch (a.x_dtype) {
        case CUDALLM_X_FP32: beam_row_kernel<float><<<rows, kThreads, 0, stream>>>(a, lists); break;
        case CUDALLM_X_FP16: beam_row_kernel<__half><<<rows, kThreads, 0, stream>>>(a, lists); break;
        default: beam_row_kernel<__nv_bfloat16><<<rows, kThreads, 0, stream>>>(a, lists); break;
    }
    CLLM_CUDA(cudaGetLastError());
    beam_group_kernel<<<a.n_groups, kThreads, 0, stream>>>(a, lists);
    CLLM_CUDA(cudaGetLastError());
}

}  // namespace cudallm
