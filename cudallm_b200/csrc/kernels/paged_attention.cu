// Attention of one new token per sequence over a paged key-value cache.
//
//   out[b][h] = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),  s_t = scale q.k_t,  m = max_t s_t,
//   lse[b][h] = m + ln sum_t exp(s_t - m)
//
// One block per (sequence, query head); each warp takes every fourth position, lanes hold the head's dims, and the
// warps' running (m, sum, out) are merged in warp order.
#include <climits>
#include <cmath>

#include "common/check.h"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"

namespace cudallm {

namespace {

constexpr int kWarps = 4;
constexpr int kDimsPerLane = 8;  // 256 / 32

template <typename X, typename KV>
__global__ void __launch_bounds__(32 * kWarps) attend_kernel(cudallm_pages pg, cudallm_attend_args a) {
    __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][256];
    const int b = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads;
    const int kvh = h / (a.n_heads / pg.n_kv_heads);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = pg.head_dim;
    const long long cap = static_cast<long long>(a.table_width) * pg.page_size;
    const int len = static_cast<int>(min(static_cast<long long>(max(a.lens[b], 0)), cap));
    const int first = a.window > 0 ? max(0, len - a.window) : 0;
    const X* q = static_cast<const X*>(a.q) + b * a.q_seq_stride + h * a.q_head_stride;
    const KV* K = static_cast<const KV*>(pg.k) + a.layer * pg.layer_stride + kvh * pg.head_stride;
    const KV* V = static_cast<const KV*>(pg.v) + a.layer * pg.layer_stride + kvh * pg.head_stride;
    float qv[kDimsPerLane], o[kDimsPerLane], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kDimsPerLane; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < hd ? as_float(q[d]) * a.scale : 0.f;
        o[i] = 0.f;
    }
    for (int t = first + warp; t < len; t += kWarps) {
        const int page = a.tables[b * a.table_stride + t / pg.page_size];
        if (page < 0 || page >= pg.n_pages) continue;
        const long long at = page * pg.page_stride + (t % pg.page_size) * pg.token_stride;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kDimsPerLane; ++i) {
            const int d = lane + 32 * i;
            if (d < hd) s = fmaf(qv[i], as_float(K[at + d]), s);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float mn = fmaxf(m, s), old = expf(m - mn), p = expf(s - mn);
        m = mn;
        l = l * old + p;
#pragma unroll
        for (int i = 0; i < kDimsPerLane; ++i) {
            const int d = lane + 32 * i;
            if (d < hd) o[i] = fmaf(p, as_float(V[at + d]), o[i] * old);
        }
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < kDimsPerLane; ++i) sm_o[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float mm = -INFINITY, ll = 0.f;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w]);
    float scale[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        scale[w] = mm == -INFINITY ? 0.f : expf(sm_m[w] - mm);
        ll += scale[w] * sm_l[w];
    }
    X* out = static_cast<X*>(a.out) + static_cast<long long>(blockIdx.x) * hd;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float v = 0.f;
        for (int w = 0; w < kWarps; ++w) v += scale[w] * sm_o[w][d];
        out[d] = from_float<X>(ll > 0.f ? v / ll : 0.f);
    }
    if (a.lse != nullptr && threadIdx.x == 0) a.lse[blockIdx.x] = mm + logf(ll);
}

template <typename X>
void launch_for(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(a.n_seq) * a.n_heads;
    if (pg.kv_dtype == CUDALLM_KV_BF16) {
        attend_kernel<X, __nv_bfloat16><<<grid, 32 * kWarps, 0, stream>>>(pg, a);
    } else {
        attend_kernel<X, __half><<<grid, 32 * kWarps, 0, stream>>>(pg, a);
    }
}

}  // namespace

size_t attend_workspace_bytes() { return kPagedCounterBytes; }

void launch_paged_attend(const cudallm_pages& pg, const cudallm_attend_args& a, cudaStream_t stream) {
    if (a.n_seq == 0) return;
    switch (a.x_dtype) {
        case CUDALLM_X_FP32: launch_for<float>(pg, a, stream); break;
        case CUDALLM_X_FP16: launch_for<__half>(pg, a, stream); break;
        default: launch_for<__nv_bfloat16>(pg, a, stream); break;
    }
    CLLM_CUDA(cudaGetLastError());
}

}  // namespace cudallm
