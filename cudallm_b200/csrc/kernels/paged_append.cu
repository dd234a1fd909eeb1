// Rotary positions of new tokens, with the store of their keys and values to the pages of a cache.
//
//   (a, b) -> factor (a cos - b sin, b cos + a sin),  angle = fl32(position * inv_freq[j])
//
// One block per token; threads walk the token's heads, one rotated pair or copied dim at a time.
#include "common/check.h"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"

namespace cudallm {

namespace {

constexpr int kThreads = 256;

template <typename X, typename KV>
__global__ void __launch_bounds__(kThreads) append_kernel(cudallm_pages pg, cudallm_append_args a) {
    __shared__ float sm_cos[128], sm_sin[128];
    const long long i = blockIdx.x;
    const int pos = a.positions[i], n = a.rotary / 2, hd = pg.head_dim;
    for (int j = threadIdx.x; j < n; j += kThreads) {
        float s, c;
        sincosf(static_cast<float>(pos) * a.inv_freq[j], &s, &c);
        sm_cos[j] = c * a.factor;
        sm_sin[j] = s * a.factor;
    }
    __syncthreads();
    long long slot = -1;
    const int row = a.rows != nullptr ? a.rows[i] : static_cast<int>(i);
    if (pos >= 0 && row >= 0 && row < a.n_rows && pos / pg.page_size < a.table_width) {
        const int page = a.tables[row * a.table_stride + pos / pg.page_size];
        if (page >= 0 && page < pg.n_pages) {
            slot = a.layer * pg.layer_stride + page * pg.page_stride + (pos % pg.page_size) * pg.token_stride;
        }
    }
    const int q_heads = a.q != nullptr ? a.n_heads : 0;
    const int units = hd - n;  // per head: n pairs, then the dims from `rotary` on
    const int total = (q_heads + 2 * pg.n_kv_heads) * units;
    for (int u = threadIdx.x; u < total; u += kThreads) {
        const int head = u / units, w = u % units;
        const bool is_q = head < q_heads, is_v = head >= q_heads + pg.n_kv_heads;
        const int kvh = is_q ? 0 : (head - q_heads) % pg.n_kv_heads;
        if (!is_q && slot < 0) continue;
        const X* src = is_q ? static_cast<const X*>(a.q) + i * a.q_token_stride + head * a.q_head_stride
                       : is_v ? static_cast<const X*>(a.v) + i * a.v_token_stride + kvh * a.v_head_stride
                              : static_cast<const X*>(a.k) + i * a.k_token_stride + kvh * a.k_head_stride;
        const bool pair = w < n;
        const int d0 = !pair ? n + w : a.interleaved ? 2 * w : w;
        const int d1 = !pair ? d0 : a.interleaved ? d0 + 1 : d0 + n;
        float v0 = as_float(src[d0]), v1 = as_float(src[d1]);
        if (pair && !is_v) {
            const float c = sm_cos[w], s = sm_sin[w];
            const float r0 = v0 * c - v1 * s, r1 = v1 * c + v0 * s;
            v0 = r0;
            v1 = r1;
        }
        if (is_q) {
            X* dst = static_cast<X*>(a.q_out) + i * a.out_token_stride + head * a.out_head_stride;
            dst[d0] = from_float<X>(pos < 0 ? 0.f : v0);
            if (pair) dst[d1] = from_float<X>(pos < 0 ? 0.f : v1);
        } else {
            KV* dst = static_cast<KV*>(is_v ? pg.v : pg.k) + slot + kvh * pg.head_stride;
            dst[d0] = from_float<KV>(v0);
            if (pair) dst[d1] = from_float<KV>(v1);
        }
    }
}

template <typename X>
void launch_for(const cudallm_pages& pg, const cudallm_append_args& a, cudaStream_t stream) {
    if (pg.kv_dtype == CUDALLM_KV_BF16) {
        append_kernel<X, __nv_bfloat16><<<a.n_tokens, kThreads, 0, stream>>>(pg, a);
    } else {
        append_kernel<X, __half><<<a.n_tokens, kThreads, 0, stream>>>(pg, a);
    }
}

}  // namespace

void launch_paged_append(const cudallm_pages& pg, const cudallm_append_args& a, cudaStream_t stream) {
    if (a.n_tokens == 0) return;
    switch (a.x_dtype) {
        case CUDALLM_X_FP32: launch_for<float>(pg, a, stream); break;
        case CUDALLM_X_FP16: launch_for<__half>(pg, a, stream); break;
        default: launch_for<__nv_bfloat16>(pg, a, stream); break;
    }
    CLLM_CUDA(cudaGetLastError());
}

}  // namespace cudallm
