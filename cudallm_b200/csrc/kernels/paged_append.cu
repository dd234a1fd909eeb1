// Rotary positions of new tokens, with the store of their keys and values to the pages of a cache.
//
//   (a, b) -> factor (a cos - b sin, b cos + a sin),  angle = fl32(position * inv_freq[j])
//
// Every input is read once and every output written once: HBM bounds it at many tokens, launch latency at few. A block
// takes one or more tokens, computes their cosines once for all heads, and its threads walk the heads in units of 8
// dims (16-byte accesses of 16-bit types): the two halves of 8 pairs, 4 interleaved pairs, or 8 dims that are copied.
// Where strides or sizes do not allow that, a unit is one pair or one dim.
#include <algorithm>
#include <cstring>

#include "common/check.h"
#include "kernels/kernels.h"
#include "kernels/launch.cuh"
#include "kernels/paged.h"
#include "kernels/paged_common.cuh"

namespace cudallm {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 8;  // of a block at most
constexpr int kBatch = 3;   // units of a thread that are loaded together

struct Params {
    cudallm_pages pg;
    cudallm_append_args a;
    int q_heads, heads;   // query heads; all heads of a token
    int tokens;           // of a block
    int pairs, pair_units, units;  // rotated pairs of a head; its units that rotate; all its units
    FastDiv by_units, by_heads;
};

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        T x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = from_float<T>(v[i]);
        uint4 raw;
        memcpy(&raw, x, 16);
        *reinterpret_cast<uint4*>(p) = raw;
    }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

// A unit of a head as its source holds it: 8 dims, or two times 8 (16-byte words); or one dim, or two.
template <typename X, bool WIDE>
struct Unit {
    uint4 raw[WIDE ? sizeof(X) : 1];
    X one[2];
};

// Dims of unit u: the first ones, and the second ones where it has two parts.
template <bool WIDE>
__device__ __forceinline__ void places(const Params& p, int u, bool& pair, int& d0, int& d1) {
    constexpr int kDims = WIDE ? 8 : 1;
    pair = u < p.pair_units;
    const bool halves = pair && !p.a.interleaved;
    d0 = pair ? u * kDims : 2 * p.pairs + (u - p.pair_units) * kDims;
    if (!WIDE && pair && p.a.interleaved) d0 = 2 * u;
    d1 = halves ? d0 + p.pairs : !WIDE && pair ? d0 + 1 : -1;
}

template <typename X, bool WIDE>
__device__ __forceinline__ void read_unit(const Params& p, int u, const X* src, Unit<X, WIDE>& r) {
    bool pair;
    int d0, d1;
    places<WIDE>(p, u, pair, d0, d1);
    if constexpr (WIDE) {
        constexpr int kWords = sizeof(X) / 2;  // of 8 dims
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            r.raw[i] = reinterpret_cast<const uint4*>(src + d0)[i];
            if (d1 >= 0) r.raw[kWords + i] = reinterpret_cast<const uint4*>(src + d1)[i];
        }
    } else {
        r.one[0] = src[d0];
        if (d1 >= 0) r.one[1] = src[d1];
    }
}

// Rotates a unit and stores it. cos and sin are the token's.
template <typename X, typename Y, bool WIDE>
__device__ __forceinline__ void write_unit(const Params& p, int u, bool rotates, bool clear, const Unit<X, WIDE>& r, Y* dst, const float* cos, const float* sin) {
    bool pair;
    int d0, d1;
    places<WIDE>(p, u, pair, d0, d1);
    if constexpr (WIDE) {
        constexpr int kWords = sizeof(X) / 2;
        X x[16];
        memcpy(x, r.raw, sizeof(X) * 16);
        float v[8], w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = as_float(x[i]);
            w[i] = as_float(x[8 + i]);
        }
        if (d1 >= 0) {
            if (rotates) {
#pragma unroll
                for (int i = 0; i < 8; ++i) turn(v[i], w[i], cos[d0 + i], sin[d0 + i]);
            }
        } else if (pair && rotates) {
#pragma unroll
            for (int i = 0; i < 4; ++i) turn(v[2 * i], v[2 * i + 1], cos[u * 4 + i], sin[u * 4 + i]);
        }
        if (clear) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w[i] = 0.f;
        }
        store8(dst + d0, v);
        if (d1 >= 0) store8(dst + d1, w);
        static_assert(sizeof(r.raw) == 2 * kWords * 16, "two times 8 dims");
    } else {
        float a = as_float(r.one[0]), b = d1 >= 0 ? as_float(r.one[1]) : 0.f;
        if (pair && rotates) turn(a, b, cos[u], sin[u]);
        if (clear) a = b = 0.f;
        dst[d0] = from_float<Y>(a);
        if (d1 >= 0) dst[d1] = from_float<Y>(b);
    }
}

template <typename X, typename KV, bool WIDE>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ Params p) {
    __shared__ float cos[kTokens][128], sin[kTokens][128];
    __shared__ long long slots[kTokens];  // where the token's keys go; -1: nowhere, -2: padding
    const cudallm_append_args& a = p.a;
    const int first = blockIdx.x * p.tokens, tokens = min(p.tokens, a.n_tokens - first);
    if (threadIdx.x < tokens) {
        const int i = first + threadIdx.x, pos = a.positions[i], row = a.rows != nullptr ? a.rows[i] : i;
        long long slot = pos < 0 ? -2 : -1;
        if (pos >= 0 && row >= 0 && row < a.n_rows && pos / p.pg.page_size < a.table_width) {
            const int page = a.tables[row * a.table_stride + pos / p.pg.page_size];
            if (page >= 0 && page < p.pg.n_pages) {
                slot = a.layer * p.pg.layer_stride + page * p.pg.page_stride + (pos % p.pg.page_size) * p.pg.token_stride;
            }
        }
        slots[threadIdx.x] = slot;
    }
    for (int j = threadIdx.x; j < tokens * p.pairs; j += kThreads) {
        const int t = j / p.pairs, k = j % p.pairs;
        float s, c;
        sincosf(static_cast<float>(a.positions[first + t]) * a.inv_freq[k], &s, &c);
        cos[t][k] = c * a.factor;
        sin[t][k] = s * a.factor;
    }
    // The heads' loads are under way before the block waits for its cosines and slots.
    const int total = tokens * p.heads * p.units, step = gridDim.y * kThreads;
    bool waited = false;
    for (int x0 = blockIdx.y * kThreads + threadIdx.x; x0 < total || !waited; x0 += kBatch * step) {
        Unit<X, WIDE> units[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int x = x0 + k * step;
            if (x >= total) break;
            const int hh = div_by(x, p.by_units), t = div_by(hh, p.by_heads), head = hh - t * p.heads;
            const long long i = first + t;
            const int kvh = head - p.q_heads;
            const X* src = kvh < 0                 ? static_cast<const X*>(a.q) + i * a.q_token_stride + head * a.q_head_stride
                           : kvh < p.pg.n_kv_heads ? static_cast<const X*>(a.k) + i * a.k_token_stride + kvh * a.k_head_stride
                                                   : static_cast<const X*>(a.v) + i * a.v_token_stride + (kvh - p.pg.n_kv_heads) * a.v_head_stride;
            read_unit<X, WIDE>(p, x - hh * p.units, src, units[k]);
        }
        if (!waited) __syncthreads();
        waited = true;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int x = x0 + k * step;
            if (x >= total) break;
            const int hh = div_by(x, p.by_units), t = div_by(hh, p.by_heads), head = hh - t * p.heads, u = x - hh * p.units;
            const long long i = first + t, slot = slots[t];
            const int kvh = head - p.q_heads;
            if (kvh < 0) {
                X* dst = static_cast<X*>(a.q_out) + i * a.out_token_stride + head * a.out_head_stride;
                write_unit<X, X, WIDE>(p, u, true, slot == -2, units[k], dst, cos[t], sin[t]);
            } else if (slot >= 0) {
                const bool is_v = kvh >= p.pg.n_kv_heads;
                KV* dst = static_cast<KV*>(is_v ? p.pg.v : p.pg.k) + slot + (is_v ? kvh - p.pg.n_kv_heads : kvh) * p.pg.head_stride;
                write_unit<X, KV, WIDE>(p, u, !is_v, false, units[k], dst, cos[t], sin[t]);
            }
        }
    }
}

bool aligned(const void* p, long long s0, long long s1, size_t es) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 * es % 16 == 0 && s1 * es % 16 == 0;
}

template <typename X, typename KV>
void launch_for(Params& p, cudaStream_t stream) {
    const cudallm_append_args& a = p.a;
    const size_t es = sizeof(X);
    const bool wide = (a.interleaved ? a.rotary % 8 == 0 : p.pairs % 8 == 0) && aligned(a.k, a.k_token_stride, a.k_head_stride, es) &&
                      aligned(a.v, a.v_token_stride, a.v_head_stride, es) &&
                      (a.q == nullptr || (aligned(a.q, a.q_token_stride, a.q_head_stride, es) &&
                                          aligned(a.q_out, a.out_token_stride, a.out_head_stride, es)));
    const int dims = wide ? 8 : 1;
    p.pair_units = wide && a.interleaved ? a.rotary / 8 : p.pairs / dims;
    p.units = p.pair_units + (p.pg.head_dim - a.rotary) / dims;
    p.by_units = fast_div(p.units);
    p.by_heads = fast_div(p.heads);
    // Blocks of about three units a thread; where that leaves SMs idle, one token and its heads spread over several blocks.
    const int token_units = p.units * p.heads, sms = num_sms();
    p.tokens = std::max(1, std::min(kTokens, kBatch * kThreads / token_units));
    if (a.n_tokens / p.tokens < 2 * sms) p.tokens = std::max(1, std::min(p.tokens, a.n_tokens / (2 * sms)));
    const int blocks = (a.n_tokens + p.tokens - 1) / p.tokens;
    const int spread = blocks >= 2 * sms ? 1 : std::max(1, std::min((p.tokens * token_units + kThreads - 1) / kThreads, 2 * sms / blocks));
    launch_kernel(wide ? append_kernel<X, KV, true> : append_kernel<X, KV, false>, dim3(blocks, spread), dim3(kThreads), 0, stream, false, p);
}

template <typename X>
void launch_for(Params& p, cudaStream_t stream) {
    p.pg.kv_dtype == CUDALLM_KV_BF16 ? launch_for<X, __nv_bfloat16>(p, stream) : launch_for<X, __half>(p, stream);
}

}  // namespace

void launch_paged_append(const cudallm_pages& pg, const cudallm_append_args& a, cudaStream_t stream) {
    if (a.n_tokens == 0) return;
    Params p;
    p.pg = pg;
    p.a = a;
    p.q_heads = a.q != nullptr ? a.n_heads : 0;
    p.heads = p.q_heads + 2 * pg.n_kv_heads;
    p.pairs = a.rotary / 2;
    switch (a.x_dtype) {
        case CUDALLM_X_FP32: launch_for<float>(p, stream); break;
        case CUDALLM_X_FP16: launch_for<__half>(p, stream); break;
        default: launch_for<__nv_bfloat16>(p, stream); break;
    }
}

}  // namespace cudallm
