// Rotary positions of new tokens, with the store of their keys and values to the pages of a cache.
//
//   (a, b) -> factor (a cos - b sin, b cos + a sin),  angle = fl32(position * inv_freq[j])
//
// Every input is read once and every output written once: HBM bounds it at many tokens, launch latency at few. A block
// takes one or more tokens, computes their cosines once for all heads, and its threads walk the heads in units of 8
// dims (16-byte accesses of 16-bit types): the two halves of 8 pairs, 4 interleaved pairs, or 8 dims that are copied.
// Where strides or sizes do not allow that, a unit is one pair or one dim, and the number of loads bounds it (16383 tokens of 48 heads x 128, bf16:
// 279 us with 60 dims rotated, 81 with 64).
//
// Measured (B200, graph replay): 16383 tokens of 48 heads x 128, bf16, 64 dims rotated interleaved, 81 us (5.0 TB/s); of 48 x 64, fp32 to
// fp16, in halves, 69 us (5.4 TB/s); 64 tokens of one step 2.9 us.
#include <algorithm>
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

constexpr int kThreads = 256;
constexpr int kTokens = 8;  // of a block at most

struct Params {
    cudallm_pages pg;
    cudallm_append_args a;
    int q_heads, heads;   // query heads; all heads of a token
    int tokens;           // of a block
    int pairs, pair_units, units;  // rotated pairs of a head; its units that rotate; all its units
};

// 8 values of a 16-byte (or two) word and back.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 (&raw)[sizeof(T) / 2], float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        memcpy(v, raw, 32);
    } else {
        const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                __half2 h;
                memcpy(&h, &w[i], 4);
                v[2 * i] = __low2float(h);
                v[2 * i + 1] = __high2float(h);
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                memcpy(&w[i], &h, 4);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                memcpy(&w[i], &h, 4);
            }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

// How heads are cut into units.
enum class Layout {
    kHalves,       // 8 pairs (j, j + n): two words of 8 dims; copied dims: one word
    kInterleaved,  // 4 pairs (2j, 2j + 1) or 8 copied dims: one word
    kSingle,       // one pair of either kind, or one copied dim
};

// What a thread does in every head: its dims from d0 on and, `other` dims further, its second part if it has one; the cosines and sines
// of the pairs that it rotates, if it does.
template <Layout L>
struct Job {
    static constexpr int kPairs = L == Layout::kHalves ? 8 : L == Layout::kInterleaved ? 4 : 1;
    int other;
    bool pair, two;
    float c[kPairs], s[kPairs];
};

// One unit as it is loaded.
template <typename X, Layout L>
struct Unit {
    static constexpr int kWords = L == Layout::kSingle ? 1 : sizeof(X) / 2;  // of 8 dims
    uint4 a[kWords], b[kWords];
    X one[2];

    __device__ __forceinline__ void load(const Job<L>& w, const X* src) {
        if constexpr (L == Layout::kSingle) {
            one[0] = src[0];
            if (w.two) one[1] = src[w.other];
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                a[i] = reinterpret_cast<const uint4*>(src)[i];
                if (L == Layout::kHalves && w.two) b[i] = reinterpret_cast<const uint4*>(src + w.other)[i];
            }
        }
    }

    // Rotated if `rotates`.
    template <typename Y>
    __device__ __forceinline__ void store(const Job<L>& w, bool rotates, Y* dst) const {
        rotates = rotates && w.pair;
        if constexpr (L == Layout::kSingle) {
            float v = as_float(one[0]), z = w.two ? as_float(one[1]) : 0.f;
            if (rotates) turn(v, z, w.c[0], w.s[0]);
            dst[0] = from_float<Y>(v);
            if (w.two) dst[w.other] = from_float<Y>(z);
        } else if (std::is_same_v<X, Y> && !rotates) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                reinterpret_cast<uint4*>(dst)[i] = a[i];
                if (L == Layout::kHalves && w.two) reinterpret_cast<uint4*>(dst + w.other)[i] = b[i];
            }
        } else {
            float v[8];
            unpack8<X>(a, v);
            if (L == Layout::kHalves && w.two) {
                float z[8];
                unpack8<X>(b, z);
                if (rotates) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) turn(v[i], z[i], w.c[i % Job<L>::kPairs], w.s[i % Job<L>::kPairs]);
                }
                store8(dst + w.other, z);
            }
            if (L == Layout::kInterleaved && rotates) {
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(v[2 * i], v[2 * i + 1], w.c[i % Job<L>::kPairs], w.s[i % Job<L>::kPairs]);
            }
            store8(dst, v);
        }
    }

    __device__ __forceinline__ void clear() {
        one[0] = one[1] = from_float<X>(0.f);
#pragma unroll
        for (int i = 0; i < kWords; ++i) a[i] = b[i] = make_uint4(0, 0, 0, 0);
    }
};

// Units of 8 pairs or of fp32 are loaded one at a time, others two at a time, by 4 (8 pairs) or 5 blocks on an SM. Measured on 16383 tokens
// of 48 heads (us; loads at a time and blocks): bf16 x 128, 64 rotated interleaved: 4 and 3 91, 2 and 5 81, 1 and 5 84; bf16 x 128 in halves:
// 2 and 3 80, 2 and 4 110 (spills), 1 and 4 80, 1 and 5 86; fp32 x 64 in halves: 2 and 3 109, 1 and 4 70, 1 and 5 85; interleaved: 1 and 4 73,
// 1 and 5 67.
template <typename X, Layout L>
constexpr bool one_load = L == Layout::kHalves || (L == Layout::kInterleaved && sizeof(X) == 4);

template <typename X, typename KV, Layout L>
__global__ void __launch_bounds__(kThreads, L == Layout::kHalves ? 4 : 5) append_kernel(const __grid_constant__ Params p) {
    constexpr int kItems = one_load<X, L> ? 1 : 2;  // heads of a thread whose loads are under way together
    __shared__ __align__(16) float cos[kTokens][128], sin[kTokens][128];
    __shared__ long long slots[kTokens];  // where the token's keys go; -1: nowhere, -2: padding
    const cudallm_append_args& a = p.a;
    grid_dep_wait();
    grid_dep_launch();
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
    // A thread has the same dims in all of its heads; at_once heads side by side, of several tokens where a token has fewer.
    // Units that rotate and units that are copied go to different warps.
    const int at_once = kThreads / p.units, turning = at_once * p.pair_units, copying = p.units - p.pair_units;
    const int place = static_cast<int>(threadIdx.x) - turning;
    const int u = place < 0 ? threadIdx.x % p.pair_units : copying > 0 ? p.pair_units + place % copying : p.units;
    const int r = place < 0 ? threadIdx.x / p.pair_units : copying > 0 ? place / copying : at_once;
    const int together = gridDim.y > 1 ? 1 : max(1, at_once / p.heads);  // tokens
    const int step = together > 1 ? p.heads : gridDim.y * at_once;
    const int h0 = together > 1 ? r % p.heads : blockIdx.y * at_once + r;  // the thread's first head
    int t0 = together > 1 ? r / p.heads : 0;
    if (t0 >= together || r >= at_once) t0 = tokens;
    Job<L> w;
    w.pair = u < p.pair_units;
    const int copied = 2 * p.pairs + (u - p.pair_units) * (L == Layout::kSingle ? 1 : 8);
    const int d0 = !w.pair ? copied : L != Layout::kSingle ? u * 8 : a.interleaved ? u * 2 : u;
    w.two = w.pair && L != Layout::kInterleaved;
    w.other = L == Layout::kSingle && a.interleaved ? 1 : p.pairs;
    const int kv = p.pg.n_kv_heads;
    __syncthreads();
#pragma unroll 1
    for (int hs = h0; hs < p.heads; hs += kItems * step) {
        // Up to kItems heads, the same ones of every token.
        const X* src[kItems];
        long long ahead[kItems];  // from a token's source to the next one's
        X* out[kItems];           // of queries
        KV* page[kItems];         // of keys and values: plus the token's slot
        bool rotates[kItems];
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
            const int h = hs + j * step, kh = h - p.q_heads, vh = kh - kv;
            out[j] = nullptr;
            page[j] = nullptr;
            rotates[j] = vh < 0;
            if (kh < 0) {
                ahead[j] = a.q_token_stride;
                src[j] = static_cast<const X*>(a.q) + h * a.q_head_stride;
                out[j] = static_cast<X*>(a.q_out) + (first + t0) * a.out_token_stride + h * a.out_head_stride + d0;
            } else if (vh < 0) {
                ahead[j] = a.k_token_stride;
                src[j] = static_cast<const X*>(a.k) + kh * a.k_head_stride;
                page[j] = static_cast<KV*>(p.pg.k) + kh * p.pg.head_stride + d0;
            } else {
                ahead[j] = a.v_token_stride;
                src[j] = static_cast<const X*>(a.v) + vh * a.v_head_stride;
                page[j] = static_cast<KV*>(p.pg.v) + vh * p.pg.head_stride + d0;
            }
            src[j] = vh < kv ? src[j] + (first + t0) * ahead[j] + d0 : nullptr;
            ahead[j] *= together;
        }
#pragma unroll 1
        for (int t = t0; t < tokens; t += together) {
            Unit<X, L> units[kItems];
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                if (src[j] == nullptr) break;
                units[j].load(w, src[j]);
                src[j] += ahead[j];
            }
            const long long slot = slots[t];
#pragma unroll
            for (int j = 0; j < Job<L>::kPairs; ++j) {
                w.c[j] = w.pair ? cos[t][u * Job<L>::kPairs + j] : 0.f;
                w.s[j] = w.pair ? sin[t][u * Job<L>::kPairs + j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                if (src[j] == nullptr) break;
                if (out[j] != nullptr) {
                    if (slot == -2) units[j].clear();
                    units[j].store(w, true, out[j]);
                    out[j] += together * a.out_token_stride;
                } else if (slot >= 0) {
                    units[j].store(w, rotates[j], page[j] + slot);
                }
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
    // Up to 8 tokens a block, since what a block sets up once costs as much as a dozen units of a thread; with fewer blocks than
    // fill the GPU four deep, fewer tokens; and with less than one token for each SM, a token's heads on several blocks.
    const int token_units = p.units * p.heads, sms = num_sms();
    p.tokens = std::max(1, std::min(kTokens, a.n_tokens / (4 * sms)));
    const int small = std::max(1, std::min(kTokens, kThreads / token_units));  // tokens that keep a block's threads busy
    if (p.tokens < small && a.n_tokens / small >= sms) p.tokens = small;
    const int blocks = (a.n_tokens + p.tokens - 1) / p.tokens;
    const int spread = blocks >= 2 * sms ? 1 : std::max(1, std::min((p.tokens * token_units + kThreads - 1) / kThreads, 2 * sms / blocks));
    auto kernel = !wide           ? append_kernel<X, KV, Layout::kSingle>
                  : a.interleaved ? append_kernel<X, KV, Layout::kInterleaved>
                                  : append_kernel<X, KV, Layout::kHalves>;
    launch_kernel(kernel, dim3(blocks, spread), dim3(kThreads), 0, stream, true, p);
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
