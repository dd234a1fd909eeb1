// Helpers shared by the paged-cache kernels: element conversion, division by a constant of the launch.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace cudallm {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// n / d for 0 <= n < 2^31 as a multiplication.
struct FastDiv {
    unsigned mul, shift;
};
inline FastDiv fast_div(int d) {
    unsigned s = 0;
    while ((1u << s) < static_cast<unsigned>(d)) ++s;
    return {static_cast<unsigned>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ __forceinline__ int div_by(int n, FastDiv f) {
    return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(n)) * f.mul) >> f.shift);
}

}  // namespace cudallm
