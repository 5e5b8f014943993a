// block_common.cuh -- pieces shared by the kernels of the block operators
// (helix_block.h): vector loads and stores of the supported types, the 8-bit
// groups' scale and rounding, and the launch helper.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../runtime/block_internal.h"

namespace hx {

// Largest of the magnitudes; NaN when one of them is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Largest of a >= 0 and two magnitudes, NaN as above.
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The scale of a group whose largest magnitude is amax, and its reciprocal,
// both within 2 ulp (an exact division takes as long as the rest of a group).
// The floor keeps the reciprocal finite for a group of zeros; max.NaN lets a
// NaN through.
__device__ __forceinline__ float group_scale(float amax, float* inv) {
    const float scale = max_nan(amax, 0x1p-100f) * (1.0f / 448.0f);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(*inv) : "f"(scale));
    return scale;
}

// Two values as e4m3, the first in the low byte; round to nearest even, NaN
// stays NaN.  Values are at most 448 in magnitude up to rounding of 1 / scale.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4)
        return v;
    else
        return __float2bfloat16_rn(v);
}

// Eight consecutive values of a 16-byte aligned address: as loaded, and as
// fp32.  Loading apart from unpacking lets a thread have all of its loads in
// flight before it looks at the first.
template <typename T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    f[4 * i + k] = __uint_as_float(w[k]);
                } else {  // a bf16 is the top half of its fp32
                    f[2 * k] = __uint_as_float(w[k] << 16);
                    f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                }
            }
        }
    }
};
__device__ __forceinline__ void st8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ uint32_t bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void st8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(bf16x2(v[0], v[1]), bf16x2(v[2], v[3]), bf16x2(v[4], v[5]), bf16x2(v[6], v[7]));
}

// Launch that reports its own error and no earlier one.
template <typename... K, typename... A>
inline int block_launch(void (*kernel)(K...), dim3 grid, dim3 block, size_t smem, void* stream, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...);
}

}  // namespace hx
