// What the paged cache's kernels share: element conversions and the checks of a cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/spork_b200.h"

namespace spork {
namespace paged_sm100 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Round to nearest even (the only rounding that a value takes on its way into the cache, or out as a result).
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A value in the cache's type: itself where it has that type already.
template <typename Dst, typename Src>
__device__ __forceinline__ Dst round_to(Src v) { return from_f32<Dst>(to_f32(v)); }
template <>
__device__ __forceinline__ __half round_to<__half, __half>(__half v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16, __nv_bfloat16>(__nv_bfloat16 v) { return v; }

// Geometry and pointers of a cache: 0 or an error code.  Rows, heads and pages may come in any order in memory, but no
// two elements at one place (a stride that is too small for what lies inside it).
inline int check_cache(const spork_paged_cache& c)
{
    if (c.num_pages < 0 || c.kv_heads < 0 || c.page_size < 1 || c.head_dim < 1) {
        return SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    if (c.type != SPORK_TYPE_F16 && c.type != SPORK_TYPE_BF16) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    if (c.num_pages == 0 || c.kv_heads == 0) {
        return 0;
    }
    if (!c.k || !c.v || (reinterpret_cast<uintptr_t>(c.k) & 1u) || (reinterpret_cast<uintptr_t>(c.v) & 1u)) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    const int64_t sizes[3] = {c.num_pages, c.kv_heads, c.page_size};
    for (const int64_t* strides : {c.k_strides, c.v_strides}) {
        // by ascending stride, each dimension has to step over all that the ones below it cover
        int order[3] = {0, 1, 2};
        for (int i = 0; i < 3; ++i) {
            for (int j = i + 1; j < 3; ++j) {
                if (strides[order[j]] < strides[order[i]]) {
                    const int t = order[i];
                    order[i] = order[j];
                    order[j] = t;
                }
            }
        }
        int64_t covered = c.head_dim;
        for (int i = 0; i < 3; ++i) {
            const int64_t n = sizes[order[i]], step = strides[order[i]];
            if (n <= 1) {
                continue;
            }
            if (step < covered || step > (int64_t)1 << 40) {
                return SPORK_ERR_BAD_ARGUMENT;
            }
            // places are counted in 64 bits, and no address space holds 2^57 bytes
            if (n - 1 > (((int64_t)1 << 56) - covered) / step) {
                return SPORK_ERR_TOO_LARGE;
            }
            covered += (n - 1) * step;
        }
    }
    return 0;
}

}  // namespace paged_sm100
}  // namespace spork
