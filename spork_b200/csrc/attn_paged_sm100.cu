// Attention of one new token per request over a paged key-value cache, for sm_100a.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <math.h>
#include <stdint.h>

#include "../../include/spork_b200.h"
#include "device_state.h"
#include "paged_sm100.h"

namespace spork {
namespace attn_paged_sm100 {

using namespace spork::paged_sm100;

constexpr int kWarps = 4;

// One block per request and query head; a warp takes every fourth key, its lanes the head dimension.  Each warp keeps the
// running maximum and sum of its own keys; they are joined at the end.
template <int D, typename T, typename Q>
__global__ void __launch_bounds__(kWarps * 32) attn_paged_kernel(const spork_attn_paged_args a)
{
    constexpr int kPer = D / 32;
    __shared__ float part_m[kWarps], part_l[kWarps], part_o[kWarps][D];
    const int h = blockIdx.x, r = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const spork_paged_cache& c = a.cache;
    const int kv = h / (a.heads / c.kv_heads);
    const int64_t len = a.lengths[r];
    bool bad = len < 0 || len > (int64_t)a.max_blocks * c.page_size;
    float q[kPer], o[kPer] = {}, m = -INFINITY, l = 0.0f;
    for (int i = 0; i < kPer; ++i) {
        q[i] = to_f32(static_cast<const Q*>(a.q)[r * a.q_request_stride + h * a.q_head_stride + lane * kPer + i]) * a.scale;
    }
    for (int64_t t = warp; t < len && !bad; t += kWarps) {
        const int32_t page = a.block_table[r * a.table_stride + t / c.page_size];
        if (page < 0 || page >= c.num_pages) {
            bad = true;
            break;
        }
        const int64_t row = t % c.page_size;
        const T* k = static_cast<const T*>(c.k) + page * c.k_strides[0] + kv * c.k_strides[1] + row * c.k_strides[2];
        const T* v = static_cast<const T*>(c.v) + page * c.v_strides[0] + kv * c.v_strides[1] + row * c.v_strides[2];
        float s = 0.0f;
        for (int i = 0; i < kPer; ++i) {
            s += q[i] * to_f32(k[lane * kPer + i]);
        }
        for (int d = 16; d > 0; d /= 2) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        }
        const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.0f : m_new;
        const float down = __expf(m - base), p = __expf(s - base);
        l = l * down + p;
        for (int i = 0; i < kPer; ++i) {
            o[i] = o[i] * down + p * to_f32(v[lane * kPer + i]);
        }
        m = m_new;
    }
    part_m[warp] = m;
    part_l[warp] = bad ? NAN : l;
    for (int i = 0; i < kPer; ++i) {
        part_o[warp][lane * kPer + i] = o[i];
    }
    __syncthreads();
    float most = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
        most = fmaxf(most, part_m[w]);
    }
    const float base = most == -INFINITY ? 0.0f : most;
    for (int w = 0; w < kWarps; ++w) {
        sum += part_l[w] * __expf(part_m[w] - base);
    }
    for (int d = threadIdx.x; d < D; d += kWarps * 32) {
        float v = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            v += part_o[w][d] * __expf(part_m[w] - base);
        }
        static_cast<T*>(a.o)[((int64_t)r * a.heads + h) * D + d] = from_f32<T>(len == 0 ? 0.0f : v / sum);
    }
    if (a.lse && threadIdx.x == 0) {
        a.lse[(int64_t)r * a.heads + h] = base + logf(sum);
    }
}

template <int D, typename T, typename Q>
static int launch(const spork_attn_paged_args& a, cudaStream_t stream)
{
    attn_paged_kernel<D, T, Q><<<dim3(a.heads, a.requests), kWarps * 32, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

template <int D, typename T>
static int launch_q(const spork_attn_paged_args& a, cudaStream_t stream)
{
    return a.q_type == SPORK_TYPE_F32 ? launch<D, T, float>(a, stream) : launch<D, T, T>(a, stream);
}

}  // namespace attn_paged_sm100
}  // namespace spork

extern "C" int spork_attn_sm100_paged_supports(int heads, int kv_heads, int head_dim, int page_size)
{
    return (heads >= 0 && kv_heads > 0 && heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128) &&
            (page_size == 8 || page_size == 16 || page_size == 32 || (page_size > 0 && page_size % 64 == 0)))
               ? 1
               : 0;
}

extern "C" int64_t spork_attn_sm100_paged_workspace(int heads, int kv_heads, int head_dim)
{
    if (!spork_attn_sm100_paged_supports(heads, kv_heads, head_dim, 8)) {
        return -(int64_t)SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    return 0;
}

extern "C" int spork_attn_sm100_paged(const spork_attn_paged_args* args, void* stream)
{
    if (!args) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    const spork_attn_paged_args& a = *args;
    const spork_paged_cache& c = a.cache;
    if (a.requests < 0 || a.max_blocks < 0 || (a.requests > 1 && a.table_stride < a.max_blocks) ||
        !spork_attn_sm100_paged_supports(a.heads, c.kv_heads, c.head_dim, c.page_size)) {
        return SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    const int rc = spork::paged_sm100::check_cache(c);
    if (rc) {
        return rc;
    }
    // TMA reads rows of the cache: addresses and strides on 16 bytes (the strides of dimensions with one element do not count)
    auto aligned16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    const int64_t sizes[3] = {c.num_pages, c.kv_heads, c.page_size};
    for (int i = 0; i < 3; ++i) {
        if (sizes[i] > 1 && ((c.k_strides[i] & 7) || (c.v_strides[i] & 7))) {
            return SPORK_ERR_BAD_ARGUMENT;
        }
    }
    if (!aligned16(c.k) || !aligned16(c.v) || (a.q_type != c.type && a.q_type != SPORK_TYPE_F32) || !(a.scale > 0.0f) ||
        !(a.scale <= 3.4028235e38f)) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    if (a.requests == 0 || a.heads == 0) {
        return 0;
    }
    const uintptr_t q_elem = a.q_type == SPORK_TYPE_F32 ? 4 : 2;
    if (!a.q || !a.lengths || !a.o || (a.max_blocks > 0 && !a.block_table) || !aligned16(a.o) ||
        (reinterpret_cast<uintptr_t>(a.q) % q_elem) || (reinterpret_cast<uintptr_t>(a.block_table) & 3u) ||
        (reinterpret_cast<uintptr_t>(a.lengths) & 3u) || (reinterpret_cast<uintptr_t>(a.lse) & 3u) || !aligned16(a.workspace)) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    if (a.requests > 65535) {
        return SPORK_ERR_TOO_LARGE;
    }
    spork::DeviceState* dev = nullptr;
    const int rc2 = spork::current_device_state(&dev);
    if (rc2) {
        return rc2;
    }
    using namespace spork::attn_paged_sm100;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c.type == SPORK_TYPE_F16) {
        return c.head_dim == 64 ? launch_q<64, __half>(a, s) : launch_q<128, __half>(a, s);
    }
    return c.head_dim == 64 ? launch_q<64, __nv_bfloat16>(a, s) : launch_q<128, __nv_bfloat16>(a, s);
}
