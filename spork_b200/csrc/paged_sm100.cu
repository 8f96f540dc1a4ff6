// The paged key-value cache's bookkeeping for sm_100a: block tables and slot maps from request lengths, and new keys and
// values written into their slots.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdint.h>

#include "../../include/spork_b200.h"
#include "device_state.h"
#include "paged_sm100.h"

namespace spork {
namespace paged_sm100 {

constexpr int kTableThreads = 1024;

__device__ __forceinline__ int32_t saturate(int64_t v) { return v > 0x7FFFFFFF ? 0x7FFFFFFF : (int32_t)v; }

// Inclusive sum over the block; `total` receives the block's.
__device__ int64_t block_scan(int64_t v, int64_t* warp_sums, int64_t& total)
{
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int d = 1; d < 32; d *= 2) {
        const int64_t w = __shfl_up_sync(0xFFFFFFFFu, v, d);
        v += lane >= d ? w : 0;
    }
    __syncthreads();
    if (lane == 31) {
        warp_sums[warp] = v;
    }
    __syncthreads();
    total = 0;
    int64_t before = 0;
    for (int w = 0; w < kTableThreads / 32; ++w) {
        before += w < warp ? warp_sums[w] : 0;
        total += warp_sums[w];
    }
    return before + v;
}

// One block; a thread per request, blocks of requests one after the other.
__global__ void __launch_bounds__(kTableThreads) tables_kernel(const spork_paged_tables_args a)
{
    __shared__ int64_t warp_sums[kTableThreads / 32];
    const int64_t page = a.page_size, capacity = (int64_t)a.max_blocks * page;
    const int64_t used = *a.free_used;
    const int64_t left = used >= 0 && used <= a.free_count ? a.free_count - used : 0;
    int64_t tokens = 0, pages = 0, granted_pages = 0, refused = 0;
    for (int r0 = 0; r0 < a.requests; r0 += kTableThreads) {
        const int r = r0 + (int)threadIdx.x;
        const bool mine = r < a.requests;
        const int64_t held = mine ? a.lengths[r] : 0, added = mine ? a.new_tokens[r] : 0;
        const int64_t adds = added > 0 ? added : 0;
        int64_t total;
        const int64_t ends = tokens + block_scan(adds, warp_sums, total);
        tokens += total;
        const bool sound = held >= 0 && added >= 0 && (adds == 0 || ends <= a.max_tokens) && held + adds <= capacity;
        const int64_t old = sound ? (held + page - 1) / page : 0;
        const int64_t need = sound ? (held + adds + page - 1) / page - old : 0;
        const int64_t until = pages + block_scan(need, warp_sums, total);
        pages += total;
        const bool granted = sound && (need == 0 || until <= left);
        block_scan(granted ? need : 0, warp_sums, total);
        granted_pages += total;
        block_scan(granted || !mine ? 0 : 1, warp_sums, total);
        refused += total;
        if (mine) {
            const int32_t* from = a.free_pages + used + (until - need);
            int32_t* row = a.block_table + r * a.table_stride;
            a.offsets[r] = saturate(ends - adds);
            a.lengths_after[r] = granted ? (int32_t)(held + adds) : (int32_t)held;
            for (int64_t i = 0; i < need && granted; ++i) {
                row[old + i] = from[i];
            }
            for (int64_t i = 0; i < adds && ends - adds + i < a.max_tokens; ++i) {
                const int64_t at = held + i;
                const int64_t of = granted ? row[at / page] : -1;
                a.slots[ends - adds + i] = of >= 0 ? of * page + at % page : -1;
            }
        }
    }
    for (int64_t t = tokens + threadIdx.x; t < a.max_tokens; t += kTableThreads) {
        a.slots[t] = -1;
    }
    if (threadIdx.x == 0) {
        a.offsets[a.requests] = saturate(tokens);
        a.info[0] = saturate(used + granted_pages);
        a.info[1] = saturate(tokens);
        a.info[2] = (int32_t)refused;
        a.info[3] = saturate(pages);
    }
}

// One block per token.
template <typename Src, typename Dst>
__global__ void store_kernel(const spork_paged_store_args a)
{
    const int64_t t = blockIdx.x;
    const int64_t slot = a.slots[t];
    const spork_paged_cache& c = a.cache;
    if (slot < 0 || slot >= (int64_t)c.num_pages * c.page_size) {
        return;
    }
    const int64_t page = slot / c.page_size, row = slot % c.page_size;
    for (int i = threadIdx.x; i < c.kv_heads * c.head_dim; i += blockDim.x) {
        const int h = i / c.head_dim, d = i % c.head_dim;
        const Src k = static_cast<const Src*>(a.k)[t * a.k_token_stride + h * a.k_head_stride + d];
        const Src v = static_cast<const Src*>(a.v)[t * a.v_token_stride + h * a.v_head_stride + d];
        static_cast<Dst*>(c.k)[page * c.k_strides[0] + h * c.k_strides[1] + row * c.k_strides[2] + d] = round_to<Dst>(k);
        static_cast<Dst*>(c.v)[page * c.v_strides[0] + h * c.v_strides[1] + row * c.v_strides[2] + d] = round_to<Dst>(v);
    }
}

template <typename Src, typename Dst>
static int launch_store(const spork_paged_store_args& a, cudaStream_t stream)
{
    store_kernel<Src, Dst><<<(unsigned)a.tokens, 256, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

}  // namespace paged_sm100
}  // namespace spork

// Whether [a, a + na) and [b, b + nb) share a byte.
static bool overlap(const void* a, int64_t na, const void* b, int64_t nb)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

extern "C" int spork_paged_sm100_tables(const spork_paged_tables_args* args, void* stream)
{
    if (!args) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    const spork_paged_tables_args& a = *args;
    if (a.requests < 0 || a.max_blocks < 0 || a.page_size < 1 || a.free_count < 0 || a.max_tokens < 0 ||
        (a.requests > 1 && a.table_stride < a.max_blocks)) {
        return SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    if (a.requests > SPORK_PAGED_MAX_REQUESTS || a.max_tokens > 0x7FFFFFFF) {
        return SPORK_ERR_TOO_LARGE;
    }
    struct Span {
        const void* p;
        int64_t bytes;
        uintptr_t align;
    };
    const int64_t n = a.requests;
    const Span spans[9] = {{a.lengths, 4 * n, 4},
                           {a.new_tokens, 4 * n, 4},
                           {a.free_pages, 4 * (int64_t)a.free_count, 4},
                           {a.free_used, 4, 4},
                           {a.block_table, n > 0 && a.max_blocks > 0 ? 4 * ((n - 1) * a.table_stride + a.max_blocks) : 0, 4},
                           {a.slots, 8 * a.max_tokens, 8},
                           {a.offsets, 4 * (n + 1), 4},
                           {a.lengths_after, 4 * n, 4},
                           {a.info, 16, 4}};
    for (int i = 0; i < 9; ++i) {
        if ((spans[i].bytes > 0 && !spans[i].p) || (reinterpret_cast<uintptr_t>(spans[i].p) & (spans[i].align - 1))) {
            return SPORK_ERR_BAD_ARGUMENT;
        }
        for (int j = 4; j < 9; ++j) {  // an output and anything else
            if (j != i && overlap(spans[i].p, spans[i].bytes, spans[j].p, spans[j].bytes)) {
                return SPORK_ERR_BAD_ARGUMENT;
            }
        }
    }
    spork::DeviceState* dev = nullptr;
    const int rc = spork::current_device_state(&dev);
    if (rc) {
        return rc;
    }
    using namespace spork::paged_sm100;
    tables_kernel<<<1, kTableThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return (int)cudaGetLastError();
}

extern "C" int spork_paged_sm100_store(const spork_paged_store_args* args, void* stream)
{
    if (!args) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    const spork_paged_store_args& a = *args;
    const int rc = spork::paged_sm100::check_cache(a.cache);
    if (rc) {
        return rc;
    }
    if (a.tokens < 0) {
        return SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    if (a.tokens > 0x7FFFFFFF) {
        return SPORK_ERR_TOO_LARGE;
    }
    if (a.src_type != a.cache.type && a.src_type != SPORK_TYPE_F32) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    if (a.tokens == 0 || a.cache.kv_heads == 0 || a.cache.num_pages == 0) {
        return 0;
    }
    const uintptr_t elem = a.src_type == SPORK_TYPE_F32 ? 4 : 2;
    if (!a.k || !a.v || !a.slots || (reinterpret_cast<uintptr_t>(a.k) % elem) || (reinterpret_cast<uintptr_t>(a.v) % elem) ||
        (reinterpret_cast<uintptr_t>(a.slots) % 8)) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    spork::DeviceState* dev = nullptr;
    const int rc2 = spork::current_device_state(&dev);
    if (rc2) {
        return rc2;
    }
    using namespace spork::paged_sm100;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.cache.type == SPORK_TYPE_F16) {
        return a.src_type == SPORK_TYPE_F32 ? launch_store<float, __half>(a, s) : launch_store<__half, __half>(a, s);
    }
    return a.src_type == SPORK_TYPE_F32 ? launch_store<float, __nv_bfloat16>(a, s)
                                        : launch_store<__nv_bfloat16, __nv_bfloat16>(a, s);
}
