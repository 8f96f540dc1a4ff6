// The paged key-value cache's bookkeeping for sm_100a: block tables and slot maps from request lengths, and new keys and
// values written into their slots.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>
#include <stdint.h>

#include "../../include/spork_b200.h"
#include "device_state.h"
#include "paged_sm100.h"
#include "ptx_sm100.cuh"

namespace spork {
namespace paged_sm100 {

using namespace spork::ptx;

// ------------------------------------------------------------------ block tables and slot maps
//
// Two sums over the requests say where each one's tokens lie in the slot map and which of the free pages it gets.  The
// list is short (it is one entry per request) and everything else depends on it, so every block takes both sums over all
// requests for itself, keeps them in shared memory, and then fills its share of the slot map and of the new table
// entries, finding the request of a token or page by bisection: one launch, and blocks that do not wait for one another.
// A decoding step is bound by the latency of one dependent chain (lengths, sums, page, slot); a queue of prompts by
// its slot map and the sums.  Measured: 256 decoding requests 4.5 us a launch; 2048 prompts of 1..1024 tokens (1.04 M in all)
// 10.6 to 11.0 us, 0.8 TB/s of what it has to read and write; 2048 of 1..128 tokens, the same sums with an eighth of the map,
// 6.3 us; 1024 of 1..1024 tokens 7.4 us.

constexpr int kTableThreads = 1024;
constexpr uint32_t kMost = 0x7FFFFFFF;

// Sums are kept at 2^31 - 1 once they are beyond it (such sums may be taken in any order), and so fit 32 bits throughout.
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return a + b < kMost ? a + b : kMost; }

// Sum over the threads of the block before this one; `total` receives the block's.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t& total)
{
    static_assert(kTableThreads == 32 * 32, "a lane for each warp's sum");
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    auto warp_scan = [&](uint32_t x) {
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t w = __shfl_up_sync(0xFFFFFFFFu, x, d);
            x = lane >= d ? plus(x, w) : x;
        }
        return x;
    };
    v = warp_scan(v);
    if (lane == 31) {
        warp_sums[warp] = v;
    }
    __syncthreads();
    const uint32_t sums = warp_scan(warp_sums[lane]);
    total = __shfl_sync(0xFFFFFFFFu, sums, 31);
    const uint32_t warps = __shfl_sync(0xFFFFFFFFu, sums, warp > 0 ? warp - 1 : 0);
    const uint32_t lanes = __shfl_up_sync(0xFFFFFFFFu, v, 1);
    return plus(warp > 0 ? warps : 0, lane > 0 ? lanes : 0);
}

// Tokens to pages: a shift where the page size is a power of two.
struct Pages {
    uint32_t size;
    int shift;  // -1: none
    __device__ __forceinline__ uint32_t of(uint32_t token) const { return shift >= 0 ? token >> shift : token / size; }
    // of 0 .. 2^31 - 1 tokens
    __device__ __forceinline__ uint32_t for_tokens(uint32_t tokens) const { return tokens > 0 ? of(tokens - 1) + 1 : 0; }
};

// Numbers of the requests in shared memory, one left out after every 32: threads that each walk through requests of their
// own then meet in no bank, whatever their share.
struct PerRequest {
    int32_t* at;
    __device__ __forceinline__ int32_t& operator[](int r) const { return at[r + (r >> 5)]; }
    static __host__ __device__ __forceinline__ int space(int requests) { return requests + (requests >> 5); }
};

// Last of the n ascending entries that is at most v (the first one is).
__device__ __forceinline__ int last_at_most(const PerRequest& entries, int n, int32_t v)
{
    int low = 0;
    while (n > 1) {
        const int half = n / 2;
        const bool up = entries[low + half] <= v;
        low = up ? low + half : low;
        n = up ? n - half : half;
    }
    return low;
}

// kPer: tokens that a thread takes one behind the other.
template <int kPer>
__global__ void __launch_bounds__(kTableThreads) tables_kernel(const spork_paged_tables_args a, const Pages page_of)
{
    // per request: first token in the slot map, first page among the granted ones, tokens held (-1: refused); until those are
    // known, the tokens that it adds and the pages that it needs (-1: its numbers cannot be)
    extern __shared__ int32_t per_request[];
    __shared__ uint32_t token_sums[kTableThreads / 32], page_sums[kTableThreads / 32];
    __shared__ uint32_t granted_pages;
    __shared__ int refused;
    const int n = a.requests;
    const int space = PerRequest::space(n);
    const PerRequest first_token{per_request}, first_page{per_request + space}, held_of{per_request + 2 * space};
    if (threadIdx.x == 0) {
        granted_pages = 0;
        refused = 0;
    }
    grid_dependency_wait();
    const int32_t used = *a.free_used;
    const uint32_t left = used >= 0 && used <= a.free_count ? a.free_count - used : 0;
    for (int r = threadIdx.x; r < n; r += kTableThreads) {
        held_of[r] = a.lengths[r];
        first_token[r] = a.new_tokens[r];
    }
    __syncthreads();
    // a thread's requests lie side by side, and nobody else looks at them before the sums are there
    const int chunk = (n + kTableThreads - 1) / kTableThreads;
    const int r0 = (int)threadIdx.x * chunk < n ? (int)threadIdx.x * chunk : n, r1 = r0 + chunk < n ? r0 + chunk : n;
    const int64_t row_tokens = (int64_t)a.max_blocks * a.page_size;
    const uint32_t capacity = row_tokens < kMost ? (uint32_t)row_tokens : kMost;
    const uint32_t room = (uint32_t)a.max_tokens;

    uint32_t mine = 0, tokens, pages;
    for (int r = r0; r < r1; ++r) {
        mine = plus(mine, first_token[r] > 0 ? first_token[r] : 0);
    }
    const uint32_t token0 = block_scan(mine, token_sums, tokens);
    uint32_t token = token0;
    mine = 0;
    for (int r = r0; r < r1; ++r) {
        const int32_t held = held_of[r], added = first_token[r];
        const uint32_t adds = added > 0 ? added : 0;
        token = plus(token, adds);
        const bool sound = held >= 0 && added >= 0 && (adds == 0 || token <= room) && (uint32_t)held + adds <= capacity;
        const uint32_t need = sound ? page_of.for_tokens(held + adds) - page_of.for_tokens(held) : 0;
        first_token[r] = adds;
        first_page[r] = sound ? (int32_t)need : -1;
        mine = plus(mine, need);
    }
    uint32_t page = block_scan(mine, page_sums, pages);
    token = token0;
    uint32_t most = 0;
    int not_granted = 0;
    for (int r = r0; r < r1; ++r) {
        const uint32_t adds = first_token[r], need = first_page[r] > 0 ? first_page[r] : 0;
        const uint32_t until = plus(page, need);
        const bool granted = first_page[r] >= 0 && (need == 0 || until <= left);
        const int32_t held = held_of[r];
        first_token[r] = (int32_t)token;
        first_page[r] = (int32_t)page;
        held_of[r] = granted ? held : -1;
        if (blockIdx.x == 0) {
            a.offsets[r] = (int32_t)token;
            a.lengths_after[r] = granted ? held + (int32_t)adds : held;
        }
        token = plus(token, adds);
        page = until;
        // what is granted ends where the last granted request with pages does
        most = granted && need > 0 ? until : most;
        not_granted += granted ? 0 : 1;
    }
    if (most > 0) {
        atomicMax(&granted_pages, most);
    }
    if (not_granted > 0) {
        atomicAdd(&refused, not_granted);
    }
    __syncthreads();

    // (not at the begin: blocks of the next launch that come so early slow the sums down, 16.4 us instead of 10.6 for the maps
    // of 2048 prompts in a stream of such launches; at the end it was 13.0)
    grid_launch_dependents();
    const int granted = (int)granted_pages;
    const int stride = gridDim.x * kTableThreads, at = blockIdx.x * kTableThreads + threadIdx.x;
    if (at == 0) {
        a.offsets[n] = (int32_t)tokens;
        a.info[0] = used + granted;
        a.info[1] = (int32_t)tokens;
        a.info[2] = refused;
        a.info[3] = (int32_t)pages;
    }
    for (uint32_t j = at; j < (uint32_t)granted; j += stride) {  // (unsigned: one step past 2^31 - 1 pages is still a number)
        const int i = (int)j;
        const int r = last_at_most(first_page, n, i);
        const uint32_t old = page_of.for_tokens(held_of[r]);
        a.block_table[r * a.table_stride + old + (i - first_page[r])] = a.free_pages[used + i];
    }
    for (int64_t t0 = (int64_t)at * kPer; t0 < a.max_tokens; t0 += (int64_t)stride * kPer) {
        int64_t slot[kPer];
        int r = t0 < tokens ? last_at_most(first_token, n, (int32_t)t0) : 0, last_r = -1, of = 0;
        uint32_t last_block = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const int64_t t = t0 + j;
            slot[j] = -1;
            if (t < tokens && t < a.max_tokens) {
                while (j > 0 && r + 1 < n && first_token[r + 1] <= t) {
                    ++r;
                }
                const int32_t held = held_of[r];
                if (held >= 0) {
                    const uint32_t place = (uint32_t)held + (uint32_t)(t - first_token[r]);
                    const uint32_t block = page_of.of(place);
                    if (kPer == 1 || r != last_r || block != last_block) {
                        const uint32_t old = page_of.for_tokens(held);
                        of = block < old ? a.block_table[r * a.table_stride + block]
                                         : a.free_pages[used + first_page[r] + (int)(block - old)];
                        last_r = r;
                        last_block = block;
                    }
                    slot[j] = of >= 0 ? (int64_t)of * page_of.size + (place - block * page_of.size) : -1;
                }
            }
        }
        if (kPer % 2 == 0 && t0 + kPer <= a.max_tokens && (reinterpret_cast<uintptr_t>(a.slots) & 15u) == 0) {
#pragma unroll
            for (int j = 0; j < kPer / 2; ++j) {
                reinterpret_cast<longlong2*>(a.slots + t0)[j] = make_longlong2(slot[2 * j], slot[kPer > 1 ? 2 * j + 1 : 0]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if (t0 + j < a.max_tokens) {
                    a.slots[t0 + j] = slot[j];
                }
            }
        }
    }
}

// ------------------------------------------------------------------ keys and values into their slots
//
// Bound by HBM: every element is read once and written once, 16 bytes of the cache at a time where pointers and strides
// allow it.  A thread keeps its place in a token's row (which half, head, column) and takes it for kTokens tokens, whose
// slots and elements it asks for before it needs the first one.  Measured: 16384 fp32 rows of 8 heads of 128 into bf16, 201 MB
// in 31.7 us, 97 % of the measured copy rate.

constexpr int kStoreThreads = 256;

template <typename T>
__device__ __forceinline__ void load_elements(const T* p, T (&x)[1]) { x[0] = *p; }
template <typename T>
__device__ __forceinline__ void load_elements(const T* p, T (&x)[8])
{
    const uint4* from = reinterpret_cast<const uint4*>(p);
    uint4* to = reinterpret_cast<uint4*>(x);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        to[i] = from[i];  // (no read-only load: the kernel before this one may still have been writing when this one began)
    }
}

template <typename Dst, typename Src>
__device__ __forceinline__ void store_elements(Dst* p, const Src (&x)[1]) { *p = round_to<Dst>(x[0]); }
template <typename Dst, typename Src>
__device__ __forceinline__ void store_elements(Dst* p, const Src (&x)[8])
{
    uint4 v;
    Dst* y = reinterpret_cast<Dst*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = round_to<Dst>(x[i]);
    }
    *reinterpret_cast<uint4*>(p) = v;
}

struct StoreShape {
    int items, per_head;  // pieces of a token's keys and values together, and of one head
    int rows;             // tokens that a block takes side by side
};

template <typename Src, typename Dst, int kElems, int kTokens>
__global__ void __launch_bounds__(kStoreThreads) store_kernel(const spork_paged_store_args a, const StoreShape shape)
{
    static_assert(kElems == 8 || kElems == 1, "16 bytes of the cache, or one element");
    const spork_paged_cache& c = a.cache;
    const int64_t slots = (int64_t)c.num_pages * c.page_size;
    grid_dependency_wait();
    grid_launch_dependents();
    for (int i = threadIdx.x; i < shape.items * shape.rows; i += kStoreThreads) {
        const int row = i / shape.items, half = shape.items / 2;
        int item = i - row * shape.items;
        const bool value = item >= half;
        item -= value ? half : 0;
        const int h = item / shape.per_head, d = (item - h * shape.per_head) * kElems;
        const int64_t token_stride = value ? a.v_token_stride : a.k_token_stride;
        const Src* src = static_cast<const Src*>(value ? a.v : a.k) + h * (value ? a.v_head_stride : a.k_head_stride) + d;
        const int64_t* strides = value ? c.v_strides : c.k_strides;
        const int64_t page_stride = strides[0], row_stride = strides[2];
        Dst* dst = static_cast<Dst*>(value ? c.v : c.k) + h * strides[1] + d;
        const int64_t t0 = (int64_t)blockIdx.x * (shape.rows * kTokens) + row;
        int64_t slot[kTokens];
        alignas(16) Src x[kTokens][kElems];
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
            const int64_t t = t0 + j * shape.rows;
            slot[j] = t < a.tokens ? a.slots[t] : -1;
        }
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
            const int64_t t = t0 + j * shape.rows;
            if (t < a.tokens) {
                load_elements(src + t * token_stride, x[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
            if (slot[j] >= 0 && slot[j] < slots) {
                const int64_t page = slots <= 0x7FFFFFFF ? (uint32_t)slot[j] / (uint32_t)c.page_size : slot[j] / c.page_size;
                store_elements(dst + page * page_stride + (slot[j] - page * c.page_size) * row_stride, x[j]);
            }
        }
    }
}

// A launch that may begin while the kernel before it in the stream is finishing (the kernels wait for it themselves).
template <typename... Params, typename... Args>
static int launch(void (*kernel)(Params...), unsigned blocks, int threads, size_t smem, cudaStream_t stream, const Args&... args)
{
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kPer>
static int launch_tables(const spork_paged_tables_args& a, DeviceState& dev, unsigned blocks, cudaStream_t stream)
{
    const size_t smem = (size_t)PerRequest::space(a.requests) * 3 * sizeof(int32_t);
    if (smem > 40 * 1024) {  // beyond what a kernel gets unasked (its static arrays included)
        static std::once_flag once[kMaxDevices];
        static cudaError_t err[kMaxDevices];
        std::call_once(once[dev.ordinal], [&] {
            err[dev.ordinal] = cudaFuncSetAttribute(tables_kernel<kPer>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                    PerRequest::space(SPORK_PAGED_MAX_REQUESTS) * 3 * (int)sizeof(int32_t));
        });
        if (err[dev.ordinal] != cudaSuccess) {
            return (int)err[dev.ordinal];
        }
    }
    const uint32_t size = (uint32_t)a.page_size;
    return launch(tables_kernel<kPer>, blocks, kTableThreads, smem, stream, a,
                  Pages{size, (size & (size - 1)) == 0 ? __builtin_ctz(size) : -1});
}

static int launch_tables(const spork_paged_tables_args& a, DeviceState& dev, cudaStream_t stream)
{
    // One token to a thread while a block on every SM holds them all: the page numbers of decoding requests are then
    // looked up side by side.  Beyond that four, which mostly are one request's and in one page.  us with one / with four:
    // 256 decoding requests 4.5 / 6.1, 4096 decoding requests 8.7 / 11.5, 2048 prompts of 1..1024 tokens 12.9 / 10.9.
    const int64_t most = dev.sm_count, wanted = (a.max_tokens + kTableThreads - 1) / kTableThreads;
    if (wanted <= most) {
        return launch_tables<1>(a, dev, (unsigned)(wanted < 1 ? 1 : wanted), stream);
    }
    return launch_tables<4>(a, dev, (unsigned)(wanted < 4 * most ? (wanted + 3) / 4 : most), stream);
}

template <typename Src, typename Dst, int kElems>
static int launch_store(const spork_paged_store_args& a, DeviceState& dev, cudaStream_t stream)
{
    const spork_paged_cache& c = a.cache;
    StoreShape shape;
    shape.per_head = c.head_dim / kElems;
    shape.items = 2 * c.kv_heads * shape.per_head;
    shape.rows = shape.items < kStoreThreads ? kStoreThreads / shape.items : 1;
    // Four tokens to a thread keep more loads under way, but leave SMs idle where there are few tokens: four once that is
    // three blocks to an SM.  fp32 rows of 8 heads of 128 into bf16, us with one / with four: 64 rows 1.75 / 2.32, 1024 rows
    // 3.26 / 3.59, 2048 rows 5.02 / 4.40, 4096 rows 9.57 / 8.50, 16384 rows 35.6 / 31.7.
    const int64_t blocks = (a.tokens + shape.rows - 1) / shape.rows;
    if (blocks >= 4 * 3 * (int64_t)dev.sm_count) {
        return launch(store_kernel<Src, Dst, kElems, 4>, (unsigned)((blocks + 3) / 4), kStoreThreads, 0, stream, a, shape);
    }
    return launch(store_kernel<Src, Dst, kElems, 1>, (unsigned)blocks, kStoreThreads, 0, stream, a, shape);
}

// Whether all pieces of 8 elements lie on the boundaries that the wide loads and stores need.  (16384 fp32 rows of 8 heads
// of 128 into bf16: 31.7 us in pieces of 8, 109 us one element at a time.)
static bool store_aligned(const spork_paged_store_args& a)
{
    const spork_paged_cache& c = a.cache;
    const int64_t src = a.src_type == SPORK_TYPE_F32 ? 4 : 8;  // elements of 16 bytes
    int64_t any = c.head_dim & 7;
    for (const void* p : {(const void*)c.k, (const void*)c.v, a.k, a.v}) {
        any |= (int64_t)(reinterpret_cast<uintptr_t>(p) & 15u);
    }
    const int64_t sizes[3] = {c.num_pages, c.kv_heads, c.page_size};
    for (int i = 0; i < 3; ++i) {
        any |= sizes[i] > 1 ? (c.k_strides[i] | c.v_strides[i]) & 7 : 0;
    }
    any |= a.tokens > 1 ? (a.k_token_stride | a.v_token_stride) & (src - 1) : 0;
    any |= c.kv_heads > 1 ? (a.k_head_stride | a.v_head_stride) & (src - 1) : 0;
    return any == 0;
}

template <typename Src, typename Dst>
static int launch_store_types(const spork_paged_store_args& a, DeviceState& dev, cudaStream_t stream)
{
    return store_aligned(a) ? launch_store<Src, Dst, 8>(a, dev, stream) : launch_store<Src, Dst, 1>(a, dev, stream);
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
    if (a.requests > SPORK_PAGED_MAX_REQUESTS || a.max_tokens >= 0x7FFFFFFF || a.free_count == 0x7FFFFFFF) {
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
    return launch_tables(a, *dev, static_cast<cudaStream_t>(stream));
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
    // a token's pieces are counted in 32 bits, with a block's step behind the last one
    const int64_t pieces = 2 * (int64_t)a.cache.kv_heads * (a.cache.head_dim / (spork::paged_sm100::store_aligned(a) ? 8 : 1));
    if (pieces > 0x7FFFFFFF - spork::paged_sm100::kStoreThreads) {
        return SPORK_ERR_TOO_LARGE;
    }
    spork::DeviceState* dev = nullptr;
    const int rc2 = spork::current_device_state(&dev);
    if (rc2) {
        return rc2;
    }
    using namespace spork::paged_sm100;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.cache.type == SPORK_TYPE_F16) {
        return a.src_type == SPORK_TYPE_F32 ? launch_store_types<float, __half>(a, *dev, s)
                                            : launch_store_types<__half, __half>(a, *dev, s);
    }
    return a.src_type == SPORK_TYPE_F32 ? launch_store_types<float, __nv_bfloat16>(a, *dev, s)
                                        : launch_store_types<__nv_bfloat16, __nv_bfloat16>(a, *dev, s);
}
