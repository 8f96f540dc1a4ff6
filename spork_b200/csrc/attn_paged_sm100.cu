// Attention of one new token per request over a paged key-value cache, for sm_100a:
//   o[r][h] = softmax(scale q[r][h] K^T) V over the keys that request r holds, key head h / (heads / kv_heads).
//
// Every key and value is read once and used by the few query heads that share it, so the kernel is bound by HBM; the
// products are small.  Work is cut along the cache: units of 64 keys (128 with a head dimension of 64: 32 KB of keys and
// values) of one (request, key head), all units in one list, request by request, and each block of the grid takes an
// equal run of that list, whatever the lengths (they are known on the device only).  A block joins what it computes of
// one (request, key head) and writes the result if it has all of it; otherwise a partial result (running maximum, sum,
// unnormalised output) goes to the workspace, and a second small kernel joins the parts in the order of the keys.  A
// block has at most two partial results: its first run and its last one.
//
// One warp copies the pages with TMA: the cache is a 5-dimensional tensor (64 elements, page rows, halves of the head
// dimension, heads, pages) with the strides that it has, so any order in memory is one tensor map; a box is a page's
// rows of one head (64 rows of it at most), swizzled for ldmatrix.  Page numbers come from the block table, and are
// checked before they are used.
//
// Four warps compute, each on keys of its own, with mma.m16n8k16.  Up to 8 query heads are rows 0-7 of the 16-row
// operand, and rows 8-15 hold what rounding to 16 bits left over: of q, if it is fp32, and of the softmax weights.  So
// both products are taken with about 22 (fp16) or 16 (bf16) bits of q and of the weights at no cost: the rows would have
// been empty, and the weights' rounding, the largest error of the usual scheme, is gone.  (tcgen05 would want 64 or 128
// rows and a trip through tensor memory for every unit; the warp instruction's rate is several times what the loads can
// feed.)  With 9 or more query heads to a key head the warps form 2 or 4 groups that share the unit, 8 heads each.
// Each warp runs its own online softmax.  Its maximum follows the scores lazily: only when one has grown by more than
// 2^8 over it are the row's lanes asked and the sums rescaled, so most units need no exchange between lanes at all.  The
// warps of a group are joined once per (request, key head), pairwise: a warp that has handed its sums over goes on.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <math.h>
#include <mutex>
#include <stdint.h>
#include <type_traits>

#include "../../include/spork_b200.h"
#include "device_state.h"
#include "paged_sm100.h"
#include "ptx_sm100.cuh"

namespace spork {
namespace attn_paged_sm100 {

using namespace spork::paged_sm100;
using namespace spork::ptx;

constexpr int kHeads = 8;          // query heads of a group of warps
// weights are 2^(x - max + 6), and max may be out of date by 8: up to 2^14, within fp16, whose small weights stay normal
constexpr float kShift = 6.0f, kSlack = 8.0f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxBlocks = 1024;   // blocks of a launch
constexpr int kComputeWarps = 4;
constexpr int kThreads = (kComputeWarps + 1) * 32;
constexpr int kBlocksPerSm = 2;
constexpr int kPairCost = 1;       // what a (request, key head) costs a block besides its units, in units
constexpr int kMaxRows = 64;       // rows of a TMA box
constexpr int kJoinThreads = 128;

// kGroups groups of warps share a unit, each with 8 query heads of its own.
template <int D, int kGroups>
struct Config {
    static constexpr int kTile = 8192 / D;                      // keys per unit
    static constexpr int kWarps = kComputeWarps / kGroups;      // warps of a group; each takes kTile / kWarps keys
    static constexpr int kKeys = kTile / kWarps;
    static constexpr int kChunk = kKeys < 32 ? kKeys : 32;      // taken at once
    static constexpr int kHalfUnit = kTile * D * 2;             // the keys (or values) of a unit, bytes
    static constexpr int kStageBytes = 2 * kHalfUnit;
    static constexpr int kStages = 3;
    static constexpr int kPadded = D + 8;                       // floats between the rows of the joining buffer: no bank conflicts
    static constexpr int kJoinFloats = kGroups * (kWarps - 1) * kHeads * kPadded;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kJoinFloats * 4;
};

struct Params {
    const void* q;
    const int32_t* table;
    const int32_t* lengths;
    void* o;
    float* lse;
    int64_t q_request_stride, q_head_stride, table_stride;
    int32_t requests, heads, kv_heads, group, head_units;  // group: query heads per key head; head_units: units along them
    int32_t max_blocks, num_pages, page_size, box_rows;
    float scale_log2e;
    bool q_pairs;  // two neighbouring elements of q may be read at once
    // workspace
    int4* joins;       // per block: {request (-1: none), key head and head unit, last block, slot of the first part}
    float2* part_ml;   // [block][slot][head of the unit]: maximum, sum
    float* part_o;     // [block][slot][head of the unit][D]
    uint32_t* status;
};

struct Bars {
    uint64_t full[4];
    uint64_t empty[4];
    int64_t warp_sums[8];
    int64_t start_base;    // the list's position of the block's first (request, head unit)
    int32_t start[2];      // which one that is
    int32_t bad[4];        // per stage: a page outside the cache
    float2 ml[kComputeWarps][kHeads];
    uint32_t abort_flag;
};
static_assert(2 * (Config<128, 1>::kSmem + (int)sizeof(Bars) + 1024) <= 228 * 1024, "two blocks to an SM");

// Units of a request: none if there is nothing to read, or nothing that may be read.
template <int kTile>
__device__ __forceinline__ int units_of(const Params& p, int r)
{
    const int64_t len = p.lengths[r];
    return len > 0 && len <= (int64_t)p.max_blocks * p.page_size ? (int)((len + kTile - 1) / kTile) : 0;
}

// A block's run through the list, one (request, head unit) after the other.  Each takes its units' places in the list
// and kPairCost more.
template <int kTile>
struct Walk {
    int r, hh, first, count, units, len;
    int64_t base, end;  // places in the list: of the current one's first unit, of the end of the run
    bool any;           // whether the block has had units before the current ones

    __device__ __forceinline__ void here(const Params& p, int64_t from)
    {
        len = p.lengths[r];
        units = (int)(((int64_t)len + kTile - 1) / kTile);
        first = from > base ? (int)(from - base) : 0;
        const int64_t last = end - base < units ? end - base : units;
        count = last > first ? (int)(last - first) : 0;
    }
    // to the next one; false at the run's end
    __device__ __forceinline__ bool next(const Params& p)
    {
        any = any || count > 0;
        base += units + kPairCost;
        if (base >= end) {
            return false;
        }
        if (++hh == p.kv_heads * p.head_units) {
            hh = 0;
            do {
                ++r;
                if (r >= p.requests) {
                    return false;
                }
            } while (units_of<kTile>(p, r) == 0);
        }
        here(p, base);
        return true;
    }
};

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t v)
{
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

// Two numbers as 16-bit values, and what that leaves over as 16-bit values.
template <typename T>
__device__ __forceinline__ void split(float x, float y, uint32_t& high, uint32_t& low)
{
    high = pack<T>(x, y);
    const float2 h = unpack<T>(high);
    low = pack<T>(x - h.x, y - h.y);
}

__device__ __forceinline__ void report_timeout(const Params& p, volatile uint32_t* abort_flag, uint32_t role, uint32_t where)
{
    *abort_flag = 1u;
    atomicCAS(p.status, 0u, 0x90000000u | (role << 24) | ((where & 0xFFu) << 16) | (blockIdx.x & 0xFFFFu));
}

// Two neighbouring elements of q as 32-bit numbers; `pairs`: they may be read at once.
template <typename Q>
__device__ __forceinline__ float2 load_two(const Q* q, bool pairs)
{
    if (pairs) {
        if constexpr (std::is_same<Q, float>::value) {
            return *reinterpret_cast<const float2*>(q);
        } else {
            return unpack<Q>(*reinterpret_cast<const uint32_t*>(q));
        }
    }
    return make_float2(to_f32(q[0]), to_f32(q[1]));
}

// Asks for the line of an address in L1 without waiting for it.
__device__ __forceinline__ void touch(const void* p)
{
    asm volatile(
        "{\n\t"
        ".reg .u16 unused;\n\t"
        "ld.global.ca.u16 unused, [%0];\n\t"
        "}" ::"l"(p));
}

// What one warp has of its 8 query heads and a run of keys: maxima, sums, unnormalised output (fragments: row g of the
// first product's operand is in [0], [1], row g + 8, its low part, in [2], [3]).
template <int D, typename T, bool kLowQ, int kChunk>
struct Softmax {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kSteps = D / 16, kPairs = kChunk / 16;
    uint32_t q_hi[kSteps][2], q_lo[kLowQ ? kSteps : 1][2];
    float acc[D / 8][4];
    float m, l;  // of row g; l: this lane's columns only

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        }
        m = -INFINITY;
        l = 0.0f;
    }

    // kChunk keys, whose rows for ldmatrix are at k_row and v_row; `keys` of them count (kRagged: not all, and the rest
    // may be anything).
    template <bool kRagged>
    __device__ __forceinline__ void add(const uint32_t (&k_row)[kPairs], const uint32_t (&v_row)[kPairs], uint32_t half,
                                        int keys, float scale)
    {
        const int lane = threadIdx.x % 32, t = lane % 4, matrix = lane / 8, row8 = lane % 8;
        float s[2 * kPairs][4];
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) {
            s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
#pragma unroll
            for (int n = 0; n < kPairs; ++n) {
                uint32_t b[4];
                ldmatrix_x4(k_row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix % 2) ^ row8) << 4), b);
                const uint32_t a1 = kLowQ ? q_lo[kLowQ ? i : 0][0] : 0u, a3 = kLowQ ? q_lo[kLowQ ? i : 0][1] : 0u;
                mma_m16n8k16<kBf16>(s[2 * n], q_hi[i][0], a1, q_hi[i][1], a3, b[0], b[1]);
                mma_m16n8k16<kBf16>(s[2 * n + 1], q_hi[i][0], a1, q_hi[i][1], a3, b[2], b[3]);
            }
        }
        float most = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2 * kPairs; ++n) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = s[n][j];
                if (kLowQ) {
                    // (a low part that is not finite has met an infinite key: the high part says what that gives)
                    x += fabsf(s[n][2 + j]) < INFINITY ? s[n][2 + j] : 0.0f;
                }
                if (kRagged && n * 8 + 2 * t + j >= keys) {
                    x = -INFINITY;
                }
                s[n][j] = x;
                most = fmaxf(most, x);
            }
        }
        most *= scale;
        if (__any_sync(0xFFFFFFFFu, most > m + kSlack)) {
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
            most = fmaxf(most, m);
            const float down = ex2(m - (most == -INFINITY ? 0.0f : most));
            m = most;
            l *= down;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                acc[i][0] *= down;
                acc[i][1] *= down;
                acc[i][2] *= down;
                acc[i][3] *= down;
            }
        }
        const float shift = m == -INFINITY ? 0.0f : kShift - m;
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
            float w[4];
            uint32_t a[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = ex2(fmaf(s[2 * n + j / 2][j % 2], scale, shift));
                l += w[j];
            }
            split<T>(w[0], w[1], a[0], a[1]);
            split<T>(w[2], w[3], a[2], a[3]);
            // a value that does not count may be NaN, and its weight of zero would not remove it
            uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
            if (kRagged) {
                const int k = n * 16 + 2 * t;
                keep0 = (k < keys ? 0xFFFFu : 0u) | (k + 1 < keys ? 0xFFFF0000u : 0u);
                keep1 = (k + 8 < keys ? 0xFFFFu : 0u) | (k + 9 < keys ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                uint32_t b[4];
                ldmatrix_x4_trans(v_row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix / 2) ^ row8) << 4), b);
                mma_m16n8k16<kBf16>(acc[2 * i], a[0], a[1], a[2], a[3], kRagged ? b[0] & keep0 : b[0],
                                    kRagged ? b[1] & keep1 : b[1]);
                mma_m16n8k16<kBf16>(acc[2 * i + 1], a[0], a[1], a[2], a[3], kRagged ? b[2] & keep0 : b[2],
                                    kRagged ? b[3] & keep1 : b[3]);
            }
        }
    }
};

template <int D, typename T, typename Q, int kGroups>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    attn_paged_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p)
{
    using Cfg = Config<D, kGroups>;
    using W = Walk<Cfg::kTile>;
    constexpr bool kLowQ = std::is_same<Q, float>::value;  // q has a low part
    constexpr int kUnitHeads = kGroups * kHeads;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars bars;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float* join = reinterpret_cast<float*>(smem_raw + (stages - smem_u32(smem_raw)) + Cfg::kStages * Cfg::kStageBytes);
    volatile uint32_t* abort_flag = &bars.abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(smem_u32(&bars.full[s]), 1);
            mbar_init(smem_u32(&bars.empty[s]), kComputeWarps);
            bars.bad[s] = 0;
        }
        bars.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kComputeWarps && lane == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    // launched early, this kernel touches nothing of its inputs, outputs or workspace before this point
    grid_dependency_wait();
    grid_launch_dependents();

    // ------------------------------------------------------------ this block's run of the list
    const int hhs = p.kv_heads * p.head_units;
    int64_t total = 0;  // places in the list
    {
        const int chunk = (p.requests + kThreads - 1) / kThreads;
        const int r0 = (int)threadIdx.x * chunk, r1 = r0 + chunk < p.requests ? r0 + chunk : p.requests;
        const auto places = [&](int r) {
            const int units = units_of<Cfg::kTile>(p, r);
            return units ? (int64_t)(units + kPairCost) * hhs : 0;
        };
        int64_t mine = 0;
        for (int r = r0; r < r1; ++r) {
            mine += places(r);
        }
        int64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int64_t w = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            upto += lane >= d ? w : 0;
        }
        if (lane == 31) {
            bars.warp_sums[warp] = upto;
        }
        __syncthreads();
        int64_t base = upto - mine;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            base += w < warp ? bars.warp_sums[w] : 0;
            total += bars.warp_sums[w];
        }
        const int64_t blocks = total < gridDim.x ? total : gridDim.x;
        if (blockIdx.x < blocks) {
            const int64_t u0 = blockIdx.x * total / blocks;
            if (u0 >= base && u0 < base + mine) {
                int r = r0;
                int64_t its = places(r);
                while (u0 >= base + its) {
                    base += its;
                    its = places(++r);
                }
                const int hh = (int)((u0 - base) / (its / hhs));
                bars.start[0] = r;
                bars.start[1] = hh;
                bars.start_base = base + hh * (its / hhs);
            }
        }
        __syncthreads();
    }
    const int64_t blocks = total < gridDim.x ? total : gridDim.x;
    const bool work = blockIdx.x < blocks;
    W walk{};
    if (work) {
        walk.r = bars.start[0];
        walk.hh = bars.start[1];
        walk.base = bars.start_base;
        walk.end = (blockIdx.x + 1) * total / blocks;
        walk.here(p, blockIdx.x * total / blocks);
    }
    if (threadIdx.x == 0) {
        // The first block whose run begins after the first unit of a (request, head unit), and before its end, names the
        // parts of it: the block before has the first one (as its first run of units or a later one), then this block and
        // those behind it as their first.
        int4 j = make_int4(-1, 0, 0, 0);
        if (work && walk.first > 0 && walk.count > 0) {
            const int64_t previous = (blockIdx.x - 1) * total / blocks;
            if (previous <= walk.base) {
                const int64_t last = walk.base + walk.units - 1;
                j = make_int4(walk.r, walk.hh, (int)(((last + 1) * blocks - 1) / total),
                              previous >= walk.base - kPairCost ? 0 : 1);
            }
        }
        p.joins[blockIdx.x] = j;
    }

    const int rows = p.box_rows;
    if (warp == kComputeWarps) {
        // -------------------------------------------------------------------------------------- copies
        const Checker ck{p.status, stages, stages + Cfg::kStages * Cfg::kStageBytes, 0, 0};
        const int boxes = Cfg::kTile / rows;
        const uint32_t box_bytes = rows * D * 2;
        uint32_t stage = 0, phase = 0, used = 0;
        bool ok = true;
        // to the first (request, head unit) from here on that has units for this block
        auto settle = [&](bool more) {
            while (more && walk.count == 0) {
                more = walk.next(p);
            }
            return more;
        };
        bool more = settle(work);
        int unit = walk.first;
        // the page of this lane's box of a unit; -1 if it is behind the last key
        auto page_of = [&](int u) {
            const int64_t at = (int64_t)u * Cfg::kTile + lane * rows;
            return lane < boxes && at < walk.len ? p.table[walk.r * p.table_stride + (uint32_t)at / (uint32_t)p.page_size] : -1;
        };
        int page = more ? page_of(unit) : -1;
        while (more) {
            const int64_t at = (int64_t)unit * Cfg::kTile + lane * rows;
            const bool mine = lane < boxes && at < walk.len;
            const int this_page = page, head = walk.hh / p.head_units;
            const int row = mine ? (int)((uint32_t)at % (uint32_t)p.page_size) : 0;
            if (++unit == walk.first + walk.count) {
                more = settle(walk.next(p));
                unit = walk.first;
                if (more) {
                    // the queries of what comes next, on their way while the units before it are worked on: a line per lane
                    constexpr int kLines = D * (int)sizeof(Q) / 128;
                    for (int i = lane; i < kUnitHeads * kLines; i += 32) {
                        const int in_group = (walk.hh % p.head_units) * kUnitHeads + i / kLines;
                        if (in_group < p.group) {
                            touch(static_cast<const Q*>(p.q) + walk.r * p.q_request_stride +
                                  (int64_t)(walk.hh / p.head_units * p.group + in_group) * p.q_head_stride +
                                  (i % kLines) * (128 / (int)sizeof(Q)));
                        }
                    }
                }
            }
            page = more ? page_of(unit) : -1;  // asked for one unit ahead
            ok = mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag);
            if (!ok && lane == 0) {
                report_timeout(p, abort_flag, 1, stage);
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) {
                break;
            }
            const bool good = mine && this_page >= 0 && this_page < p.num_pages;
            const uint32_t bad = __ballot_sync(0xFFFFFFFFu, mine && !good), valid = __ballot_sync(0xFFFFFFFFu, good);
            const uint32_t full = smem_u32(&bars.full[stage]);
            const uint32_t keys = stages + stage * Cfg::kStageBytes + lane * box_bytes;
            if (lane == 0) {
                bars.bad[stage] = bad != 0;
                mbar_arrive_expect_tx(full, 2 * box_bytes * __popc(valid));
            }
            __syncwarp();
            if (good && ck.smem(keys, box_bytes, 1024, 0x501) && ck.smem(keys + Cfg::kHalfUnit, box_bytes, 1024, 0x502) &&
                ck.tma_coords(0, 2, row, this_page, 0x503)) {
                tma_load_5d(keys, &map_k, full, 0, row, 0, head, this_page);
                tma_load_5d(keys + Cfg::kHalfUnit, &map_v, full, 0, row, 0, head, this_page);
            }
            ++used;
            if (++stage == Cfg::kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (!ok) {
            // copies that are still under way end before the block does (each wait has its limit)
            for (uint32_t s = 0; s < Cfg::kStages; ++s) {
                const uint32_t fills = used / Cfg::kStages + (s < used % Cfg::kStages ? 1 : 0);
                if (fills > 0) {
                    volatile uint32_t not_aborted = 0;
                    mbar_wait(smem_u32(&bars.full[s]), (fills - 1) & 1u, &not_aborted);
                }
            }
        }
    } else {
        // ------------------------------------------------------------------------------------- products
        const int group = warp / Cfg::kWarps, part = warp % Cfg::kWarps;  // group of warps, warp of the group
        const int g = lane / 4, t = lane % 4;                             // row (query head) and column pair of a fragment
        const int matrix = lane / 8, row8 = lane % 8;
        using S = Softmax<D, T, kLowQ, Cfg::kChunk>;
        constexpr int kPairs = S::kPairs, kSteps = S::kSteps, kChunks = Cfg::kKeys / Cfg::kChunk;
        // shared-memory offsets of this lane's ldmatrix rows: keys (matrices 0, 1 | 2, 3 are keys 0-7 | 8-15) and values
        // (matrices 0, 2 | 1, 3); a box of `rows` rows holds its halves of 64 columns one behind the other
        auto row_at = [&](int r) { return (uint32_t)((r / rows) * rows * D * 2 + (r % rows) * 128); };
        uint32_t k_at[kChunks][kPairs], v_at[kChunks][kPairs];
        for (int c = 0; c < kChunks; ++c) {
            for (int i = 0; i < kPairs; ++i) {
                const int r = part * Cfg::kKeys + c * Cfg::kChunk + i * 16 + row8;
                k_at[c][i] = row_at(r + (matrix / 2) * 8);
                v_at[c][i] = row_at(r + (matrix % 2) * 8) + Cfg::kHalfUnit;
            }
        }
        const uint32_t half = rows * 128;
        uint32_t stage = 0, phase = 0;
        bool ok = true, joined = false;
        S sm;

        for (bool more = work; more; more = walk.next(p)) {
            if (walk.count == 0) {
                continue;
            }
            const int kv = walk.hh / p.head_units, in_group = (walk.hh % p.head_units) * kUnitHeads + group * kHeads + g;
            const bool head_here = in_group < p.group;
            // q: rows g and, for what rounding left over, g + 8 of the A operand
            {
                const Q* q = static_cast<const Q*>(p.q) + walk.r * p.q_request_stride +
                             (int64_t)(kv * p.group + (head_here ? in_group : 0)) * p.q_head_stride + 2 * t;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float2 x = load_two(q + i * 16 + j * 8, p.q_pairs);
                        x = head_here ? x : make_float2(0.0f, 0.0f);
                        if (kLowQ) {
                            split<T>(x.x, x.y, sm.q_hi[i][j], sm.q_lo[kLowQ ? i : 0][j]);
                        } else {
                            sm.q_hi[i][j] = pack<T>(x.x, x.y);
                        }
                    }
                }
            }
            sm.clear();
            int bad = 0;

            for (int u = walk.first; u < walk.first + walk.count; ++u) {
                if (ok && !mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
                    report_timeout(p, abort_flag, 2, stage);
                    ok = false;
                }
                ok = __all_sync(0xFFFFFFFFu, ok);
                bad |= *const_cast<volatile int32_t*>(&bars.bad[stage]);
                const uint32_t base = stages + stage * Cfg::kStageBytes;
                const int64_t left = walk.len - (int64_t)u * Cfg::kTile - part * Cfg::kKeys;  // keys from this warp's first on
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    uint32_t k_row[kPairs], v_row[kPairs];
#pragma unroll
                    for (int i = 0; i < kPairs; ++i) {
                        k_row[i] = base + k_at[c][i];
                        v_row[i] = base + v_at[c][i];
                    }
                    const int keys = left > Cfg::kTile ? Cfg::kTile : (int)left - c * Cfg::kChunk;
                    if (ok && keys >= Cfg::kChunk) {
                        sm.template add<false>(k_row, v_row, half, keys, p.scale_log2e);
                    } else if (ok && keys > 0) {
                        sm.template add<true>(k_row, v_row, half, keys, p.scale_log2e);
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&bars.empty[stage]));
                }
                if (++stage == Cfg::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }

            // ------------------------------------------------- the warps of the group joined, the result or part written
            float o[D / 8][2], m = sm.m, l = sm.l;
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
            l = bad ? NAN : l;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] = sm.acc[i][0] + sm.acc[i][2];
                o[i][1] = sm.acc[i][1] + sm.acc[i][3];
            }
            // Warps kWarps / 2 .. kWarps - 1 hand their sums to warps 0 .., and so on.  Named barriers of the two warps:
            // 2 w - 1 says that warp w's buffer is full, 2 w that it is free again (w: among all compute warps).
            bool mine = true;
#pragma unroll
            for (int from = Cfg::kWarps / 2; from > 0; from /= 2) {
                if (part >= from && part < 2 * from) {
                    float* to = join + ((group * (Cfg::kWarps - 1) + part - 1) * kHeads + g) * Cfg::kPadded + 2 * t;
                    if (joined) {
                        named_barrier_sync(2 * warp, 64);
                    }
                    if (t == 0) {
                        bars.ml[warp][g] = make_float2(m, l);
                    }
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        *reinterpret_cast<float2*>(to + i * 8) = make_float2(o[i][0], o[i][1]);
                    }
                    named_barrier_arrive(2 * warp - 1, 64);
                    mine = false;
                } else if (part < from) {
                    const int other = warp + from;
                    const float* at = join + ((group * (Cfg::kWarps - 1) + part + from - 1) * kHeads + g) * Cfg::kPadded + 2 * t;
                    named_barrier_sync(2 * other - 1, 64);
                    const float2 ml = bars.ml[other][g];
                    const float most = fmaxf(m, ml.x), to = most == -INFINITY ? 0.0f : most;
                    const float down = ex2(m - to), other_down = ex2(ml.x - to);
                    l = l * down + ml.y * other_down;
                    m = most;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const float2 x = *reinterpret_cast<const float2*>(at + i * 8);
                        o[i][0] = o[i][0] * down + x.x * other_down;
                        o[i][1] = o[i][1] * down + x.y * other_down;
                    }
                    named_barrier_arrive(2 * other, 64);
                }
            }
            joined = true;
            if (mine && head_here) {
                if (walk.count == walk.units) {
                    const int64_t row = (int64_t)walk.r * p.heads + kv * p.group + in_group;
                    const float by = 1.0f / l;
                    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + row * D) + t;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        out[i * 4] = pack<T>(o[i][0] * by, o[i][1] * by);
                    }
                    if (p.lse && t == 0) {
                        p.lse[row] = ((m == -INFINITY ? 0.0f : m) - kShift + log2f(l)) * kLn2;
                    }
                } else {
                    const int64_t row = ((int64_t)blockIdx.x * 2 + (walk.any ? 1 : 0)) * kUnitHeads + group * kHeads + g;
                    float* out = p.part_o + row * D + 2 * t;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        *reinterpret_cast<float2*>(out + i * 8) = make_float2(o[i][0], o[i][1]);
                    }
                    if (t == 0) {
                        p.part_ml[row] = make_float2(m, l);
                    }
                }
            }
            __syncwarp();
        }
        // the last buffers that were handed over have been taken (their barriers are left as they were found)
        if (joined && part > 0) {
            named_barrier_sync(2 * warp, 64);
        }
        // requests without units: no keys, or lengths that cannot be
        for (int r = blockIdx.x; r < p.requests; r += gridDim.x) {
            if (units_of<Cfg::kTile>(p, r) == 0) {
                const bool empty = p.lengths[r] == 0;
                const uint32_t fill = empty ? 0u : pack<T>(NAN, NAN);
                uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + (int64_t)r * p.heads * D);
                for (int i = threadIdx.x; i < p.heads * (D / 2); i += kComputeWarps * 32) {
                    o[i] = fill;
                }
                for (int i = threadIdx.x; p.lse && i < p.heads; i += kComputeWarps * 32) {
                    p.lse[(int64_t)r * p.heads + i] = empty ? -INFINITY : NAN;
                }
            }
        }
    }
}

// Joins the parts of one query head of a (request, head unit): block x of the first kernel named them in joins[x].  Most
// blocks find nothing to join or a few parts, so a part is one warp's read and its maximum, sum and output are asked for
// at once; of many parts each warp takes every fourth, and the warps are joined at the end.
template <int D, typename T>
__global__ void __launch_bounds__(kJoinThreads) attn_paged_join_kernel(const Params p, int unit_heads)
{
    constexpr int kWarps = kJoinThreads / 32, kPer = D / 32;
    __shared__ float2 ml[kWarps];
    __shared__ float sums[kWarps][D];
    grid_dependency_wait();
    grid_launch_dependents();
    const int4 j = p.joins[blockIdx.x];
    const int h = blockIdx.y, head = (j.y % p.head_units) * unit_heads + h;
    if (j.x < 0 || head >= p.group) {
        return;
    }
    const int parts = j.z - (int)blockIdx.x + 2;  // of blocks blockIdx.x - 1 .. j.z
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float m = -INFINITY, l = 0.0f, o[kPer] = {};
    constexpr int kAtOnce = 4;
    for (int i0 = warp; i0 < parts; i0 += kAtOnce * kWarps) {
        float2 part[kAtOnce];
        float x[kAtOnce][kPer];
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const int i = i0 + n * kWarps;
            if (i < parts) {
                const int64_t row = (((int64_t)blockIdx.x - 1 + i) * 2 + (i == 0 ? j.w : 0)) * unit_heads + h;
                part[n] = p.part_ml[row];
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    x[n][k] = p.part_o[row * D + lane + k * 32];
                }
            } else {
                part[n] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    x[n][k] = 0.0f;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kAtOnce; ++n) {
            const float most = fmaxf(m, part[n].x), to = most == -INFINITY ? 0.0f : most;
            const float down = ex2(m - to), other = ex2(part[n].x - to);
            m = most;
            l = l * down + part[n].y * other;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                o[k] = o[k] * down + x[n][k] * other;
            }
        }
    }
    if (lane == 0) {
        ml[warp] = make_float2(m, l);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        sums[warp][lane + k * 32] = o[k];
    }
    __syncthreads();
    float most = -INFINITY, total = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
        most = fmaxf(most, ml[w].x);
    }
    const float to = most == -INFINITY ? 0.0f : most;
    float weight[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        weight[w] = ex2(ml[w].x - to);
        total += ml[w].y * weight[w];
    }
    const int64_t row = (int64_t)j.x * p.heads + (j.y / p.head_units) * p.group + head;
    const float by = 1.0f / total;
    if (threadIdx.x < D / 2) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            a += sums[w][2 * threadIdx.x] * weight[w];
            b += sums[w][2 * threadIdx.x + 1] * weight[w];
        }
        reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + row * D)[threadIdx.x] = pack<T>(a * by, b * by);
    }
    if (p.lse && threadIdx.x == 0) {
        p.lse[row] = (to - kShift + log2f(total)) * kLn2;
    }
}

// ------------------------------------------------------------------ host side

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled_fn()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<EncodeTiledFn>(sym);
        }
    });
    return fn;
}

// Query heads of a key head are taken 8, 16 or 32 at a time (groups of warps that share the keys in shared memory).
static int groups_of(int group) { return group <= kHeads ? 1 : group <= 2 * kHeads ? 2 : 4; }
static int blocks_of(int sm_count) { return kBlocksPerSm * sm_count; }

static int make_map(CUtensorMap* map, void* base, const spork_paged_cache& c, const int64_t* strides)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) {
        return SPORK_ERR_DRIVER;
    }
    // a dimension of one element may carry any stride: give it one that the map takes
    const auto bytes = [&](int64_t stride, int64_t n) { return (cuuint64_t)(n > 1 ? stride * 2 : 16); };
    const cuuint64_t dims[5] = {64, (cuuint64_t)c.page_size, (cuuint64_t)(c.head_dim / 64), (cuuint64_t)c.kv_heads,
                                (cuuint64_t)(c.num_pages > 0 ? c.num_pages : 1)};
    const cuuint64_t steps[4] = {bytes(strides[2], c.page_size), 128, bytes(strides[1], c.kv_heads),
                                 bytes(strides[0], c.num_pages)};
    const cuuint32_t box[5] = {64, (cuuint32_t)(c.page_size < kMaxRows ? c.page_size : kMaxRows), (cuuint32_t)(c.head_dim / 64), 1, 1};
    const cuuint32_t elem_strides[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, c.type == SPORK_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                          base, dims, steps, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : SPORK_ERR_DRIVER;
}

struct Workspace {
    int64_t joins, ml, o, bytes;
    Workspace(int blocks, int groups, int D)
    {
        const int64_t rows = (int64_t)blocks * 2 * groups * kHeads;
        joins = 0;
        ml = joins + (int64_t)blocks * 16;
        o = ml + rows * 8;
        bytes = o + rows * D * 4;
    }
};

static cudaLaunchConfig_t launch_config(cudaLaunchAttribute* attr, dim3 grid, int threads, int smem, cudaStream_t stream)
{
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <int D, typename T, typename Q, int kGroups>
static int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, bool joined, DeviceState& dev,
                  cudaStream_t stream)
{
    using Cfg = Config<D, kGroups>;
    auto kernel = attn_paged_kernel<D, T, Q, kGroups>;
    static std::once_flag attr_once[kMaxDevices];
    static cudaError_t attr_err[kMaxDevices];
    std::call_once(attr_once[dev.ordinal], [&] {
        attr_err[dev.ordinal] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
    });
    if (attr_err[dev.ordinal] != cudaSuccess) {
        return (int)attr_err[dev.ordinal];
    }
    const int blocks = blocks_of(dev.sm_count);
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = launch_config(&attr, dim3(blocks), kThreads, Cfg::kSmem, stream);
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, p);
    if (e == cudaSuccess && joined) {
        const int heads = p.group < kGroups * kHeads ? p.group : kGroups * kHeads;
        cfg = launch_config(&attr, dim3(blocks, heads), kJoinThreads, 0, stream);
        e = cudaLaunchKernelEx(&cfg, attn_paged_join_kernel<D, T>, p, kGroups * kHeads);
    }
    return (int)e;
}

template <int D, typename T, typename Q>
static int launch_groups(int groups, const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, bool joined,
                         DeviceState& dev, cudaStream_t stream)
{
    return groups == 1   ? launch<D, T, Q, 1>(map_k, map_v, p, joined, dev, stream)
           : groups == 2 ? launch<D, T, Q, 2>(map_k, map_v, p, joined, dev, stream)
                         : launch<D, T, Q, 4>(map_k, map_v, p, joined, dev, stream);
}

template <int D, typename T>
static int launch_q(bool f32, int groups, const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, bool joined,
                    DeviceState& dev, cudaStream_t stream)
{
    return f32 ? launch_groups<D, T, float>(groups, map_k, map_v, p, joined, dev, stream)
               : launch_groups<D, T, T>(groups, map_k, map_v, p, joined, dev, stream);
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
    using namespace spork::attn_paged_sm100;
    if (!spork_attn_sm100_paged_supports(heads, kv_heads, head_dim, 8)) {
        return -(int64_t)SPORK_ERR_UNSUPPORTED_SHAPE;
    }
    spork::DeviceState* dev = nullptr;
    const int rc = spork::current_device_state(&dev);
    if (rc) {
        return -(int64_t)rc;
    }
    const int groups = groups_of(heads / kv_heads);
    return Workspace(blocks_of(dev->sm_count), groups, head_dim).bytes;
}

extern "C" int spork_attn_sm100_paged(const spork_attn_paged_args* args, void* stream)
{
    using namespace spork::attn_paged_sm100;
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
        !(a.scale * kLog2e <= 3.4028235e38f)) {
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
    spork::DeviceState* dev = nullptr;
    const int rc2 = spork::current_device_state(&dev);
    if (rc2) {
        return rc2;
    }
    const int group = a.heads / c.kv_heads, groups = groups_of(group), blocks = blocks_of(dev->sm_count);
    const Workspace w(blocks, groups, c.head_dim);
    if (blocks > kMaxBlocks) {
        return SPORK_ERR_TOO_LARGE;
    }
    if (!a.workspace || a.workspace_bytes < w.bytes) {
        return SPORK_ERR_BAD_ARGUMENT;
    }
    CUtensorMap map_k, map_v;
    int rc3;
    if ((rc3 = make_map(&map_k, c.num_pages > 0 ? c.k : a.o, c, c.k_strides)) != 0 ||
        (rc3 = make_map(&map_v, c.num_pages > 0 ? c.v : a.o, c, c.v_strides)) != 0) {
        return rc3;
    }
    Params p{};
    p.q = a.q;
    p.table = a.block_table;
    p.lengths = a.lengths;
    p.o = a.o;
    p.lse = a.lse;
    p.q_request_stride = a.q_request_stride;
    p.q_head_stride = a.q_head_stride;
    p.table_stride = a.table_stride;
    p.requests = a.requests;
    p.heads = a.heads;
    p.kv_heads = c.kv_heads;
    p.group = group;
    p.head_units = (group + groups * kHeads - 1) / (groups * kHeads);
    p.max_blocks = a.max_blocks;
    p.num_pages = c.num_pages;
    p.page_size = c.page_size;
    p.box_rows = c.page_size < kMaxRows ? c.page_size : kMaxRows;
    p.scale_log2e = a.scale * kLog2e;
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    p.joins = reinterpret_cast<int4*>(ws + w.joins);
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    p.part_o = reinterpret_cast<float*>(ws + w.o);
    p.status = dev->status_word;
    p.q_pairs = ((reinterpret_cast<uintptr_t>(a.q) % (2 * q_elem)) | ((a.q_request_stride | a.q_head_stride) & 1)) == 0;
    // one unit at most for every request: nothing to join
    const bool joined = (int64_t)a.max_blocks * c.page_size > 8192 / c.head_dim;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = a.q_type == SPORK_TYPE_F32;
    if (c.type == SPORK_TYPE_F16) {
        return c.head_dim == 64 ? launch_q<64, __half>(f32, groups, map_k, map_v, p, joined, *dev, s)
                                : launch_q<128, __half>(f32, groups, map_k, map_v, p, joined, *dev, s);
    }
    return c.head_dim == 64 ? launch_q<64, __nv_bfloat16>(f32, groups, map_k, map_v, p, joined, *dev, s)
                            : launch_q<128, __nv_bfloat16>(f32, groups, map_k, map_v, p, joined, *dev, s);
}
