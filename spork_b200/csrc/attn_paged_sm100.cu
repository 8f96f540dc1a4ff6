// Attention of one new token per request over a paged key-value cache, for sm_100a:
//   o[r][h] = softmax(scale q[r][h] K^T) V over the keys that request r holds, key head h / (heads / kv_heads).
//
// Every key and value is read once and used by the few query heads that share it, so the kernel is bound by HBM; the
// products are small.  Work is cut along the cache: units of 64 keys of one (request, key head), all units in one list,
// request by request, and each block of the grid takes an equal run of that list, whatever the lengths (they are known
// on the device only).  A block joins what it computes of one (request, key head) and writes the result if it has all
// of it; otherwise a partial result (running maximum, sum, unnormalised output) goes to the workspace, and a second
// small kernel joins the parts in the order of the keys.  A block has at most two partial results: its first run and its
// last one.
//
// One warp copies the pages with TMA: the cache is a 5-dimensional tensor (64 elements, page rows, halves of the head
// dimension, heads, pages) with the strides that it has, so any order in memory is one tensor map; a box is a page's
// rows of one head (64 rows of it at most), swizzled for ldmatrix.  Page numbers come from the block table, and are
// checked before they are used.
//
// The other warps compute, each on its own 16 (or 32) keys of a unit, with mma.m16n8k16.  Up to 8 query heads are rows
// 0-7 of the 16-row operand, and rows 8-15 hold what rounding to 16 bits left over: of q, if it is fp32, and of the
// softmax weights.  So both products are taken with about 22 (fp16) or 16 (bf16) bits of q and of the weights at no
// cost: the rows would have been empty, and the weights' rounding, the largest error of the usual scheme, is gone.
// Each warp runs its own online softmax, and the warps of a block are joined once per run, not once per unit.
// (tcgen05 would want 64 or 128 rows and a trip through tensor memory for every unit; the warp instruction's rate is
// several times what the loads can feed.)
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

constexpr int kTile = 64;          // keys per unit
constexpr int kHeads = 8;          // query heads of a group of warps
constexpr int kPadded = 72;        // floats between the rows of the joining buffer (64 columns): no bank conflicts
constexpr float kShift = 8.0f;     // weights are 2^(x - max + 8): up to 2^8, so that fp16 keeps the small ones normal
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxBlocks = 1024;   // blocks of a launch that a joined result can have parts from
constexpr int kJoinThreads = 256;

// kGroups groups of warps share a unit, each with 8 query heads of its own.
template <int D, int kGroups>
struct Config {
    static constexpr int kWarps = kGroups == 4 ? 2 : 4;         // warps of a group; each takes kTile / kWarps keys
    static constexpr int kKeys = kTile / kWarps;
    static constexpr int kCompute = kGroups * kWarps;
    static constexpr int kThreads = (kCompute + 1) * 32;
    static constexpr int kBlocksPerSm = kGroups == 1 ? 2 : 1;
    static constexpr int kHalves = D / 64;
    static constexpr int kHalfUnit = kTile * D * 2;             // the keys (or values) of a unit, bytes
    static constexpr int kStageBytes = 2 * kHalfUnit;
    static constexpr int kStages = 96 * 1024 / kStageBytes * (kGroups == 1 ? 1 : 2);
    static constexpr int kJoinFloats = kGroups * kWarps * kHeads * kPadded;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kJoinFloats * 4 + 1024;
    static_assert(kSmem * kBlocksPerSm <= 227 * 1024 - 1024 * kBlocksPerSm, "shared memory");
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
    // workspace
    int4* joins;       // per block: {request (-1: none), key head and head unit, last block, slot of the first part}
    float2* part_ml;   // [block][slot][head of the unit]: maximum, sum
    float* part_o;     // [block][slot][head of the unit][D]
    uint32_t* status;
};

struct Bars {
    uint64_t full[16];
    uint64_t empty[16];
    int64_t warp_sums[16];
    int32_t bad[16];       // per stage: a page outside the cache
    int32_t start[3];      // request, head unit, unit of the block's first key
    uint32_t abort_flag;
    float2 ml[4 * 8 * kHeads / 2];
};
static_assert(sizeof(Bars) <= 1024 + 512, "barriers");

// Units of a request: none if there is nothing to read, or nothing that may be read.
__device__ __forceinline__ int units_of(const Params& p, int r)
{
    const int64_t len = p.lengths[r];
    return len > 0 && len <= (int64_t)p.max_blocks * p.page_size ? (int)((len + kTile - 1) / kTile) : 0;
}

// A block's run through the list of units, one (request, head unit) after the other.
struct Walk {
    int r, hh, first, count, units, len;
    int64_t left;

    __device__ __forceinline__ void here(const Params& p)
    {
        len = p.lengths[r];
        units = (len + kTile - 1) / kTile;
        count = units - first < left ? units - first : (int)left;
    }
    // to the next one; false at the run's end
    __device__ __forceinline__ bool next(const Params& p)
    {
        left -= count;
        if (left <= 0) {
            return false;
        }
        first = 0;
        if (++hh == p.kv_heads * p.head_units) {
            hh = 0;
            do {
                ++r;
            } while (units_of(p, r) == 0);
        }
        here(p);
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

template <int D, typename T, typename Q, int kGroups>
__global__ void __launch_bounds__(Config<D, kGroups>::kThreads, Config<D, kGroups>::kBlocksPerSm)
    attn_paged_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p)
{
    using Cfg = Config<D, kGroups>;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr bool kLowQ = std::is_same<Q, float>::value;  // q has a low part
    constexpr int kUnitHeads = kGroups * kHeads;
    extern __shared__ uint8_t smem_raw[];
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* behind = smem_raw + (stages - smem_u32(smem_raw)) + Cfg::kStages * Cfg::kStageBytes;
    float* join = reinterpret_cast<float*>(behind);
    __shared__ Bars bars;
    volatile uint32_t* abort_flag = &bars.abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(smem_u32(&bars.full[s]), 1);
            mbar_init(smem_u32(&bars.empty[s]), Cfg::kCompute);
            bars.bad[s] = 0;
        }
        bars.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == Cfg::kCompute && lane == 0) {
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    // launched early, this kernel touches nothing of its inputs, outputs or workspace before this point
    grid_dependency_wait();
    grid_launch_dependents();

    // ------------------------------------------------------------ this block's run of the list of units
    const int hhs = p.kv_heads * p.head_units;
    int64_t total = 0;
    {
        const int chunk = (p.requests + Cfg::kThreads - 1) / Cfg::kThreads;
        const int r0 = (int)threadIdx.x * chunk, r1 = r0 + chunk < p.requests ? r0 + chunk : p.requests;
        int64_t mine = 0;
        for (int r = r0; r < r1; ++r) {
            mine += units_of(p, r);
        }
        int64_t upto = mine;
        for (int d = 1; d < 32; d *= 2) {
            const int64_t w = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            upto += lane >= d ? w : 0;
        }
        if (lane == 31) {
            bars.warp_sums[warp] = upto;
        }
        __syncthreads();
        int64_t before = 0;
        for (int w = 0; w < Cfg::kThreads / 32; ++w) {
            before += w < warp ? bars.warp_sums[w] : 0;
            total += bars.warp_sums[w];
        }
        total *= hhs;
        const int64_t blocks = total < gridDim.x ? total : gridDim.x;
        int64_t base = (before + upto - mine) * hhs;
        if (blockIdx.x < blocks) {
            const int64_t u0 = blockIdx.x * total / blocks;
            if (u0 >= base && u0 < base + mine * hhs) {
                int r = r0, units = units_of(p, r);
                while (u0 >= base + (int64_t)units * hhs) {
                    base += (int64_t)units * hhs;
                    units = units_of(p, ++r);
                }
                bars.start[0] = r;
                bars.start[1] = (int)((u0 - base) / units);
                bars.start[2] = (int)((u0 - base) % units);
            }
        }
        __syncthreads();
    }
    const int64_t blocks = total < gridDim.x ? total : gridDim.x;
    const int64_t u0 = blocks ? blockIdx.x * total / blocks : 0, u1 = blocks ? (blockIdx.x + 1) * total / blocks : 0;
    Walk walk{};
    walk.left = blockIdx.x < blocks ? u1 - u0 : 0;
    if (walk.left > 0) {
        walk.r = bars.start[0];
        walk.hh = bars.start[1];
        walk.first = bars.start[2];
        walk.here(p);
    }
    if (threadIdx.x == 0 && p.joins) {
        // the block whose run is the second one with keys of a (request, head unit) names the parts of it
        int4 j = make_int4(-1, 0, 0, 0);
        if (walk.left > 0 && walk.first > 0) {
            const int64_t begin = u0 - walk.first, end = begin + walk.units, previous = (blockIdx.x - 1) * total / blocks;
            if (previous <= begin) {
                j = make_int4(walk.r, walk.hh, (int)((end * blocks - 1) / total), previous == begin ? 0 : 1);
            }
        }
        p.joins[blockIdx.x] = j;
    }

    const int rows = p.box_rows;
    if (warp == Cfg::kCompute) {
        // -------------------------------------------------------------------------------------- copies
        const Checker ck{p.status, stages, stages + Cfg::kStages * Cfg::kStageBytes, 0, 0};
        const int boxes = kTile / rows;
        const uint32_t box_bytes = rows * D * 2;
        uint32_t stage = 0, phase = 0, used = 0;
        bool ok = true;
        bool more = walk.left > 0;
        int unit = walk.first;
        // the page of this lane's box of a unit; -1 if it is behind the last key
        auto page_of = [&](const Walk& w, int u) {
            const int at = u * kTile + lane * rows;
            return lane < boxes && at < w.len ? p.table[w.r * p.table_stride + at / p.page_size] : -1;
        };
        int page = more ? page_of(walk, unit) : -1;
        while (more && ok) {
            const int at = unit * kTile + lane * rows;
            const bool mine = lane < boxes && at < walk.len;
            const int this_page = page, head = walk.hh / p.head_units;
            if (++unit == walk.first + walk.count) {
                more = walk.next(p);
                unit = walk.first;
            }
            page = more ? page_of(walk, unit) : -1;  // asked for one unit ahead
            if (!mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag)) {
                if (lane == 0) {
                    report_timeout(p, abort_flag, 1, stage);
                }
                ok = false;
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
                ck.tma_coords(0, 2, at % p.page_size, this_page, 0x503)) {
                tma_load_5d(keys, &map_k, full, 0, at % p.page_size, 0, head, this_page);
                tma_load_5d(keys + Cfg::kHalfUnit, &map_v, full, 0, at % p.page_size, 0, head, this_page);
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
        constexpr int kPairs = Cfg::kKeys / 16;                           // 16-key steps of a warp
        constexpr int kSteps = D / 16;
        // shared-memory offsets of this lane's ldmatrix rows: keys (matrices 0, 1 | 2, 3 are keys 0-7 | 8-15) and values
        // (matrices 0, 2 | 1, 3); a box of `rows` rows holds its halves of 64 columns one behind the other
        auto row_at = [&](int r) { return (uint32_t)((r / rows) * rows * D * 2 + (r % rows) * 128); };
        uint32_t k_row[kPairs], v_row[kPairs];
        for (int i = 0; i < kPairs; ++i) {
            k_row[i] = row_at(part * Cfg::kKeys + i * 16 + (matrix / 2) * 8 + row8);
            v_row[i] = row_at(part * Cfg::kKeys + i * 16 + (matrix % 2) * 8 + row8) + Cfg::kHalfUnit;
        }
        const uint32_t half = rows * 128;
        float* my_join = join + (group * Cfg::kWarps + part) * kHeads * kPadded;
        float2* group_ml = bars.ml + group * Cfg::kWarps * kHeads;
        uint32_t stage = 0, phase = 0;
        bool ok = true;

        for (bool more = walk.left > 0; more; more = walk.next(p)) {
            const int kv = walk.hh / p.head_units, in_group = (walk.hh % p.head_units) * kUnitHeads + group * kHeads + g;
            const bool head_here = in_group < p.group;
            // q: rows g and, for what rounding left over, g + 8 of the A operand
            uint32_t q_hi[kSteps][2], q_lo[kLowQ ? kSteps : 1][2];
            {
                const Q* q = static_cast<const Q*>(p.q) + walk.r * p.q_request_stride +
                             (int64_t)(kv * p.group + (head_here ? in_group : 0)) * p.q_head_stride + 2 * t;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float x = head_here ? to_f32(q[i * 16 + j * 8]) : 0.0f;
                        const float y = head_here ? to_f32(q[i * 16 + j * 8 + 1]) : 0.0f;
                        if (kLowQ) {
                            split<T>(x, y, q_hi[i][j], q_lo[kLowQ ? i : 0][j]);
                        } else {
                            q_hi[i][j] = pack<T>(x, y);
                        }
                    }
                }
            }
            float acc[D / 8][4];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
            }
            float m = -INFINITY, l = 0.0f;  // of row g; l: this lane's columns only
            bool bad = false;

            for (int u = walk.first; u < walk.first + walk.count; ++u) {
                if (ok && !mbar_wait(smem_u32(&bars.full[stage]), phase, abort_flag)) {
                    report_timeout(p, abort_flag, 2, stage);
                    ok = false;
                }
                ok = __all_sync(0xFFFFFFFFu, ok);
                bad = bad || *const_cast<volatile int32_t*>(&bars.bad[stage]) != 0;
                const int first_key = u * kTile + part * Cfg::kKeys;
                if (ok && first_key < walk.len) {
                    const uint32_t base = stages + stage * Cfg::kStageBytes;
                    // scores of Cfg::kKeys keys: 8 at a time
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
                            ldmatrix_x4(base + k_row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix % 2) ^ row8) << 4), b);
                            const uint32_t a1 = kLowQ ? q_lo[kLowQ ? i : 0][0] : 0u, a3 = kLowQ ? q_lo[kLowQ ? i : 0][1] : 0u;
                            mma_m16n8k16<kBf16>(s[2 * n], q_hi[i][0], a1, q_hi[i][1], a3, b[0], b[1]);
                            mma_m16n8k16<kBf16>(s[2 * n + 1], q_hi[i][0], a1, q_hi[i][1], a3, b[2], b[3]);
                        }
                    }
                    const int keys = walk.len - first_key;  // that count; the rest may be anything
                    const bool ragged = keys < Cfg::kKeys;
                    float most = -INFINITY;
#pragma unroll
                    for (int n = 0; n < 2 * kPairs; ++n) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float x = s[n][j];
                            if (kLowQ) {
                                // (a part that is not finite has met an infinite key: the high part says what it gives)
                                x += fabsf(s[n][2 + j]) < INFINITY ? s[n][2 + j] : 0.0f;
                            }
                            x *= p.scale_log2e;
                            if (ragged && n * 8 + 2 * t + j >= keys) {
                                x = -INFINITY;
                            }
                            s[n][j] = x;
                            most = fmaxf(most, x);
                        }
                    }
                    most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
                    const float m_new = fmaxf(m, most);
                    const float shift = m_new == -INFINITY ? 0.0f : m_new - kShift;
                    if (__any_sync(0xFFFFFFFFu, m_new > m)) {
                        const float down = ex2(m - (m_new == -INFINITY ? 0.0f : m_new));
                        l *= down;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            acc[i][0] *= down;
                            acc[i][1] *= down;
                            acc[i][2] *= down;
                            acc[i][3] *= down;
                        }
                        m = m_new;
                    }
#pragma unroll
                    for (int n = 0; n < kPairs; ++n) {
                        float w[4];
                        uint32_t a[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            w[j] = ex2(s[2 * n + j / 2][j % 2] - shift);
                            l += w[j];
                        }
                        split<T>(w[0], w[1], a[0], a[1]);
                        split<T>(w[2], w[3], a[2], a[3]);
                        // a value that does not count may be NaN, and its weight of zero would not remove it
                        uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
                        if (ragged) {
                            const int k = n * 16 + 2 * t;
                            keep0 = (k < keys ? 0xFFFFu : 0u) | (k + 1 < keys ? 0xFFFF0000u : 0u);
                            keep1 = (k + 8 < keys ? 0xFFFFu : 0u) | (k + 9 < keys ? 0xFFFF0000u : 0u);
                        }
#pragma unroll
                        for (int i = 0; i < kSteps; ++i) {
                            uint32_t b[4];
                            ldmatrix_x4_trans(base + v_row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix / 2) ^ row8) << 4), b);
                            mma_m16n8k16<kBf16>(acc[2 * i], a[0], a[1], a[2], a[3], b[0] & keep0, b[1] & keep1);
                            mma_m16n8k16<kBf16>(acc[2 * i + 1], a[0], a[1], a[2], a[3], b[2] & keep0, b[3] & keep1);
                        }
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
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
            if (bad) {
                l = NAN;
            }
            if (t == 0) {
                group_ml[part * kHeads + g] = make_float2(m, l);
            }
            named_barrier_sync(1 + group, Cfg::kWarps * 32);
            float m_all = -INFINITY;
#pragma unroll
            for (int w = 0; w < Cfg::kWarps; ++w) {
                m_all = fmaxf(m_all, group_ml[w * kHeads + g].x);
            }
            const float down = ex2(m - (m_all == -INFINITY ? 0.0f : m_all));
            const bool whole = walk.count == walk.units;
            const int slot = walk.first > 0 || walk.left == u1 - u0 ? 0 : 1;
#pragma unroll
            for (int c = 0; c < Cfg::kHalves; ++c) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float* a = acc[c * 8 + i];
                    *reinterpret_cast<float2*>(my_join + g * kPadded + i * 8 + 2 * t) =
                        make_float2((a[0] + a[2]) * down, (a[1] + a[3]) * down);
                }
                named_barrier_sync(1 + group, Cfg::kWarps * 32);
                // a thread takes four columns at a time
                for (int i = part * 32 + lane; i < kHeads * 16; i += Cfg::kWarps * 32) {
                    const int h = i / 16, column = (i % 16) * 4;
                    const int head = (walk.hh % p.head_units) * kUnitHeads + group * kHeads + h;
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float m_h = -INFINITY, l_h = 0.0f;
#pragma unroll
                    for (int w = 0; w < Cfg::kWarps; ++w) {
                        const float4 x = *reinterpret_cast<const float4*>(
                            join + ((group * Cfg::kWarps + w) * kHeads + h) * kPadded + column);
                        sum.x += x.x;
                        sum.y += x.y;
                        sum.z += x.z;
                        sum.w += x.w;
                        m_h = fmaxf(m_h, group_ml[w * kHeads + h].x);
                    }
                    const float base = m_h == -INFINITY ? 0.0f : m_h;
#pragma unroll
                    for (int w = 0; w < Cfg::kWarps; ++w) {
                        const float2 ml = group_ml[w * kHeads + h];
                        l_h += ml.y * ex2(ml.x - base);
                    }
                    if (head < p.group) {
                        if (whole) {
                            const int64_t row = (int64_t)walk.r * p.heads + kv * p.group + head;
                            const float by = 1.0f / l_h;
                            uint2 out;
                            out.x = pack<T>(sum.x * by, sum.y * by);
                            out.y = pack<T>(sum.z * by, sum.w * by);
                            *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + row * D + c * 64 + column) = out;
                            if (p.lse && c == 0 && column == 0) {
                                p.lse[row] = (base - kShift + log2f(l_h)) * kLn2;
                            }
                        } else {
                            const int64_t row = ((int64_t)blockIdx.x * 2 + slot) * kUnitHeads + group * kHeads + h;
                            *reinterpret_cast<float4*>(p.part_o + row * D + c * 64 + column) = sum;
                            if (c == 0 && column == 0) {
                                p.part_ml[row] = make_float2(m_h, l_h);
                            }
                        }
                    }
                }
                named_barrier_sync(1 + group, Cfg::kWarps * 32);
            }
        }
        // requests without units: no keys, or lengths that cannot be
        for (int r = blockIdx.x; r < p.requests; r += gridDim.x) {
            if (units_of(p, r) == 0) {
                const bool empty = p.lengths[r] == 0;
                const uint32_t fill = empty ? 0u : pack<T>(NAN, NAN);
                uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + (int64_t)r * p.heads * D);
                for (int i = threadIdx.x; i < p.heads * (D / 2); i += Cfg::kCompute * 32) {
                    o[i] = fill;
                }
                for (int i = threadIdx.x; p.lse && i < p.heads; i += Cfg::kCompute * 32) {
                    p.lse[(int64_t)r * p.heads + i] = empty ? -INFINITY : NAN;
                }
            }
        }
    }
}

// Joins the parts of one query head of a (request, head unit): block x of the first kernel named them in joins[x].
template <int D, typename T>
__global__ void __launch_bounds__(kJoinThreads) attn_paged_join_kernel(const Params p, int unit_heads)
{
    constexpr int kLanes = D / 4, kRows = kJoinThreads / kLanes;  // threads along a part's columns; parts at a time
    __shared__ float weight[kMaxBlocks + 1];
    __shared__ float2 seen[kJoinThreads / 32];
    __shared__ float4 sums[kRows][kLanes];
    grid_dependency_wait();
    grid_launch_dependents();
    const int4 j = p.joins[blockIdx.x];
    const int h = blockIdx.y, head = (j.y % p.head_units) * unit_heads + h;
    if (j.x < 0 || head >= p.group) {
        return;
    }
    const int parts = j.z - (int)blockIdx.x + 2;  // of blocks blockIdx.x - 1 .. j.z
    auto row_of = [&](int i) {
        return (((int64_t)blockIdx.x - 1 + i) * 2 + (i == 0 ? j.w : 0)) * unit_heads + h;
    };
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    float most = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) {
        most = fmaxf(most, p.part_ml[row_of(i)].x);
    }
    for (int d = 16; d > 0; d /= 2) {
        most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    }
    if (lane == 0) {
        seen[warp].x = most;
    }
    __syncthreads();
    for (int w = 0; w < kJoinThreads / 32; ++w) {
        most = fmaxf(most, seen[w].x);
    }
    const float base = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < parts; i += kJoinThreads) {
        const float2 ml = p.part_ml[row_of(i)];
        weight[i] = ex2(ml.x - base);
        sum += ml.y * weight[i];
    }
    for (int d = 16; d > 0; d /= 2) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    }
    if (lane == 0) {
        seen[warp].y = sum;
    }
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < kJoinThreads / 32; ++w) {
        sum += seen[w].y;
    }
    const int column = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = first; i < parts; i += kRows) {
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + row_of(i) * D + column * 4);
        const float w = weight[i];
        v.x += x.x * w;
        v.y += x.y * w;
        v.z += x.z * w;
        v.w += x.w * w;
    }
    sums[first][column] = v;
    __syncthreads();
    if (threadIdx.x < kLanes) {
        for (int i = 1; i < kRows; ++i) {
            const float4 x = sums[i][column];
            v.x += x.x;
            v.y += x.y;
            v.z += x.z;
            v.w += x.w;
        }
        const int64_t row = (int64_t)j.x * p.heads + (j.y / p.head_units) * p.group + head;
        const float by = 1.0f / sum;
        uint2 out;
        out.x = pack<T>(v.x * by, v.y * by);
        out.y = pack<T>(v.z * by, v.w * by);
        *reinterpret_cast<uint2*>(static_cast<T*>(p.o) + row * D + column * 4) = out;
        if (p.lse && threadIdx.x == 0) {
            p.lse[row] = (base - kShift + log2f(sum)) * kLn2;
        }
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
static int blocks_of(int groups, int sm_count) { return (groups == 1 ? 2 : 1) * sm_count; }

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
    const cuuint32_t box[5] = {64, (cuuint32_t)(c.page_size < kTile ? c.page_size : kTile), (cuuint32_t)(c.head_dim / 64), 1, 1};
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
    const int blocks = blocks_of(kGroups, dev.sm_count);
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = launch_config(&attr, dim3(blocks), Cfg::kThreads, Cfg::kSmem, stream);
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
    return Workspace(blocks_of(groups, dev->sm_count), groups, head_dim).bytes;
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
    const int group = a.heads / c.kv_heads, groups = groups_of(group), blocks = blocks_of(groups, dev->sm_count);
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
    p.box_rows = c.page_size < kTile ? c.page_size : kTile;
    p.scale_log2e = a.scale * kLog2e;
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    p.joins = reinterpret_cast<int4*>(ws + w.joins);
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    p.part_o = reinterpret_cast<float*>(ws + w.o);
    p.status = dev->status_word;
    // one unit at most for every request: nothing to join
    const bool joined = (int64_t)a.max_blocks * c.page_size > kTile;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = a.q_type == SPORK_TYPE_F32;
    if (c.type == SPORK_TYPE_F16) {
        return c.head_dim == 64 ? launch_q<64, __half>(f32, groups, map_k, map_v, p, joined, *dev, s)
                                : launch_q<128, __half>(f32, groups, map_k, map_v, p, joined, *dev, s);
    }
    return c.head_dim == 64 ? launch_q<64, __nv_bfloat16>(f32, groups, map_k, map_v, p, joined, *dev, s)
                            : launch_q<128, __nv_bfloat16>(f32, groups, map_k, map_v, p, joined, *dev, s);
}
