// Attention of one new token per request over a paged key-value cache, for sm_100a:
//   o[r][h] = softmax(scale q[r][h] K^T) V over the keys that request r holds, key head h / (heads / kv_heads).
//
// Every key and value is read once for up to 32 query heads that share it, and once more for every further 32.  With up
// to 16 of them the products are small and the kernel is bound by HBM; from 17 on it is bound by the products, as every
// instruction takes 8 heads (48 requests of 700..5003 keys, 2 key heads of 64: 20.3 us with 16 heads to one, 29 with
// 32, 43 with 64, 75 with 128, of 10.4 to 11.5 that the bytes take).  Work is cut along the cache: units of 64 keys (128
// with a head dimension of 64: 32 KB of keys and values) of one (request, key head), all units in one list, request by
// request, and each block of the grid takes an equal run of that list, whatever the lengths (they are known on the
// device only).  A block joins what it computes of one (request, key head) and writes the result if it has all of it.
// Otherwise it leaves a partial result (running maximum, sum, unnormalised output) in the workspace and counts itself
// in; the block that comes last joins the parts, in the order of the keys.  So one launch does, and what is added to
// what does not depend on who was last.
//
// One warp copies the pages with TMA: the cache is a 5-dimensional tensor (64 elements, page rows, halves of the head
// dimension, heads, pages) with the strides that it has, so any order in memory is one tensor map; a box is a page's
// rows of one head (64 rows of it at most), swizzled for ldmatrix.  Page numbers come from the block table, and are
// checked before they are used.  With a unit goes a note that says what it is; only the copying warp walks the list.
//
// Four warps compute, each on keys of its own, with mma.m16n8k16.  Up to 8 query heads are rows 0-7 of the 16-row
// operand, and rows 8-15 hold what rounding to 16 bits left over: of q, if it is fp32, and of the softmax weights.  So
// both products are taken with about 22 (fp16) or 16 (bf16) bits of q and of the weights at no cost: the rows would
// have been empty, and the weights' rounding, the largest error of the usual scheme, is gone.  (Rows of fp32 queries are
// brought into the 16-bit type's range by a power of two first.)  (tcgen05 would want 64 or 128 rows and a trip through
// tensor memory for every unit; up to 16 heads to one the warp instruction's rate is several times what the loads feed.)
// With 9 or more query heads to a key head the warps form 2 or 4 groups that share the unit, 8 heads each.  Each warp
// runs its own online softmax.  Its maximum follows the scores lazily: only when one has grown by more than 2^8 over it are the row's
// lanes asked and the sums rescaled, so most units need no exchange between lanes at all.  The warps of a group are
// joined once per (request, key head): each gets the others' sums for its share of the columns, and writes that (or
// leaves it in the workspace, and joins that share of the parts).
//
// Measured (us a launch, in a stream of them; the share of the measured copy rate): 64 requests of 4096..8192 keys, 64
// query and 8 key heads of 128, bf16, 1.68 GB: 245..254 (101..105 %); 16 of 4096 keys, 16 heads of 128, 537 MB:
// 85..88 (93..96 %); one of 131072 keys, 32 / 8 heads: 85..88 (93..96 %); 23 of 1..6001 keys, 40 / 8 heads, fp32 q: 46..48 (80..83 %);
// 256 of 8..64 keys, 64 / 8 heads of 128, where each block has 6 or 7 short (request, key head)s one behind the other:
// 18.5 (39 %).  Of a short launch's time about 1.5 us pass until a block knows its run (one trip to memory and a scan),
// 2 until its first keys are there, and 1.5 to 2.5 in the joining of parts.  ncu (16 requests of the first shape, 8
// heads to one): no local memory, mma.sync at 17 % of its peak rate; of 11.5 warps between two instructions 5.9 wait
// for memory and 2.5 for a fixed latency.
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
constexpr int kMaxBlocks = 512;    // blocks of a launch
constexpr int kComputeWarps = 4;
// the computing warps, the copying one, and three idle ones that complete the second warpgroup, so that whole warpgroups
// can trade registers
constexpr int kThreads = 256;
constexpr int kBlocksPerSm = 2;
constexpr int kComputeRegs = 192, kCopyRegs = 64;
// setmaxnreg.inc waits, without a limit, for registers to be free: the trade must fit what the block was launched with
static_assert(kComputeRegs + kCopyRegs <= 2 * (65536 / (kThreads * kBlocksPerSm)), "register trade exceeds the launch allocation");
// What a (request, key head) costs a block besides its units, in units: its end takes about as long as a unit's work.
constexpr int kPairCost = 1;
// A (request, key head) of so many units or fewer is not cut: joining parts takes longer than three units do (one request of
// 317 keys, units of 128: 6.5 us whole, 7.5 in three parts).
constexpr int kWhole = 4;
// Places of a block's run, at least: of 4, short requests queue up behind one another (4 requests of 128 keys, 8 key heads:
// 6.6 us with 2, 9.4 with 4); of 1, long ones come to more parts (no slower where measured, but never faster).
constexpr int kMinRun = 2;
constexpr int kMaxRows = 64;       // rows of a TMA box
constexpr int kLengths = 512;      // requests whose lengths a block keeps in shared memory
// Parts that are joined at a time.  One request of 8192 keys on all SMs, 37 parts: 13.3 us with 10, 13.5 with 16, 14.4 with 40
// in one step.
constexpr int kFan = 10;
constexpr int kLevels = 3;         // of joining: kFan^kLevels is more than the blocks of a launch

// kGroups groups of warps share a unit, each with 8 query heads of its own.
template <int D, int kGroups>
struct Config {
    static constexpr int kTile = 8192 / D;                      // keys per unit
    static constexpr int kWarps = kComputeWarps / kGroups;      // warps of a group; each takes kTile / kWarps keys
    static constexpr int kKeys = kTile / kWarps;
    static constexpr int kChunk = kKeys < 32 ? kKeys : 32;      // taken at once
    static constexpr int kHalfUnit = kTile * D * 2;             // the keys (or values) of a unit, bytes
    static constexpr int kStageBytes = 2 * kHalfUnit;
    // Two: with three the loads of SMs that are served better crowd out those of the others, and equal runs end up to a
    // fifth of their time apart (16 requests of 4096 keys, 16 heads of 128: 89.0 us with three, 85.6 with two).
    static constexpr int kStages = 2;
    static constexpr int kShare = D / 8 / kWarps;               // groups of 8 columns that a warp joins
    static constexpr int kHanded = kHeads * kShare * 8;         // floats from one warp to another
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kComputeWarps * (kWarps - 1) * kHanded * 4;
};

struct Params {
    const void* q;
    const int32_t* table;
    const int32_t* lengths;
    void* o;
    float* lse;
    int64_t q_request_stride, q_head_stride, table_stride;
    int32_t requests, heads, kv_heads, group, head_units;  // group: query heads per key head; head_units: units along them
    int32_t capacity;  // keys that a table row has room for (2^31 - 1 at most)
    int32_t num_pages, page_size, box_rows;
    float scale_log2e;
    bool q_pairs;  // two neighbouring elements of q may be read at once
    // workspace
    uint32_t* arrived; // [level][block][slot][warp]: parts that are there, of those whose first one is that; zero between calls
    float2* part_ml;   // [block][slot][warp][head]: maximum, sum
    float* part_o;     // [block][slot][warp][lane][the lane's columns of the warp's share of D]
    uint32_t* status;
};

// What a unit is.
struct alignas(16) Note {
    int r, kv, head;         // request, key head, first of the unit's query heads among those of the key head
    int keys;                // keys that count from the unit's first one on (may be more than it has)
    int position, count;     // which of the block's units of this (request, key head), and how many those are
    int flags;               // bits as below
    int parts, first;        // the blocks that have units of this (request, key head): how many, and the first one
    int next_r, next_kv, next_head;  // with the last of the block's units: what comes next (-1: nothing)
};
// nothing more; the first part is a later one of its block's (is_later); a bad page
constexpr int kDone = 1, kFirstLater = 2, kBad = 4;

struct Bars {
    uint64_t full[4], empty[4];
    uint64_t handed[kComputeWarps], taken[kComputeWarps];  // a group's warps have handed over, and taken, what is for each
    Note note[4];
    uint32_t warp_sums[8];
    uint32_t start[3];       // the block's first (request, head unit): request, which head unit, its place in the list
    float2 ml[kComputeWarps][kHeads];  // each warp's maxima and sums
    int32_t lengths[kLengths];  // of the first requests
    uint32_t abort_flag;
};
static_assert(kBlocksPerSm * (Config<128, 1>::kSmem + (int)sizeof(Bars) + 1024) <= 228 * 1024, "shared memory of the blocks of an SM");

// Units of a request: none if there is nothing to read, or nothing that may be read.
template <int kTile>
__host__ __device__ __forceinline__ int units_of(const Params& p, int len)
{
    return len > 0 && len <= p.capacity ? (int)(((uint32_t)len + kTile - 1) / kTile) : 0;
}

// The list cut into equal runs: block b's begins at place b * total / blocks.  (The host has made sure that a list has
// fewer than 2^31 places.)
struct Cut {
    uint32_t total, blocks, each, rest;
    __host__ __device__ __forceinline__ Cut(uint32_t places, uint32_t grid)
        : total(places), blocks(places < grid * kMinRun ? (places + kMinRun - 1) / kMinRun : grid)
    {
        each = blocks ? total / blocks : 0;
        rest = total - each * blocks;
    }
    __host__ __device__ __forceinline__ uint32_t begin(uint32_t b) const { return b * each + b * rest / blocks; }
    // the block whose run has a place
    __host__ __device__ __forceinline__ uint32_t at(uint32_t place) const
    {
        return (uint32_t)(((uint64_t)(place + 1) * blocks - 1) / total);
    }
};

// A block's run through the list, one (request, head unit) after the other.  Each takes its units' places in the list
// and kPairCost more.  One of kWhole units or fewer belongs to the block that has its middle unit's place.
template <int kTile>
struct Walk {
    int r, kv, hu, first, count, units, len;
    uint32_t base, from, end;  // places in the list: of the current one's first unit, of the run's begin and end

    __host__ __device__ __forceinline__ void here()
    {
        if (units <= kWhole) {
            const uint32_t middle = base + units / 2;
            first = 0;
            count = middle >= from && middle < end ? units : 0;
        } else {
            first = from > base ? (int)(from - base) : 0;
            const int last = (int)(end - base) < units ? (int)(end - base) : units;
            count = last > first ? last - first : 0;
        }
    }
    // to the next one; false at the run's end
#pragma nv_exec_check_disable
    template <typename Length>
    __host__ __device__ __forceinline__ bool next(const Params& p, const Length& length)
    {
        base += units + kPairCost;
        if (base >= end) {
            return false;
        }
        if (++hu == p.head_units) {
            hu = 0;
            if (++kv == p.kv_heads) {
                kv = 0;
                do {
                    if (++r >= p.requests) {
                        return false;
                    }
                    len = length(r);
                    units = units_of<kTile>(p, len);
                } while (units == 0);
            }
        }
        here();
        return true;
    }
};

// Where a block's part of a (request, head unit) goes in the workspace: a run that begins in front of it (and of its
// predecessor's cost) has other units first, and at its begin it may have a part of those.
__host__ __device__ __forceinline__ bool is_later(uint32_t from, uint32_t base) { return from + kPairCost < base; }

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

// What one warp has of its 8 query heads and a run of keys: maxima, sums, unnormalised output (fragments: row g of the
// first product's operand is in [0], [1], row g + 8, its low part, in [2], [3]); and the weights of the unit at hand.
template <int D, typename T, bool kLowQ, int kKeys>
struct Softmax {
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kSteps = D / 16, kPairs = kKeys / 16;
    uint32_t q_hi[kSteps][2], q_lo[kLowQ ? kSteps : 1][2];
    float acc[D / 8][4];
    float m, l;  // of row g; l: this lane's columns only
    float row_scale;  // kLowQ: what turns a score of row g into a power of two's exponent
    uint32_t weights[kPairs][4];

    // The queries as they are (kLowQ: 32 bits), on their way into the registers that begin() makes operands of.  Nothing is
    // done with what is loaded, so that nothing waits for it here.  `pairs`: two neighbours may be read at once.
    template <typename Q>
    __device__ __forceinline__ void ask_for(const Q* q, bool pairs)
    {
        if (pairs) {
#pragma unroll
            for (int i = 0; i < 2 * kSteps; ++i) {
                if constexpr (kLowQ) {
                    const uint2 x = *reinterpret_cast<const uint2*>(q + i * 8);
                    q_hi[i / 2][i % 2] = x.x;
                    q_lo[i / 2][i % 2] = x.y;
                } else {
                    q_hi[i / 2][i % 2] = *reinterpret_cast<const uint32_t*>(q + i * 8);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kSteps; ++i) {
                if constexpr (kLowQ) {
                    q_hi[i / 2][i % 2] = reinterpret_cast<const uint32_t*>(q)[i * 8];
                    q_lo[i / 2][i % 2] = reinterpret_cast<const uint32_t*>(q)[i * 8 + 1];
                } else {
                    const uint16_t* x = reinterpret_cast<const uint16_t*>(q) + i * 8;
                    q_hi[i / 2][i % 2] = x[0] | (uint32_t)x[1] << 16;
                }
            }
        }
    }

    // (kLowQ) Each row is brought by a power of two, which its scale takes back, to where two 16-bit parts hold it: the
    // exponent of its largest finite element becomes 14 in fp16, so that elements down to 2^-17 of that one keep 22 bits and
    // no smaller one is off by more than 2^-39 of it; bf16 has fp32's range, and only rows near its ends are moved.  (Sums
    // of products with keys of any size stay within fp32 then, too.)
    __device__ __forceinline__ void begin(float scale)
    {
        if constexpr (kLowQ) {
            constexpr int kLeast = kBf16 ? -60 : 14, kMost = kBf16 ? 60 : 14;
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t x = q_hi[i][j] & 0x7FFFFFFFu, y = q_lo[i][j] & 0x7FFFFFFFu;
                    most = max(most, x < 0x7F800000u ? x : 0u);
                    most = max(most, y < 0x7F800000u ? y : 0u);
                }
            }
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
            const int exponent = max((int)(most >> 23), 1) - 127;
            // -113 .. 140: in two factors within range
            const int up = most > 0 ? max(kLeast, min(kMost, exponent)) - exponent : 0;
            const int up0 = up / 2, up1 = up - up0;
            const float by0 = __int_as_float((127 + up0) << 23), by1 = __int_as_float((127 + up1) << 23);
            row_scale = scale * __int_as_float((127 - up0) << 23) * __int_as_float((127 - up1) << 23);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    split<T>(__uint_as_float(q_hi[i][j]) * by0 * by1, __uint_as_float(q_lo[i][j]) * by0 * by1, q_hi[i][j], q_lo[i][j]);
                }
            }
        }
    }

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        }
        m = -INFINITY;
        l = 0.0f;
    }

    // Weights of a unit's keys, whose rows for ldmatrix are at `row`; `keys` of them count (kRagged: not all, and the rest
    // may be anything).
    template <bool kRagged>
    __device__ __forceinline__ void take_keys(const uint32_t (&row)[kPairs], uint32_t base, uint32_t half, int keys, float scale_log2e)
    {
        const float scale = kLowQ ? row_scale : scale_log2e;
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
                if (!kRagged || n * 16 < keys) {
                    uint32_t b[4];
                    ldmatrix_x4(base + row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix % 2) ^ row8) << 4), b);
                    const uint32_t a1 = kLowQ ? q_lo[kLowQ ? i : 0][0] : 0u, a3 = kLowQ ? q_lo[kLowQ ? i : 0][1] : 0u;
                    mma_m16n8k16<kBf16>(s[2 * n], q_hi[i][0], a1, q_hi[i][1], a3, b[0], b[1]);
                    mma_m16n8k16<kBf16>(s[2 * n + 1], q_hi[i][0], a1, q_hi[i][1], a3, b[2], b[3]);
                }
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
            const bool nothing_yet = __all_sync(0xFFFFFFFFu, m == -INFINITY);
            m = most;
            if (!nothing_yet) {
                l *= down;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    acc[i][0] *= down;
                    acc[i][1] *= down;
                    acc[i][2] *= down;
                    acc[i][3] *= down;
                }
            }
        }
        const float shift = m == -INFINITY ? 0.0f : kShift - m;
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = ex2(fmaf(s[2 * n + j / 2][j % 2], scale, shift));
                l += w[j];
            }
            split<T>(w[0], w[1], weights[n][0], weights[n][1]);
            split<T>(w[2], w[3], weights[n][2], weights[n][3]);
        }
    }

    // The same unit's values.
    template <bool kRagged>
    __device__ __forceinline__ void take_values(const uint32_t (&row)[kPairs], uint32_t base, uint32_t half, int keys)
    {
        const int lane = threadIdx.x % 32, t = lane % 4, matrix = lane / 8, row8 = lane % 8;
#pragma unroll
        for (int n = 0; n < kPairs; ++n) {
            if (kRagged && n * 16 >= keys) {
                continue;
            }
            const uint32_t(&a)[4] = weights[n];
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
                ldmatrix_x4_trans(base + row[n] + (i / 4) * half + ((((i % 4) * 2 + matrix / 2) ^ row8) << 4), b);
                mma_m16n8k16<kBf16>(acc[2 * i], a[0], a[1], a[2], a[3], kRagged ? b[0] & keep0 : b[0],
                                    kRagged ? b[1] & keep1 : b[1]);
                mma_m16n8k16<kBf16>(acc[2 * i + 1], a[0], a[1], a[2], a[3], kRagged ? b[2] & keep0 : b[2],
                                    kRagged ? b[3] & keep1 : b[3]);
            }
        }
    }
};

// A warp's share of a result: lane (g, t) has row g's columns 8 i + 2 t and + 1 of it, and the row's maximum and sum.
template <int kShare>
struct Part {
    float2 o[kShare];
    float m, l;

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < kShare; ++i) {
            o[i] = make_float2(0.0f, 0.0f);
        }
        m = -INFINITY;
        l = 0.0f;
    }

    // With others, in order: one common maximum, so that the weights do not wait for one another.  (One that is not there has
    // the maximum -infinity, the sum 0 and an output of 0.)
    template <int kMost>
    __device__ __forceinline__ void join(const float2 (&ml)[kMost], const float2 (&its_o)[kMost][kShare])
    {
        float most = m;
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            most = fmaxf(most, ml[j].x);
        }
        const float to = most == -INFINITY ? 0.0f : most, down = ex2(m - to);
        l *= down;
#pragma unroll
        for (int i = 0; i < kShare; ++i) {
            o[i].x *= down;
            o[i].y *= down;
        }
        m = most;
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            const float its = ex2(ml[j].x - to);
            l += ml[j].y * its;
#pragma unroll
            for (int i = 0; i < kShare; ++i) {
                o[i].x += its_o[j][i].x * its;
                o[i].y += its_o[j][i].y * its;
            }
        }
    }
};

// A row of the output: the share's columns from `o` on, and where `lse` is not null the logarithm of the sum.
template <typename T, int kShare>
__device__ __forceinline__ void write_result(const Part<kShare>& all, T* o, float* lse)
{
    const int t = threadIdx.x % 4;
    const float by = 1.0f / all.l;
    uint32_t* out = reinterpret_cast<uint32_t*>(o) + t;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
        out[i * 4] = pack<T>(all.o[i].x * by, all.o[i].y * by);
    }
    if (lse && t == 0) {
        *lse = ((all.m == -INFINITY ? 0.0f : all.m) - kShift + log2f(all.l)) * kLn2;
    }
}

// A part in the workspace: maxima and sums by head, and each lane's columns side by side.
template <int kShare>
__device__ __forceinline__ void write_part(const Part<kShare>& all, float2* part_ml, float* part_o, uint32_t place)
{
    const int lane = threadIdx.x % 32;
    float4* out = reinterpret_cast<float4*>(part_o) + (place * 32 + lane) * (kShare / 2);
#pragma unroll
    for (int i = 0; i < kShare / 2; ++i) {
        __stcg(out + i, make_float4(all.o[2 * i].x, all.o[2 * i].y, all.o[2 * i + 1].x, all.o[2 * i + 1].y));
    }
    if (lane % 4 == 0) {
        __stcg(part_ml + place * kHeads + lane / 4, make_float2(all.m, all.l));
    }
}

// (Predicated, not branched around: with branches the compiler keeps more registers than there are.)
template <int kShare>
__device__ __forceinline__ void read_part(float2& ml, float2 (&o)[kShare], const float2* part_ml, const float* part_o,
                                          uint32_t place, bool there)
{
    const int lane = threadIdx.x % 32;
    const float4* from = reinterpret_cast<const float4*>(part_o) + (place * 32 + lane) * (kShare / 2);
    ml = make_float2(-INFINITY, 0.0f);
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %3, 0;\n\t"
        "@p ld.global.cg.v2.f32 {%0, %1}, [%2];\n\t"
        "}"
        : "+f"(ml.x), "+f"(ml.y)
        : "l"(part_ml + place * kHeads + lane / 4), "r"((int)there));
#pragma unroll
    for (int i = 0; i < kShare; i += 2) {
        o[i] = o[i + 1] = make_float2(0.0f, 0.0f);
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %5, 0;\n\t"
            "@p ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];\n\t"
            "}"
            : "+f"(o[i].x), "+f"(o[i].y), "+f"(o[i + 1].x), "+f"(o[i + 1].y)
            : "l"(from + i / 2), "r"((int)there));
    }
}

// Where part i of those of blocks first .. is: the first one in that block's slot first_slot, the others in slot 0.
__device__ __forceinline__ uint32_t place_of(int first, int first_slot, int i)
{
    return ((first + i) * 2 + (i == 0 ? first_slot : 0)) * kComputeWarps + threadIdx.x / 32;
}

// A warp counts its share of this block's part in, which it has written.  The last of every kFan joins these in order and
// leaves the result where the first of them was, and so on; the last of all writes the row of the output (o null: there is
// none).  (The main loop bears no spills for this: with 200 bytes of them to a thread the kernel took up to 1.4 times as
// long, since little of L1 is left beside the stages.  ptxas reports none, but for 20 bytes stored and 24 loaded where 9 to 16
// heads of 128 with 16-bit queries share a key head; where those are was not looked at.)
template <typename T, int kShare>
__device__ __forceinline__ void join_parts(uint32_t* arrived, float2* part_ml, float* part_o, int first, int parts,
                                           int first_slot, T* o, float* lse)
{
    const int lane = threadIdx.x % 32;
    int mine = (int)blockIdx.x - first, step = 1;  // part i of a level is where part i * step of the lowest one was
    for (int n = parts; n > 1; n = (n + kFan - 1) / kFan, step *= kFan, mine /= kFan) {
        const int begin = mine / kFan * kFan, members = n - begin < kFan ? n - begin : kFan;
        if (members > 1) {
            uint32_t* counter = arrived + place_of(first, first_slot, begin * step);
            __syncwarp();
            uint32_t before = 0;
            if (lane == 0) {
                // releases what the warp has written, and acquires what the others had when they counted themselves in
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
            }
            before = __shfl_sync(0xFFFFFFFFu, before, 0);
            __syncwarp();
            if (before != (uint32_t)members - 1u) {
                return;
            }
            if (lane == 0) {
                *counter = 0u;  // for the next launch
            }
            Part<kShare> all;
            all.clear();
            constexpr int kAtOnce = kShare <= 4 ? 8 : kShare == 8 ? 4 : 2;
            for (int k = 0; k < members; k += kAtOnce) {
                float2 ml[kAtOnce], x[kAtOnce][kShare];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    read_part(ml[j], x[j], part_ml, part_o, place_of(first, first_slot, (begin + k + j) * step), k + j < members);
                }
                all.join(ml, x);
            }
            if (n <= kFan) {
                if (o) {
                    write_result(all, o, lse);
                }
                return;
            }
            write_part(all, part_ml, part_o, place_of(first, first_slot, begin * step));
        }
        arrived += gridDim.x * 2 * kComputeWarps;  // (one alone is its own join, where it is)
    }
}

template <int D, typename T, typename Q, int kGroups>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    attn_paged_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p)
{
    using Cfg = Config<D, kGroups>;
    constexpr bool kLowQ = std::is_same<Q, float>::value;  // q has a low part
    constexpr int kUnitHeads = kGroups * kHeads;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Bars bars;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const uint32_t stages = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t handed = stages + Cfg::kStages * Cfg::kStageBytes;
    volatile uint32_t* abort_flag = &bars.abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(smem_u32(&bars.full[s]), 1);
            mbar_init(smem_u32(&bars.empty[s]), kComputeWarps);
        }
        for (int g = 0; g < kGroups; ++g) {
            mbar_init(smem_u32(&bars.handed[g]), Cfg::kWarps);
            mbar_init(smem_u32(&bars.taken[g]), Cfg::kWarps);
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
    const int chunk = (p.requests + kThreads - 1) / kThreads;
    const int r0 = (int)threadIdx.x * chunk, r1 = r0 + chunk < p.requests ? r0 + chunk : p.requests;
    const auto places_of = [&](int len) {
        const int units = units_of<Cfg::kTile>(p, len);
        return units ? (uint32_t)(units + kPairCost) * hhs : 0u;
    };
    uint32_t mine = 0;  // places of this thread's requests
    for (int r = r0; r < r1; ++r) {
        const int len = p.lengths[r];
        if (r < kLengths) {
            bars.lengths[r] = len;
        }
        mine += places_of(len);
    }
    const auto length = [&](int r) { return r < kLengths ? bars.lengths[r] : p.lengths[r]; };
    uint32_t base = mine, places = 0;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t w = __shfl_up_sync(0xFFFFFFFFu, base, d);
        base += lane >= d ? w : 0;
    }
    if (lane == 31) {
        bars.warp_sums[warp] = base;
    }
    __syncthreads();
    base -= mine;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        base += w < warp ? bars.warp_sums[w] : 0;
        places += bars.warp_sums[w];
    }
    const Cut cut(places, gridDim.x);
    const bool work = blockIdx.x < cut.blocks;
    const uint32_t from = work ? cut.begin(blockIdx.x) : 0;
    if (work && from - base < mine) {
        int r = r0;
        uint32_t its = places_of(length(r));
        while (from - base >= its) {
            base += its;
            its = places_of(length(++r));
        }
        const uint32_t each = its / hhs, hh = (from - base) / each;
        bars.start[0] = r;
        bars.start[1] = hh;
        bars.start[2] = base + hh * each;
    }
    __syncthreads();
    Walk<Cfg::kTile> walk{};
    if (work) {
        walk.r = bars.start[0];
        walk.kv = p.head_units == 1 ? bars.start[1] : bars.start[1] / p.head_units;
        walk.hu = bars.start[1] - walk.kv * p.head_units;
        walk.base = bars.start[2];
        walk.from = from;
        walk.end = cut.begin(blockIdx.x + 1);
        walk.len = length(walk.r);
        walk.units = units_of<Cfg::kTile>(p, walk.len);
        walk.here();
    }
    // to the first (request, head unit) from here on that has units for this block
    auto settle = [&](bool more) {
        while (more && walk.count == 0) {
            more = walk.next(p, length);
        }
        return more;
    };
    bool more = settle(work);

    const int rows = p.box_rows;
    if (warp >= kComputeWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCopyRegs));
        if (warp > kComputeWarps) {
            return;
        }
        // -------------------------------------------------------------------------------------- copies
        const Checker ck{p.status, stages, stages + Cfg::kStages * Cfg::kStageBytes, 0, 0};
        const int boxes = Cfg::kTile / rows;
        const uint32_t box_bytes = rows * D * 2;
        uint32_t stage = 0, phase = 0, used = 0;
        bool ok = true;
        int unit = walk.first;
        // A unit with its note, and this lane's box of it: its page and its first row there.
        struct Plan {
            Note note;
            int page, row;
            bool mine;
        };
        auto look_ahead = [&] {
            Plan plan;
            plan.page = plan.row = 0;
            plan.mine = false;
            plan.note.next_r = -1;
            plan.note.next_kv = plan.note.next_head = 0;
            plan.note.flags = kDone;
            if (!more) {
                return plan;
            }
            const int first = unit * Cfg::kTile, keys = walk.len - first;
            if (lane < boxes && lane * rows < keys) {
                const uint32_t at = (uint32_t)(first + lane * rows), block = at / (uint32_t)p.page_size;
                plan.mine = true;
                plan.row = (int)(at - block * (uint32_t)p.page_size);
                plan.page = p.table[walk.r * p.table_stride + block];
            }
            plan.note.r = walk.r;
            plan.note.kv = walk.kv;
            plan.note.head = walk.hu * kUnitHeads;
            plan.note.keys = keys;
            plan.note.position = unit - walk.first;
            plan.note.count = walk.count;
            plan.note.flags = 0;
            plan.note.parts = 1;
            plan.note.first = 0;
            if (++unit == walk.first + walk.count) {
                if (walk.count != walk.units) {
                    const uint32_t first_block = cut.at(walk.base);
                    plan.note.first = (int)first_block;
                    plan.note.parts = (int)(cut.at(walk.base + walk.units - 1) - first_block) + 1;
                    plan.note.flags = is_later(cut.begin(first_block), walk.base) ? kFirstLater : 0;
                }
                more = settle(walk.next(p, length));
                unit = walk.first;
                if (more) {
                    plan.note.next_r = walk.r;
                    plan.note.next_kv = walk.kv;
                    plan.note.next_head = walk.hu * kUnitHeads;
                }
            }
            return plan;
        };
        // the run's units, then a note of its end; a page is asked for while the two units before its own are copied
        Plan plan = look_ahead(), next = look_ahead();
        while (true) {
            const bool end = plan.note.flags & kDone;
            ok = mbar_wait(smem_u32(&bars.empty[stage]), phase ^ 1u, abort_flag);
            if (!ok && lane == 0) {
                report_timeout(p, abort_flag, 1, stage);
            }
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) {
                break;
            }
            const bool good = plan.mine && plan.page >= 0 && plan.page < p.num_pages;
            const uint32_t bad = __ballot_sync(0xFFFFFFFFu, plan.mine && !good), valid = __ballot_sync(0xFFFFFFFFu, good);
            const uint32_t full = smem_u32(&bars.full[stage]);
            const uint32_t keys = stages + stage * Cfg::kStageBytes + lane * box_bytes;
            if (lane == 0) {
                plan.note.flags |= bad ? kBad : 0;
                bars.note[stage] = plan.note;
                mbar_arrive_expect_tx(full, 2 * box_bytes * __popc(valid));
            }
            __syncwarp();
            if (good && ck.smem(keys, box_bytes, 1024, 0x501) && ck.smem(keys + Cfg::kHalfUnit, box_bytes, 1024, 0x502) &&
                ck.tma_coords(0, 2, plan.row, plan.page, 0x503)) {
                tma_load_5d(keys, &map_k, full, 0, plan.row, 0, plan.note.kv, plan.page);
                tma_load_5d(keys + Cfg::kHalfUnit, &map_v, full, 0, plan.row, 0, plan.note.kv, plan.page);
            }
            ++used;
            if (end) {
                break;
            }
            if (++stage == Cfg::kStages) {
                stage = 0;
                phase ^= 1u;
            }
            plan = next;
            next = look_ahead();
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kComputeRegs));
        const int group = warp / Cfg::kWarps, part = warp % Cfg::kWarps;  // group of warps, warp of the group
        const int g = lane / 4, t = lane % 4;                             // row (query head) and column pair of a fragment
        const int matrix = lane / 8, row8 = lane % 8;
        using S = Softmax<D, T, kLowQ, Cfg::kChunk>;
        constexpr int kPairs = S::kPairs, kChunks = Cfg::kKeys / Cfg::kChunk;
        S sm;
        sm.clear();
        auto ask_for = [&](int r, int kv, int head) {
            // (rows of heads that do not exist get the first one's queries; nobody looks at what they come to)
            const int in_group = head + group * kHeads + g;
            sm.ask_for(static_cast<const Q*>(p.q) + r * p.q_request_stride +
                           (int64_t)(kv * p.group + (in_group < p.group ? in_group : 0)) * p.q_head_stride + 2 * t,
                       p.q_pairs);
        };
        if (more) {
            ask_for(walk.r, walk.kv, walk.hu * kUnitHeads);
        }
        // offsets in a stage of this lane's ldmatrix rows: keys (matrices 0, 1 | 2, 3 are keys 0-7 | 8-15) and values
        // (matrices 0, 2 | 1, 3); a box of `rows` rows holds its halves of 64 columns one behind the other
        auto row_at = [&](int r) { return (uint32_t)((r / rows) * rows * D * 2 + (r % rows) * 128); };
        uint32_t k_row[kChunks][kPairs], v_row[kChunks][kPairs];
        for (int c = 0; c < kChunks; ++c) {
            for (int i = 0; i < kPairs; ++i) {
                const int r = part * Cfg::kKeys + c * Cfg::kChunk + i * 16 + row8;
                k_row[c][i] = row_at(r + (matrix / 2) * 8);
                v_row[c][i] = row_at(r + (matrix % 2) * 8) + Cfg::kHalfUnit;
            }
        }
        const uint32_t half = rows * 128;
        uint32_t stage = 0, phase = 0, times = 0;  // times: that sums have been handed over
        bool ok = true;
        int bad = 0;
        // every lane polls; false if the wait was given up
        auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t role, uint32_t where) {
            const bool done = mbar_wait(smem_u32(bar), parity, abort_flag);
            if (!done) {
                report_timeout(p, abort_flag, role, where);
            }
            return __all_sync(0xFFFFFFFFu, done);
        };

        while (true) {
            ok = wait(&bars.full[stage], phase, 2, stage);
            const Note& note = bars.note[stage];
            const int4 what = *reinterpret_cast<const int4*>(&note.r), which = *reinterpret_cast<const int4*>(&note.position);
            const int4 next = *reinterpret_cast<const int4*>(&note.first);  // first block of the parts; what comes next
            const int left = what.w - part * Cfg::kKeys, flags = which.z;
            if (!ok || (flags & kDone)) {
                break;
            }
            if (which.x == 0) {
                sm.begin(p.scale_log2e);
                bad = 0;
            }
            bad |= flags & kBad;
            const bool last = which.x + 1 == which.y;
            const uint32_t memory = stages + stage * Cfg::kStageBytes;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int keys = left - c * Cfg::kChunk;
                if (keys >= Cfg::kChunk) {
                    sm.template take_keys<false>(k_row[c], memory, half, keys, p.scale_log2e);
                } else if (keys > 0) {
                    sm.template take_keys<true>(k_row[c], memory, half, keys, p.scale_log2e);
                }
                if (c == kChunks - 1 && last && next.y >= 0) {
                    // the old queries have done their work: the next ones arrive while the values are worked on
                    ask_for(next.y, next.z, next.w);
                }
                if (keys >= Cfg::kChunk) {
                    sm.template take_values<false>(v_row[c], memory, half, keys);
                } else if (keys > 0) {
                    sm.template take_values<true>(v_row[c], memory, half, keys);
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
            if (!last) {
                continue;
            }

            // ------------------------------------------------- the warps of the group joined, the result or part written
            // Each warp hands every other one of its group that one's share of the columns, and joins its own.
            float l = sm.l + __shfl_xor_sync(0xFFFFFFFFu, sm.l, 1);
            l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
            l = bad ? NAN : l;
            constexpr int kWarps = Cfg::kWarps, kShare = Cfg::kShare;
            // where row g of what warp `from` has for warp `to` is; groups of 8 columns change places by row (their number
            // is xored to it), so that no two rows' meet in a bank
            auto handed_at = [&](int to, int from) {
                return handed + ((group * kWarps + to) * (kWarps - 1) + (from < to ? from : from - 1)) * (Cfg::kHanded * 4) +
                       (g * kShare + ((kShare == 2 ? g >> 1 : g) & (kShare - 1))) * 32 + t * 8;
            };
            Part<kShare> all;
            all.m = sm.m;
            all.l = l;
            if (kWarps > 1) {
                ok = wait(&bars.taken[group], (times & 1u) ^ 1u, 3, group);
                if (!ok) {
                    break;
                }
            }
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const uint32_t row = handed_at(w, part);
#pragma unroll
                for (int i = 0; i < kShare; ++i) {
                    const float(&a)[4] = sm.acc[w * kShare + i];
                    const float2 o = make_float2(a[0] + a[2], a[1] + a[3]);
                    if (w == part) {
                        all.o[i] = o;
                    } else {
                        st_shared_f2(row ^ (i * 32), o);
                    }
                }
            }
            if constexpr (kWarps > 1) {
                if (t == 0) {
                    bars.ml[warp][g] = make_float2(sm.m, l);
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&bars.handed[group]));
                }
                ok = wait(&bars.handed[group], times & 1u, 4, group);
                if (!ok) {
                    break;
                }
                float2 ml[kWarps - 1], o[kWarps - 1][kShare];
#pragma unroll
                for (int w = 0; w < kWarps - 1; ++w) {
                    const int other = w < part ? w : w + 1;
                    const uint32_t row = handed_at(part, other);
                    ml[w] = bars.ml[group * kWarps + other][g];
#pragma unroll
                    for (int i = 0; i < kShare; ++i) {
                        o[w][i] = ld_shared_f2(row ^ (i * 32));
                    }
                }
                all.join(ml, o);
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(smem_u32(&bars.taken[group]));
                }
                ++times;
            }
            const int in_group = what.z + group * kHeads + g;
            const int64_t row = (int64_t)what.x * p.heads + what.y * p.group + in_group;
            T* o = in_group < p.group ? static_cast<T*>(p.o) + row * D + part * kShare * 8 : nullptr;
            float* lse = p.lse && part == 0 ? p.lse + row : nullptr;
            if (which.w == 1) {
                if (o) {
                    write_result(all, o, lse);
                }
            } else {
                const int first_slot = flags & kFirstLater ? 1 : 0, i = (int)blockIdx.x - next.x;
                write_part(all, p.part_ml, p.part_o, place_of(next.x, first_slot, i));
                join_parts<T, kShare>(p.arrived, p.part_ml, p.part_o, next.x, which.w, first_slot, o, lse);
            }
            sm.clear();  // (here, so that nothing of the old sums is kept through the above)
            __syncwarp();
        }
        if (!ok) {
            // The copying warp may have gone by its end note.  Then only the unit in front of that can be on its way, the one
            // in the other stage having been used by all warps, and a warp that gives up before it lands stands at it here.
            // (The same wait on the copying warp's way out cost 0.4 to 1 % of a launch's time.)
            static_assert(Cfg::kStages == 2, "one unit in front of the end note that may be on its way");
            volatile uint32_t not_aborted = 0;
            mbar_wait(smem_u32(&bars.full[stage]), phase, &not_aborted);
        }
        // requests without units: no keys, or lengths that cannot be
        for (int r = blockIdx.x; r < p.requests; r += gridDim.x) {
            const int len = length(r);
            if (units_of<Cfg::kTile>(p, len) == 0) {
                const uint32_t fill = len == 0 ? 0u : pack<T>(NAN, NAN);
                uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + (int64_t)r * p.heads * D);
                for (int64_t i = threadIdx.x; i < (int64_t)p.heads * (D / 2); i += kComputeWarps * 32) {
                    o[i] = fill;
                }
                for (int64_t i = threadIdx.x; p.lse && i < p.heads; i += kComputeWarps * 32) {
                    p.lse[(int64_t)r * p.heads + i] = len == 0 ? -INFINITY : NAN;
                }
            }
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

// Query heads of a key head are taken 8, 16 or 32 at a time (groups of warps that share the keys in shared memory): the
// fewest that hold them all, as empty rows cost a group's time.  us with 8 / 16 / 32 for 64 requests of 4096..8192 keys, 8 to
// one, D = 128: 245 / 252 / 333; the same with 16 to one, with 16 / 32: 246 / 345.  For 48 requests of 700..5003 keys, D = 64:
// 4 and 8 to one 19.5 / 21.6 / 29.1 and 18.3 / 20.0 / 27.1, 16 to one 20.3 / 27.2.
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

// What the list of units depends on besides the lengths.
static int fill_shape(Params& p, int requests, int heads, int kv_heads, int head_dim, int page_size, int max_blocks)
{
    const int group = heads / kv_heads, unit_heads = groups_of(group) * kHeads;
    p.requests = requests;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.group = group;
    p.head_units = (group + unit_heads - 1) / unit_heads;
    const int64_t capacity = (int64_t)max_blocks * page_size;
    p.capacity = capacity < 0x7FFFFFFF ? (int32_t)capacity : 0x7FFFFFFF;
    // places in the list, at most: of one request (below 2^57), and of all of them
    const int64_t places = (p.capacity / (8192 / head_dim) + 1 + kPairCost) * (int64_t)kv_heads * p.head_units;
    return requests == 0 || places <= 0x7FFFFFFE / requests ? 0 : SPORK_ERR_TOO_LARGE;
}

struct Workspace {
    int64_t ml, o, bytes;
    Workspace(int blocks, int groups, int D)
    {
        const int64_t rows = (int64_t)blocks * 2 * kComputeWarps * kHeads;
        ml = SPORK_ATTN_PAGED_COUNTERS;
        o = ml + rows * 8;
        bytes = o + rows * (D * groups / kComputeWarps) * 4;
    }
};

template <int D, typename T, typename Q, int kGroups>
static int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p, DeviceState& dev, cudaStream_t stream)
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
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_of(dev.sm_count));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, p);
}

template <int D, typename T, typename Q>
static int launch_groups(int groups, const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p,
                         DeviceState& dev, cudaStream_t stream)
{
    return groups == 1   ? launch<D, T, Q, 1>(map_k, map_v, p, dev, stream)
           : groups == 2 ? launch<D, T, Q, 2>(map_k, map_v, p, dev, stream)
                         : launch<D, T, Q, 4>(map_k, map_v, p, dev, stream);
}

template <int D, typename T>
static int launch_q(bool f32, int groups, const CUtensorMap& map_k, const CUtensorMap& map_v, const Params& p,
                    DeviceState& dev, cudaStream_t stream)
{
    return f32 ? launch_groups<D, T, float>(groups, map_k, map_v, p, dev, stream)
               : launch_groups<D, T, T>(groups, map_k, map_v, p, dev, stream);
}

}  // namespace attn_paged_sm100
}  // namespace spork

namespace spork {
namespace attn_paged_sm100 {

// What block `block` of a launch on sm_count SMs works on, as the kernel finds it.
template <int kTile>
static int plan(const Params& p, const int32_t* lengths, uint32_t grid, uint32_t block, int32_t* out, int capacity)
{
    const auto length = [&](int r) { return lengths[r]; };
    const int hhs = p.kv_heads * p.head_units;
    uint32_t places = 0;
    const auto places_of = [&](int r) {
        const int units = units_of<kTile>(p, lengths[r]);
        return units ? (uint32_t)(units + kPairCost) * hhs : 0u;
    };
    for (int r = 0; r < p.requests; ++r) {
        places += places_of(r);
    }
    const Cut cut(places, grid);
    if (block >= cut.blocks) {
        return 0;
    }
    Walk<kTile> walk{};
    walk.from = cut.begin(block);
    walk.end = cut.begin(block + 1);
    while (walk.from - walk.base >= places_of(walk.r)) {
        walk.base += places_of(walk.r++);
    }
    walk.len = lengths[walk.r];
    walk.units = units_of<kTile>(p, walk.len);
    const uint32_t each = walk.units + kPairCost, hh = (walk.from - walk.base) / each;
    walk.base += hh * each;
    walk.kv = hh / p.head_units;
    walk.hu = hh % p.head_units;
    walk.here();
    int n = 0;
    do {
        if (walk.count == 0) {
            continue;
        }
        if (n < capacity) {
            const bool whole = walk.count == walk.units;
            const int first = whole ? (int)block : (int)cut.at(walk.base);
            const int32_t row[9] = {walk.r, walk.kv, walk.hu, walk.first, walk.count, walk.units, first,
                                    whole ? 1 : (int)cut.at(walk.base + walk.units - 1) - first + 1,
                                    !whole && is_later(cut.begin(block), walk.base) ? 1 : 0};
            for (int i = 0; i < 9; ++i) {
                out[n * 9 + i] = row[i];
            }
        }
        ++n;
    } while (walk.next(p, length));
    return n;
}

}  // namespace attn_paged_sm100
}  // namespace spork

extern "C" int spork_attn_sm100_paged_plan(const int32_t* lengths, int requests, int heads, int kv_heads, int head_dim,
                                           int page_size, int max_blocks, int sm_count, int block, int32_t* out, int capacity)
{
    using namespace spork::attn_paged_sm100;
    if (!spork_attn_sm100_paged_supports(heads, kv_heads, head_dim, page_size) || heads == 0 || requests < 0 || max_blocks < 0 ||
        (requests > 0 && !lengths) || sm_count < 1 || block < 0 || block >= blocks_of(sm_count) || capacity < 0 ||
        (capacity > 0 && !out)) {
        return -1;
    }
    Params p{};
    if (fill_shape(p, requests, heads, kv_heads, head_dim, page_size, max_blocks) != 0) {
        return -1;
    }
    const uint32_t grid = (uint32_t)blocks_of(sm_count);
    return head_dim == 128 ? plan<64>(p, lengths, grid, (uint32_t)block, out, capacity)
                           : plan<128>(p, lengths, grid, (uint32_t)block, out, capacity);
}

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
    static_assert(kFan * kFan * kFan >= kMaxBlocks && kLevels == 3, "levels of joining");
    if (blocks > kMaxBlocks || (int64_t)kLevels * blocks * 2 * kComputeWarps * 4 > SPORK_ATTN_PAGED_COUNTERS) {
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
    const int rc4 = fill_shape(p, a.requests, a.heads, c.kv_heads, c.head_dim, c.page_size, a.max_blocks);
    if (rc4) {
        return rc4;
    }
    p.num_pages = c.num_pages;
    p.page_size = c.page_size;
    p.box_rows = c.page_size < kMaxRows ? c.page_size : kMaxRows;
    p.scale_log2e = a.scale * kLog2e;
    uint8_t* ws = static_cast<uint8_t*>(a.workspace);
    p.arrived = reinterpret_cast<uint32_t*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + w.ml);
    p.part_o = reinterpret_cast<float*>(ws + w.o);
    p.status = dev->status_word;
    p.q_pairs = ((reinterpret_cast<uintptr_t>(a.q) % (2 * q_elem)) | ((a.q_request_stride | a.q_head_stride) & 1)) == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f32 = a.q_type == SPORK_TYPE_F32;
    if (c.type == SPORK_TYPE_F16) {
        return c.head_dim == 64 ? launch_q<64, __half>(f32, groups, map_k, map_v, p, *dev, s)
                                : launch_q<128, __half>(f32, groups, map_k, map_v, p, *dev, s);
    }
    return c.head_dim == 64 ? launch_q<64, __nv_bfloat16>(f32, groups, map_k, map_v, p, *dev, s)
                            : launch_q<128, __nv_bfloat16>(f32, groups, map_k, map_v, p, *dev, s);
}
