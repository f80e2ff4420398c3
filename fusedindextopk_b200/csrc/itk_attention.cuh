// Attention of packed, paged and shared-prefix batches on the tensor cores.
//
//     s_j = scale * q . k_j,   m = max_j s_j,   l = sum_j exp(s_j - m),   out = sum_j exp(s_j - m) v_j / l
//
// over the prefix keys (all of them) and the request's own keys (the first min(N, N - Q + i + 1) of them for row i
// of Q when causal).  Scores, statistics and sums are fp32; the weights are rounded to the element type once, for the
// product with the values (half a step of 16 bits each, against the output's own half step), and summed unrounded.  fp16
// weights lose bits below 2^-14, so they are held 2^7 times larger (Element::kHeadroom): what falls below half a step is less than
// 2^-32 of the largest weight a key, instead of 2^-25, of which 131072 keys behind one strong one lost 0.4 % of a sum.
//
// Rows.  The G = heads / kv_heads query heads of a key head share its keys, so one 128-row tile holds TT = 128 / G
// consecutive tokens x G heads (row r = token r / G, head r % G): a single token of a decode step fills G rows of a
// tile instead of one, and a prompt's tile needs its diagonal mask on few key tiles.
//
// Units.  An item is one key head, up to 2 TT tokens and a range of 128-key tiles.
//   pair mode  (more than TT tokens): two row tiles A and B walk the same key tiles; every key tile read from L2
//              serves 256 rows;
//   split mode (at most TT tokens): one row tile; even key tiles go to lane A, odd ones to lane B, which are then two
//              independent softmax states over the same rows, joined like any two partial results.  The tensor work
//              and the softmax of one lane overlap the other's although there is one row tile only.
// A plan kernel (one CTA) turns the lengths on the device into a list of items, longest first, cuts long ones into
// chunks of keys where that spreads the work better, and lays out the partial results; the CTAs of the attention
// kernel take the items from the list as they get free; a third kernel joins the partial results.  Small calls plan
// themselves in the attention kernel (attn_small_plan).  No length is read by the host.
//
// Attention kernel, one CTA per SM, 12 warps: 0-3 softmax of lane A, 4-7 softmax of lane B (one row per thread), 8 and 9
// UMMA issuers of lane A and B, 10 TMA producer (it also takes the items), 11 guard.  A key tile is worked on in two
// steps of 64 keys.  TMEM: two buffers of 64 score columns per lane, so that the scores of step i + 1 are computed while
// the softmax works on step i (the weights P overwrite the first half of their scores as 16-bit pairs and are the A
// operand of P V from there), and O_A, O_B.  The row maximum is only moved when it grows by more than 2^8 (kAttnLazy):
// until then weights are at most 2^8 (2^15 as fp16) and O needs no rescaling; when it does, the row's own softmax warp
// rescales O in TMEM after the last P V issued so far.
//
// What bounds it (B200, 4736 x 8192 rows, 32 / 8 heads, bf16, no mask).  D = 128: 0.52 ms, 1220 TFLOP/s; the tensor unit is
// busy 74 % of the time (58 % of it with products: the N = 64 score products read 1.5 times the shared memory that
// their arithmetic takes time for); without the exponentials it takes 0.50 ms, with an eighth of the products
// 0.43 ms.  D = 64: 0.43 ms, 735 TFLOP/s, bound by the softmax warps: 16 exponentials a cycle and SM alone take 0.26 ms, 61 % of it.
// Single tokens (split mode): 6.1 TB/s of keys and values, 0.94 of the measured copy rate, and 5.5 when the power cap (1000 W)
// holds in a long run.  One token over 8192 keys, 15.5 us: small plan 2, first keys 2, keys 4 (at the rate of memory), epilogue and
// end 2, the join 3 behind a gap of 1.
// Measured and left out (D = 128 / 64, ms): 128-key steps with single score buffers 0.76 / 0.64; UMMAs issued under
// a lane comparison 1.16 / 0.99 (see elect_one); four softmax warps a scheduler with 96 registers 0.64 / 0.55; the lanes'
// exponentials in turns 0.70 / 0.61; setmaxnreg (ptxas spills); every register spilled in the softmax loop costs, as
// shared memory takes all of L1 (76 bytes: 0.55 / 0.50 against 0.53 / 0.46 then).
//
// Masked places.  Scores behind a row's last key are replaced, not added to, so keys may hold anything there.  A value
// row that some row of the item does not see could still reach it as 0 * inf: the guard warp zeroes value rows
// behind the request's end in shared memory and, on the tiles where rows differ in what they see, zeroes non-finite
// values and reports them, and the epilogue adds them back to the rows that do see them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/itk_b200.h"
#include "itk_ptx.cuh"

namespace itk {

constexpr int kAttnTile = 128;                 // rows of a row tile, keys of a key tile
constexpr int kAttnThreads = 384;
constexpr int kAttnSoftmaxWarps = 4;           // per lane
constexpr int kAttnMmaWarp = 8, kAttnLoadWarp = 10, kAttnGuardWarp = 11;   // kAttnMmaWarp + x issues for lane x
constexpr int kAttnTmemColumns = 512;
constexpr int kAttnHalf = 64;                  // keys of a step: half a tile
constexpr int kAttnColumnS = 0, kAttnColumnO = 256;   // lane B: + 128; step i of a lane uses S columns 64 * (i % 2)
constexpr int kAttnMaxStages = 10;
constexpr int kAttnQueue = 4;                  // units of work the producer may be ahead of the last reader
constexpr int kAttnReaders = 2 * kAttnSoftmaxWarps + 3;    // warps that read them: softmax, issuers, guard
constexpr int kAttnPoison = 16;                // items the guard may be ahead of an epilogue, with room to spare
constexpr int kAttnPolynomial = 8;             // one pair of weights in so many takes exp2_polynomial (4: no gain, none: 4 % slower)
constexpr float kAttnLazy = 8.0f;              // log2 of how far weights may exceed 1 before the maximum moves
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kLog2e = 1.44269504088896340736f;

constexpr int kAttnSharedTail = 2048;

template <int DIM>
struct AttnShape {
    static constexpr int kChunks = DIM / 64;                    // 128-byte wide column chunks
    static constexpr int kTileBytes = kAttnTile * DIM * 2;
    static constexpr int kStages = DIM == 128 ? 5 : 10;         // 160 KB of key and value tiles in flight
    static constexpr int kSmemTiles = (2 + kStages) * kTileBytes;
    static constexpr int kSmemBytes = kSmemTiles + kAttnSharedTail;
};

// One unit of work for every key head.
struct AttnItem {
    int q_first, tokens;      // packed row tokens [q_first, q_first + tokens)
    int tile_begin, tiles;    // 128-key tiles of the segment
    int keys;                 // keys of the segment that any row of the item may see
    int visible, slope;       // token i sees min(keys, visible + slope * i) of them
    int request;              // whose block table row to use; -1: the prefix
    int k_first;              // first row of packed own keys
    int partial, slot, slots; // row of the partial results of the whole entry (-1: write the output), first slot, slots
};

// Up to kAttnCombineRows rows (of every key head) that have partial results to join.
constexpr int kAttnCombineRows = 16;
struct AttnCombine {
    int q_first, tokens;      // of the entry they belong to
    int partial, slots;       // own partial results of the entry
    int row_first, pad[3];
};

struct AttnCounters {
    int items, combines;
    int rows_end, rows_begin; // behind the rows of the last request, at those of the first
    int next;                 // the first unit of work (item, key head) that no CTA has taken yet
};

struct AttnWorkspace {
    AttnCounters* counters;
    int* entry_first;         // [requests + 1] own entries before a request
    int2* prefix_slots;       // per prefix entry: first partial row, slots
    AttnItem* items;
    AttnCombine* combines;
    float* partial_lse;       // log2 of the sum of exponentials of a partial row
    float* partial_out;       // [partial_rows, DIM], normalised
    int max_items, max_entries, max_combines, max_partial_rows;     // max_entries: own ones
};

struct AttnParams {
    CUtensorMap map_q, map_q_one, map_k, map_v, map_k_prefix, map_v_prefix;     // map_q_one: for items of a single token
    itk_attention_args a;
    AttnWorkspace w;
    int* status;
    int group, tile_tokens, sm_count, withhold_loads;
    int q_bytes, q_bytes_one;                      // of a box of map_q, of map_q_one
    int small_plan;                                // no plan kernel ran: see attn_small_plan
    int out_sectors;                               // rows of the output start on 32-byte boundaries
    float inverse_sms;                             // 1 / sm_count
    float scale_log2, lazy;                        // lazy: kAttnLazy in units of the scores
    uint32_t wait_polls;
};

// ------------------------------------------------------------------ PTX

// Programmatic dependent launch: the next kernel of the stream may start its prologue; what it reads of this one it
// reads behind grid_wait, which returns when this one has completed.
__device__ __forceinline__ void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Waits for the phase with the given parity, `polls` probes at most; each may be parked until the phase completes or the
// hardware's own limit runs out, 4.1 us (with hints of 1 and 20 us alike).  (The bound is a count, not a time: a deadline costs
// registers that the softmax loop does not have.)
__device__ __forceinline__ bool attn_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t polls) {
    for (uint32_t n = 0; n < polls; ++n) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag != 0) return false;
    }
    *abort_flag = 1;
    return false;
}

// True in one thread of the warp, always the same one.  The tcgen05 instructions take their operands from uniform
// registers: under this predicate, with operands that come out of a broadcast, they are moved there once; under a
// comparison with the lane id every issue paid about 100 cycles (4 UMMAs and two commits: 590 cycles).
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    return elected != 0;
}

__device__ __forceinline__ int uniform(int value) { return __shfl_sync(0xffffffffu, value, 0); }

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// 16-bit floating-point operands, fp32 accumulator, M = 128.
__host__ __device__ constexpr uint32_t umma_idesc_16bit(bool bf16, int n, bool b_mn_major) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
           ((static_cast<uint32_t>(n) >> 3) << 17) | ((128u >> 4) << 24);
}

// MN-major operand (rows of the tile are the K dimension), 128-byte swizzle: 64-column chunks are `chunk_bytes` apart,
// eight-row groups 1024 bytes.
__device__ __forceinline__ uint64_t umma_desc_sw128_mnmajor(uint32_t smem_address, uint32_t chunk_bytes) {
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((smem_address & 0x3FFFFu) >> 4);
    desc |= static_cast<uint64_t>(chunk_bytes >> 4) << 16;
    desc |= static_cast<uint64_t>(1024 >> 4) << 32;
    desc |= static_cast<uint64_t>(1) << 46;
    desc |= static_cast<uint64_t>(2) << 61;
    return desc;
}

__device__ __forceinline__ void umma_16bit_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void umma_16bit_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_load_16(uint32_t tmem_address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(tmem_address)
        : "memory");
}

__device__ __forceinline__ void tmem_store_16(uint32_t tmem_address, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(tmem_address), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A read of shared memory that the compiler does not replace by the registers the values were written from.
__device__ __forceinline__ int4 load_shared_again(const int4* address) {
    int4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem_u32(address)) : "memory");
    return v;
}

__device__ __forceinline__ float2 neg2(float2 a) { return make_float2(-a.x, -a.y); }

// Maximum of three; a NaN among them is passed over.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 32 bytes, a whole sector: rows lie far apart, so half-sector stores would take twice the time.
__device__ __forceinline__ void store_sector(void* address, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(address), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t ra, rb, rd;
    asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
    return d;
}

__device__ __forceinline__ void mask_scores(uint32_t (&s)[32], int limit) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
        if (k >= limit) s[k] = 0xff800000u;
}

// A NaN is no maximum; its weight is NaN all the same.
__device__ __forceinline__ float top_of(const uint32_t (&s)[32]) {
    float most[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        most[c] = fmaxf(__uint_as_float(s[16 * c]), __uint_as_float(s[16 * c + 1]));
#pragma unroll
        for (int k = 2; k < 16; k += 2) most[c] = max3(most[c], __uint_as_float(s[16 * c + k]), __uint_as_float(s[16 * c + k + 1]));
    }
    return max3(most[0], most[1], -INFINITY);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^z on the FMA pipe, for some of the weights: the special-function unit gives 16 exponentials a cycle to an SM, which
// is what the softmax is short of.  z = n + f with n the nearest whole number (adding 1.5 * 2^23 leaves it in the low bits),
// 2^f by a polynomial of degree 5, fitted for the least relative error on [-1/2, 1/2] by iteratively reweighted least
// squares (7.5e-8 in exact arithmetic, 2.2e-7 as evaluated in fp32), 2^n by its exponent bits.  Below the normal range the
// result is 0, as exp2_fast's is; NaN stays NaN.  z <= 127 is all that is asked for (weights are at most
// 2^(kAttnLazy + kHeadroom)).
__device__ __forceinline__ float2 exp2_polynomial(float2 z) {
    auto both = [](float x) { return make_float2(x, x); };
    const float2 shifted = add2(z, both(12582912.0f));
    const float2 f = add2(z, neg2(add2(shifted, both(-12582912.0f))));
    float2 q = fma2(both(0.0013276471520115847f), f, both(0.009675541330697653f));
    q = fma2(q, f, both(0.05550713274959883f));
    q = fma2(q, f, both(0.24022119723933577f));
    q = fma2(q, f, both(0.6931469670638649f));
    q = fma2(q, f, both(1.0000000716546569f));
    const float low = q.x * __uint_as_float((__float_as_uint(shifted.x) << 23) + 0x3f800000u);
    const float high = q.y * __uint_as_float((__float_as_uint(shifted.y) << 23) + 0x3f800000u);
    return make_float2(z.x < -126.0f ? 0.0f : low, z.y < -126.0f ? 0.0f : high);
}

template <typename T>
struct Element;

template <>
struct Element<__nv_bfloat16> {
    static constexpr bool kBf16 = true;
    static constexpr float kHeadroom = 0.0f;         // log2 of how much larger than 1 the weight of the maximum is held
    static constexpr uint32_t kExponent = 0x7f80u;
    static __device__ __forceinline__ uint32_t pack(float low, float high) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
        return r;
    }
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};

template <>
struct Element<__half> {
    static constexpr bool kBf16 = false;
    static constexpr float kHeadroom = 7.0f;
    static constexpr uint32_t kExponent = 0x7c00u;
    static __device__ __forceinline__ uint32_t pack(float low, float high) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
        return r;
    }
    static __device__ __forceinline__ float value(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
};

static_assert(kAttnLazy + Element<__half>::kHeadroom <= 15.0f, "fp16 weights stay finite");

// ------------------------------------------------------------------ plan

// Lengths of one request, clamped to the buffers they index, its rows also to the end of the last request's: the entries of
// a prefix cover the rows up to there, and the join looks the prefix's results up by the row.
struct AttnRequest {
    int q_first, q_count, k_first, k_count;
};

// Where the last request's rows end.
__device__ __forceinline__ int attn_rows_end(const itk_attention_args& p) { return min(max(p.cu_q[p.requests], 0), p.tokens); }

__device__ __forceinline__ AttnRequest attn_request(const itk_attention_args& p, int b, bool& bad) {
    AttnRequest r;
    const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], rows_end = attn_rows_end(p);
    r.q_first = min(max(q0, 0), rows_end);
    r.q_count = max(min(max(q1, 0), rows_end) - r.q_first, 0);
    bad |= q0 != r.q_first || q1 != r.q_first + r.q_count;
    if (p.cu_k != nullptr) {
        const int k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
        r.k_first = min(max(k0, 0), p.own.page_size);
        r.k_count = max(min(max(k1, 0), p.own.page_size) - r.k_first, 0);
        bad |= k0 != r.k_first || k1 != r.k_first + r.k_count;
    } else {
        const int n = p.lens_k[b];
        const long long room = static_cast<long long>(p.own.table_pages) * p.own.page_size;
        r.k_first = 0;
        r.k_count = static_cast<int>(min(static_cast<long long>(min(max(n, 0), ITK_MAX_ATTENTION_KEYS)), room));
        bad |= n != r.k_count;
    }
    return r;
}

constexpr int kAttnBins = 256;
constexpr int kAttnTries = 8;
constexpr int kAttnMinChunk = 2;    // key tiles of a chunk at least: below that a chunk's fixed cost outweighs its keys
// When the items do not fit one wave, the CTAs take them from the list as they get free, the longest first.  Entries of up
// to half a CTA's fair share are not cut then (cutting 592 equal ones, four waves, into halves cost 532 -> 778 us); longer
// ones are cut into kAttnWaves-ths of the share, which is what the last one taken may run beyond the others, but not
// below the length at which writing and joining their partial results shows.
constexpr int kAttnWaves = 6, kAttnWaveChunk = 24;
static_assert(kAttnMinChunk >= 2, "a split item of one tile is its entry's only item: it has one slot and no lane B");
// Relative cost of a key tile: a pair tile is bound by tensor and exponential work for 256 rows, a split tile by
// the time its keys take to arrive.
constexpr int kAttnPairCost = 4, kAttnSplitCost = 3;

constexpr int kAttnCached = 1024;   // requests whose lengths the plan keeps in shared memory

struct AttnEntry {
    AttnItem item;
    int tiles, unit;          // key tiles, cost of one
    bool pair, prefix;
};

// Lengths and first entries of the requests: in shared memory for batches that fit it, else from global memory.
struct AttnRequests {
    const AttnRequest* cached;
    const int* first;         // [requests + 1] own entries before a request
    bool is_cached;
};

// Entry e of the list "prefix entries, then the entries of request 0, 1, ...": up to 2 TT consecutive tokens of one
// request (of any requests for the prefix, which they all see).
__device__ __forceinline__ AttnEntry attn_entry(const AttnParams& p, const AttnRequests& requests, int e, int prefix_entries, int rows_end) {
    const int span = 2 * p.tile_tokens;
    AttnEntry r;
    r.prefix = e < prefix_entries;
    if (r.prefix) {
        r.item.q_first = e * span;
        r.item.tokens = min(span, rows_end - e * span);
        r.item.keys = p.a.prefix_keys;
        r.item.visible = p.a.prefix_keys;
        r.item.slope = 0;
        r.item.request = -1;
        r.item.k_first = 0;
    } else {
        const int own = e - prefix_entries;
        int low = 0, high = p.a.requests;       // first[low] <= own < first[high]
        while (high - low > 1) {
            const int middle = (low + high) >> 1;
            if (requests.first[middle] <= own) {
                low = middle;
            } else {
                high = middle;
            }
        }
        bool bad = false;
        const AttnRequest q = requests.is_cached ? requests.cached[low] : attn_request(p.a, low, bad);
        const int first = (own - requests.first[low]) * span;
        r.item.q_first = q.q_first + first;
        r.item.tokens = min(span, q.q_count - first);
        r.item.request = low;
        r.item.k_first = q.k_first;
        if (p.a.causal) {
            r.item.visible = q.k_count - q.q_count + first + 1;
            r.item.slope = 1;
            r.item.keys = max(0, min(q.k_count, r.item.visible + r.item.tokens - 1));
        } else {
            r.item.visible = r.item.keys = q.k_count;
            r.item.slope = 0;
        }
    }
    r.tiles = (r.item.keys + kAttnTile - 1) / kAttnTile;
    r.pair = r.item.tokens > p.tile_tokens;
    r.unit = r.pair ? kAttnPairCost : kAttnSplitCost;
    return r;
}

// Key chunks of an entry when a chunk may cost `cost` and entries up to `whole` are not cut.
__device__ __forceinline__ int attn_chunks(const AttnEntry& e, int cost, int whole) {
    if (whole > 0 && static_cast<long long>(e.tiles) * e.unit <= whole) return e.tiles > 0 ? 1 : 0;
    const unsigned per = max(kAttnMinChunk, e.pair ? (cost + kAttnPairCost - 1) / kAttnPairCost : (cost + kAttnSplitCost - 1) / kAttnSplitCost);
    return static_cast<int>((static_cast<unsigned>(e.tiles) + per - 1) / per);
}

// Slots of an entry cut into `chunks` (0: no key at all), and whether its results are partial ones.
__device__ __forceinline__ bool attn_slots(const AttnParams& p, AttnEntry& entry, int chunks) {
    const int longest_chunk = chunks > 0 ? (entry.tiles + chunks - 1) / chunks : 0;
    entry.item.slots = chunks * (!entry.pair && longest_chunk > 1 ? 2 : 1);
    entry.item.partial = -1;
    return p.a.prefix_keys > 0 || entry.item.slots > 1;
}

// Chunk c of `count` of an entry whose slots are set; the first tiles % count chunks are one tile longer.
__device__ __forceinline__ AttnItem attn_chunk(const AttnEntry& entry, int c, int count) {
    AttnItem item = entry.item;
    const int even = entry.tiles / count, odd = entry.tiles - even * count;
    item.tile_begin = c * even + min(c, odd);
    item.tiles = even + (c < odd ? 1 : 0);
    item.slot = c * (entry.item.slots / count);
    return item;
}

// A fair share of the work of all SMs, in fp32: it only has to be near.  (A chunk costs at most 2^29, more than any
// entry, 2^24 tiles of cost 4, does.)
__device__ __forceinline__ int attn_share(const AttnParams& p, unsigned long long cost) {
    return static_cast<int>(fminf(ceilf(static_cast<float>(cost) * p.a.kv_heads * p.inverse_sms) + 1.0f, 536870912.0f));
}

// Requests whose rows overlap (lengths that decrease in between) may have more entries in all than 31 bits count; the sums
// stay at this, which is more than any buffer holds.  A warp's own sum, of 32 requests with up to 2^24 entries, fits.
constexpr int kAttnMostEntries = 1 << 30;

// Sum of the values of the lanes before this one; `total`: of all lanes.
__device__ __forceinline__ int warp_prefix(int value, int lane, int& total) {
    int upto = value;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, step);
        if (lane >= step) upto += other;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    return upto - value;
}

// Most of a small call's time before its first key is read goes by in here: one pass over the lengths, entries kept in
// registers, six block barriers when the items fit one wave (their order does not matter then), no 64-bit division
// (those took half of 7.8 us for one request).
template <int THREADS>
__global__ void __launch_bounds__(THREADS) itk_attention_plan_kernel(const __grid_constant__ AttnParams p) {
    __shared__ int warp_sums[THREADS / 32];
    __shared__ int carry, rows_end;
    __shared__ unsigned long long total_cost;
    __shared__ int counts[kAttnTries], longest, item_count, combine_count, partial_rows;
    __shared__ int bins[kAttnBins];
    __shared__ AttnRequest cache[kAttnCached];
    __shared__ int cached_first[kAttnCached + 1];
    const bool is_cached = p.a.requests <= kAttnCached;
    int* entry_first = is_cached ? cached_first : p.w.entry_first;
    const AttnRequests requests{cache, entry_first, is_cached};
    const int tx = threadIdx.x, lane = tx & 31, warp = tx >> 5;
    const int span = 2 * p.tile_tokens, kv_heads = p.a.kv_heads;
    grid_launch_dependents();
    if (tx == 0) {
        carry = 0;
        total_cost = 0;
        longest = item_count = combine_count = partial_rows = 0;
    }
    if (tx == 32) rows_end = attn_rows_end(p.a);
    if (tx < kAttnTries) counts[tx] = 0;
    for (int i = tx; i < kAttnBins; i += THREADS) bins[i] = 0;
    // (the barriers of the first pass below stand between these and their first readers: there is at least one request)

    // own entries before every request
    bool bad = false;
    for (int base = 0; base < p.a.requests; base += THREADS) {
        const int b = base + tx;
        int mine = 0;
        if (b < p.a.requests) {
            const AttnRequest request = attn_request(p.a, b, bad);
            if (is_cached) cache[b] = request;
            mine = (request.q_count + span - 1) / span;
        }
        int total;
        const int in_warp = warp_prefix(mine, lane, total);
        if (lane == 31) warp_sums[warp] = total;
        __syncthreads();
        int before = carry;
        for (int w = 0; w < warp; ++w) before = min(before + warp_sums[w], kAttnMostEntries);
        if (b < p.a.requests) entry_first[b] = before + in_warp;
        __syncthreads();
        if (tx == THREADS - 1) carry = min(before + total, kAttnMostEntries);
    }
    if (bad) atomicOr(p.status, ITK_SERVING_BAD_LENGTHS);
    __syncthreads();
    const int prefix_entries = p.a.prefix_keys > 0 ? (rows_end + span - 1) / span : 0;
    const int entries = prefix_entries + min(carry, p.w.max_entries);

    // every thread keeps its first entry; larger batches work the others out again in every pass
    AttnEntry kept{};
    if (tx < entries) kept = attn_entry(p, requests, tx, prefix_entries, rows_end);
    auto entry_at = [&](int e) { return e == tx ? kept : attn_entry(p, requests, e, prefix_entries, rows_end); };

    // the chunk length that spreads the work over the SMs in one wave, if there is one
    unsigned long long cost = 0;
    for (int e = tx; e < entries; e += THREADS) {
        const AttnEntry entry = entry_at(e);
        cost += static_cast<unsigned long long>(entry.tiles) * entry.unit;
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, step);
    if (lane == 0 && cost != 0) atomicAdd(&total_cost, cost);
    __syncthreads();
    const int share = attn_share(p, total_cost);
    int mine[kAttnTries] = {};
    for (int e = tx; e < entries; e += THREADS) {
        const AttnEntry entry = entry_at(e);
#pragma unroll
        for (int k = 0; k < kAttnTries; ++k) mine[k] += max(1, attn_chunks(entry, share + share / kAttnTries * k, 0));
    }
#pragma unroll
    for (int k = 0; k < kAttnTries; ++k) {
        const int sum = __reduce_add_sync(0xffffffffu, mine[k]);
        if (lane == 0 && sum != 0) atomicAdd(&counts[k], sum);
    }
    __syncthreads();
    int chunk = min(share, max(share / kAttnWaves, kAttnWaveChunk * kAttnPairCost)), whole = share / 2;
    bool one_wave = false;
    for (int k = kAttnTries - 1; k >= 0; --k)
        if (static_cast<long long>(counts[k]) * kv_heads <= p.sm_count) {
            chunk = share + share / kAttnTries * k;
            whole = 0;
            one_wave = true;
        }

    // more than a wave: the costliest items first, by a counting sort over 256 cost classes
    int top = 1;
    auto bin_of = [&](const AttnEntry& entry, int chunks) {
        const int item_cost = (entry.tiles + chunks - 1) / chunks * entry.unit;
        return kAttnBins - 1 - static_cast<int>(static_cast<long long>(item_cost) * (kAttnBins - 1) / top);
    };
    if (!one_wave) {
        int most = 0;
        for (int e = tx; e < entries; e += THREADS) {
            const AttnEntry entry = entry_at(e);
            const int chunks = max(1, attn_chunks(entry, chunk, whole));
            most = max(most, (entry.tiles + chunks - 1) / chunks * entry.unit);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) atomicMax(&longest, most);
        __syncthreads();
        top = max(longest, 1);
        for (int e = tx; e < entries; e += THREADS) {
            const AttnEntry entry = entry_at(e);
            const int chunks = max(1, attn_chunks(entry, chunk, whole));
            atomicAdd(&bins[bin_of(entry, chunks)], chunks);
        }
        __syncthreads();
        if (warp == 0) {
            int sum = 0, held[kAttnBins / 32];
#pragma unroll
            for (int i = 0; i < kAttnBins / 32; ++i) {
                held[i] = bins[lane * (kAttnBins / 32) + i];
                sum += held[i];
            }
            int total;
            int before = warp_prefix(sum, lane, total);
#pragma unroll
            for (int i = 0; i < kAttnBins / 32; ++i) {
                bins[lane * (kAttnBins / 32) + i] = before;
                before += held[i];
            }
            if (lane == 31) item_count = before;
        }
        __syncthreads();
    }
    for (int e = tx; e < entries; e += THREADS) {
        AttnEntry entry = entry_at(e);
        const int chunks = attn_chunks(entry, chunk, whole);               // 0: no key at all
        const int rows = entry.item.tokens * p.group;
        const bool joined = attn_slots(p, entry, chunks);
        if (joined && entry.item.slots > 0) {
            const int needed = entry.item.slots * rows * kv_heads;
            const int first = atomicAdd(&partial_rows, needed);
            // (the host sizes the buffer so that this always fits; nothing is written behind it if it did not)
            entry.item.partial = first + needed <= p.w.max_partial_rows ? first : -2;
            if (entry.item.partial == -2) atomicOr(p.status, ITK_SERVING_BAD_LENGTHS);
        }
        const int usable = entry.item.partial < 0 ? 0 : entry.item.slots;
        if (entry.prefix) {
            p.w.prefix_slots[e] = make_int2(entry.item.partial, usable);
        } else if (joined) {
            const int records = (rows + kAttnCombineRows - 1) / kAttnCombineRows;
            const int at = atomicAdd(&combine_count, records);
            for (int r = 0; r < records; ++r)
                if (at + r < p.w.max_combines)
                    p.w.combines[at + r] = AttnCombine{entry.item.q_first, entry.item.tokens, entry.item.partial, usable, r * kAttnCombineRows, {}};
        }
        if (chunks == 0 && joined) entry.item.tokens = 0;           // the prefix alone: a place in the list, but nothing to do
        const int count = max(1, chunks);
        const int place = atomicAdd(one_wave ? &item_count : &bins[bin_of(entry, count)], count);
        for (int c = 0; c < count; ++c)
            if (place + c < p.w.max_items) p.w.items[place + c] = attn_chunk(entry, c, count);
    }
    __syncthreads();
    if (tx == 0) *p.w.counters = AttnCounters{min(item_count, p.w.max_items), min(combine_count, p.w.max_combines), rows_end,
                                               min(max(p.a.cu_q[0], 0), p.a.tokens), p.sm_count};
}

// The plan of a call with at most 32 requests and 32 entries that fit one wave of CTAs uncut: every CTA's producer warp
// works out the whole of it for itself, a request and an entry per lane, and takes the one unit that has the CTA's number.
// That saves the plan's launch and the wait for it.  CTA 0 also writes down what the join needs.  `cache` and `first` are
// scratch for the requests.  Returns whether there is a unit.
constexpr int kAttnSmallEntries = 32;

__device__ __forceinline__ bool attn_small_plan(const AttnParams& p, AttnRequest* cache, int* first, int4* unit, int lane) {
    const int span = 2 * p.tile_tokens, kv_heads = p.a.kv_heads;
    const int rows_end = attn_rows_end(p.a);
    bool bad = false;
    int mine = 0, own;
    if (lane < p.a.requests) {
        const AttnRequest request = attn_request(p.a, lane, bad);
        cache[lane] = request;
        mine = (request.q_count + span - 1) / span;
    }
    first[lane] = warp_prefix(mine, lane, own);
    if (bad && blockIdx.x == 0) atomicOr(p.status, ITK_SERVING_BAD_LENGTHS);
    __syncwarp();
    const int prefix_entries = p.a.prefix_keys > 0 ? (rows_end + span - 1) / span : 0;
    const bool there = lane < prefix_entries + own;             // (the host has counted them: 32 at most)
    AttnEntry entry{};
    entry.unit = 1;
    if (there) entry = attn_entry(p, AttnRequests{cache, first, true}, lane, prefix_entries, rows_end);
    const int cost = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(entry.tiles) * entry.unit);
    const int share = attn_share(p, static_cast<unsigned>(cost));
    // (a loop, not unrolled: code that runs once waits for its instructions, 1 us for eight copies of this)
    int chunk = 1 << 30;            // nothing is cut: that fits a wave
#pragma unroll 1
    for (int t = 0; t < kAttnTries; ++t) {
        const int length = share + share / kAttnTries * t;
        const int wanted = there ? max(1, attn_chunks(entry, length, 0)) : 0;
        if (static_cast<int>(__reduce_add_sync(0xffffffffu, wanted)) * kv_heads <= p.sm_count) {
            chunk = length;
            break;
        }
    }

    const int chunks = there ? attn_chunks(entry, chunk, 0) : 0, count = there ? max(1, chunks) : 0;
    const bool joined = there && attn_slots(p, entry, chunks);
    const int rows = there ? entry.item.tokens * p.group : 0;
    int items, partial, records;
    const int place = warp_prefix(count, lane, items);
    const int first_row = warp_prefix(joined ? entry.item.slots * rows * kv_heads : 0, lane, partial);
    if (joined && entry.item.slots > 0) entry.item.partial = partial <= p.w.max_partial_rows ? first_row : -2;
    const int index = static_cast<int>(blockIdx.x) / kv_heads, head = static_cast<int>(blockIdx.x) - index * kv_heads;
    const bool found = index >= place && index < place + count && !(chunks == 0 && joined);
    if (found) {
        const AttnItem item = attn_chunk(entry, index - place, count);
        unit[0] = make_int4(item.q_first, item.tokens, item.tile_begin, item.tiles);
        unit[1] = make_int4(item.keys, item.visible, item.slope, item.request);
        unit[2] = make_int4(item.k_first, item.partial, item.slot, item.slots);
        unit[3] = make_int4(head, 1, 0, 0);
    }
    if (blockIdx.x == 0) {
        const int usable = entry.item.partial < 0 ? 0 : entry.item.slots;
        if (there && entry.prefix) p.w.prefix_slots[lane] = make_int2(entry.item.partial, usable);
        const int wanted = joined && !entry.prefix ? (rows + kAttnCombineRows - 1) / kAttnCombineRows : 0;
        const int at = warp_prefix(wanted, lane, records);
        for (int r = 0; r < wanted; ++r)
            if (at + r < p.w.max_combines)
                p.w.combines[at + r] = AttnCombine{entry.item.q_first, entry.item.tokens, entry.item.partial, usable, r * kAttnCombineRows, {}};
        if (lane == 0) *p.w.counters = AttnCounters{items, min(records, p.w.max_combines), rows_end, min(max(p.a.cu_q[0], 0), p.a.tokens), 0};
    }
    __syncwarp();
    return __any_sync(0xffffffffu, found) != 0;
}

// ------------------------------------------------------------------ attention

struct AttnShared {
    uint64_t q_full[2], q_empty[2];
    uint64_t kv_full[kAttnMaxStages], kv_empty[kAttnMaxStages], guard_full[kAttnMaxStages];
    uint64_t s_full[2][2], p_full[2][2];      // lane, step parity
    uint64_t pv_done[2], o_full[2], o_empty[2];
    uint64_t item_full[kAttnQueue], item_empty[kAttnQueue];
    int poison[kAttnPoison];
    AttnRequest small_requests[kAttnSmallEntries];
    int small_first[kAttnSmallEntries];
    int4 items[kAttnQueue][4];                // the CTA's next units of work: the item, then (key head, 1) or (-, 0) at the end
    uint32_t tmem_base;
    int abort;
};
static_assert(sizeof(AttnShared) <= kAttnSharedTail, "barriers fit the tail of the shared-memory block");

// What an item means for one lane.
struct AttnLanes {
    bool pair;
    int first_visible;        // keys that every row sees
    int tiles[2];             // key tiles of lane A, B
};

__device__ __forceinline__ AttnLanes attn_lanes(const AttnItem& item, int tile_tokens) {
    AttnLanes r;
    r.pair = item.tokens > tile_tokens;
    r.first_visible = max(0, min(item.visible, item.keys));
    r.tiles[0] = r.pair ? item.tiles : (item.tiles + 1) / 2;
    r.tiles[1] = r.pair ? item.tiles : item.tiles / 2;
    return r;
}

static_assert(sizeof(AttnItem) == 48, "items are read as three 16-byte vectors");

__device__ __forceinline__ AttnItem attn_item(const int4& a, const int4& b, const int4& c) {
    return AttnItem{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
}

// Where key tile t of a segment lies.
__device__ __forceinline__ int attn_page(const AttnParams& p, const AttnItem& item, int t) {
    const itk_kv_segment& seg = item.request < 0 ? p.a.prefix : p.a.own;
    const int32_t* table = item.request < 0 ? p.a.prefix_table : p.a.table;
    if (table == nullptr) return 0;
    if (item.request >= 0) table += item.request * seg.table_stride;
    const int page = table[t / (seg.page_size / kAttnTile)];
    if (page < 0 || page >= seg.pages) {
        atomicOr(p.status, ITK_SERVING_BAD_PAGE);
        return page < 0 ? 0 : seg.pages - 1;
    }
    return page;
}

template <typename T>
__device__ __forceinline__ const T* attn_value_row(const AttnParams& p, const AttnItem& item, int head, int key) {
    const itk_kv_segment& seg = item.request < 0 ? p.a.prefix : p.a.own;
    long long row = item.k_first + key;
    long long page = 0;
    if ((item.request < 0 ? p.a.prefix_table : p.a.table) != nullptr) {
        page = attn_page(p, item, key / kAttnTile);
        row = key % seg.page_size;
    }
    return static_cast<const T*>(item.request < 0 ? p.a.v_prefix : p.a.v) + page * seg.v_page_stride + row * seg.v_row_stride + head * seg.v_head_stride;
}

// Ring position of the value tile t of an item.  Pair: K0 V0 K1 V1 ...  Split (the lanes take turns and each is one key
// tile ahead of its values): K0 K1 V0 K2 V1 K3 ... V(n-1).
__device__ __forceinline__ int ring_value(bool pair, int t, int tiles) {
    return pair ? 2 * t + 1 : min(2 * t + 2, 2 * tiles - 1);
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kAttnThreads, 1) itk_attention_kernel(const __grid_constant__ AttnParams p) {
    using Shape = AttnShape<DIM>;
    constexpr int kStages = Shape::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* smem_q = smem;
    uint8_t* smem_kv = smem + 2 * Shape::kTileBytes;
    AttnShared& sh = *reinterpret_cast<AttnShared*>(smem + Shape::kSmemTiles);
    const int warp = uniform(static_cast<int>(threadIdx.x) >> 5);
    const int lane = static_cast<int>(threadIdx.x) & 31;

    if ((smem_u32(smem) & 1023u) != 0u) {   // the same in every thread
        if (threadIdx.x == 0) atomicOr(p.status, ITK_SERVING_BAD_SHARED_BASE);
        return;
    }
    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 2);       // both issuers
            for (int h = 0; h < 2; ++h) {
                mbar_init(&sh.s_full[i][h], 1);
                mbar_init(&sh.p_full[i][h], kAttnSoftmaxWarps);
            }
            mbar_init(&sh.pv_done[i], 1);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.o_empty[i], kAttnSoftmaxWarps);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sh.kv_full[i], 1);
            mbar_init(&sh.kv_empty[i], 2);
            mbar_init(&sh.guard_full[i], 1);
        }
        for (int i = 0; i < kAttnQueue; ++i) {
            mbar_init(&sh.item_full[i], 1);
            mbar_init(&sh.item_empty[i], kAttnReaders);
        }
        for (int i = 0; i < kAttnPoison; ++i) sh.poison[i] = 0;
        sh.abort = 0;
        fence_mbar_init();
        prefetch_tensormap(&p.map_q);
        prefetch_tensormap(&p.map_k);
        prefetch_tensormap(&p.map_v);
    }
    // Rows behind a single token's stay zero until longer items have left theirs there, so that multiplying them costs little
    // power; while the plan runs this takes no time of its own.  (Without a plan kernel it would cost a single token 1 us.)
    if (!p.small_plan) {
        for (int i = p.group * (DIM / 8) + static_cast<int>(threadIdx.x); i < kAttnTile * (DIM / 8); i += kAttnThreads) {
            const int row = i / (DIM / 8), vector = i % (DIM / 8);
            for (int tile = 0; tile < 2; ++tile)
                *reinterpret_cast<uint4*>(smem_q + tile * Shape::kTileBytes + (vector / 8) * (kAttnTile * 128) + row * 128 +
                                          (vector % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    bool planned = false;                // the producer: the unit of a small call is in the queue
    if (warp == kAttnLoadWarp && p.small_plan != 0) planned = attn_small_plan(p, sh.small_requests, sh.small_first, sh.items[0], lane);
    if (warp == kAttnMmaWarp) {          // the first issuer owns TMEM
        tmem_alloc(&sh.tmem_base, kAttnTmemColumns);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    tcgen05_fence_after_sync();
    grid_wait();                         // the plan's list from here on
    const uint32_t tmem = static_cast<uint32_t>(uniform(static_cast<int>(sh.tmem_base)));
    volatile int* abort_flag = &sh.abort;
    // a wait of the whole warp: its lanes leave together
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, attn_wait(bar, parity, abort_flag, p.wait_polls)) != 0;
    };
    bool ok = true;
    AttnItem item;
    int head;
    // The units of work, for all warps but the producer that hands them out: take() reads the next one, done() gives its
    // place in the queue back (a softmax warp reads it once more before its epilogue).
    int units = 0;
    auto read_unit = [&](int unit) {
        const int4* source = sh.items[unit % kAttnQueue];
        item = attn_item(load_shared_again(source), load_shared_again(source + 1), load_shared_again(source + 2));
        const int4 tail = load_shared_again(source + 3);
        head = tail.x;
        return tail.y != 0;
    };
    auto done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.item_empty[(units - 1) % kAttnQueue]);
    };
    auto take = [&]() {
        ok = wait(&sh.item_full[units % kAttnQueue], (units / kAttnQueue) & 1);
        return ok && read_unit(units++);
    };

    if (warp == kAttnLoadWarp) {
        // ============================================================ TMA producer
        int ring = 0;                 // tiles loaded so far
        int q_uses[2] = {0, 0};
        const int kv_heads = p.a.kv_heads;
        // The first unit of a CTA is the one with its number, the others are taken when their turn comes.
        int unit = static_cast<int>(blockIdx.x), next_unit = 0;
        for (; ok; unit = __shfl_sync(0xffffffffu, next_unit, 0)) {
            int4* place = sh.items[units % kAttnQueue];
            bool there;
            if (p.small_plan != 0) {
                // (at most one unit: nothing in the queue is waited for)
                there = units == 0 && planned;
                if (!there && lane == 0) place[3] = make_int4(0, 0, 0, 0);
                __syncwarp();
                if (there) {
                    item = attn_item(load_shared_again(place), load_shared_again(place + 1), load_shared_again(place + 2));
                    head = load_shared_again(place + 3).x;
                }
            } else {
                const int index = min(unit / kv_heads, p.w.max_items - 1);
                // read before it is known whether there is such an item: the loads overlap
                const int4* source = reinterpret_cast<const int4*>(p.w.items + index);
                const int4 a = source[0], b = source[1], c = source[2];
                there = unit < p.w.counters->items * kv_heads;
                item = attn_item(a, b, c);
                head = unit - index * kv_heads;
                if (there && lane == 0) next_unit = atomicAdd(&p.w.counters->next, 1);
                if (there && item.tokens == 0) continue;              // nothing to do
                ok = wait(&sh.item_empty[units % kAttnQueue], ((units / kAttnQueue) & 1) ^ 1);
                if (!ok) break;
                if (lane == 0) {
                    place[0] = a;
                    place[1] = b;
                    place[2] = c;
                    place[3] = make_int4(head, there ? 1 : 0, 0, 0);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.item_full[units % kAttnQueue]);
            ++units;
            if (!there) break;
            const AttnLanes l = attn_lanes(item, p.tile_tokens);
            if (item.tiles == 0 || p.withhold_loads != 0) continue;
            // A single token's box holds its own queries only.  The rows beside them would be other requests', multiplied for
            // nothing, and the power cap is what holds a batch of single tokens back when steps follow each other (64
            // tokens over 65 to 32768 keys, 64/8 heads: 318 us, 333 with them; in a short run 304 and 307).
            const CUtensorMap* map_q = item.tokens == 1 ? &p.map_q_one : &p.map_q;
            const int q_bytes = item.tokens == 1 ? p.q_bytes_one : p.q_bytes;
            for (int tile = 0; ok && tile < (l.pair ? 2 : 1); ++tile) {
                ok = wait(&sh.q_empty[tile], (q_uses[tile] & 1) ^ 1);
                ++q_uses[tile];
                if (ok && lane == 0) {
                    mbar_arrive_expect_tx(&sh.q_full[tile], q_bytes);
                    for (int c = 0; c < Shape::kChunks; ++c)
                        tma_load_3d(smem_q + tile * Shape::kTileBytes + c * (kAttnTile * 128), map_q, &sh.q_full[tile], c * 64,
                                    head * p.group, item.q_first + tile * p.tile_tokens);
                }
            }
            const itk_kv_segment& seg = item.request < 0 ? p.a.prefix : p.a.own;
            const CUtensorMap* map_k = item.request < 0 ? &p.map_k_prefix : &p.map_k;
            const CUtensorMap* map_v = item.request < 0 ? &p.map_v_prefix : &p.map_v;
            const bool table = (item.request < 0 ? p.a.prefix_table : p.a.table) != nullptr;
            const int steps = 2 * item.tiles;
            int k_next = 0, v_next = 0;
            int k_pages = 0, v_pages = 0;       // pages of 32 key (value) tiles, one per lane
            for (int s = 0; ok && s < steps; ++s) {
                // pair: K V K V; split: K K V K V K ... V V
                const bool key_tile = l.pair ? (s & 1) == 0 : (s < 2 ? s < item.tiles : (k_next < item.tiles && (s & 1) != 0));
                const int t = key_tile ? k_next++ : v_next++;
                int& pages = key_tile ? k_pages : v_pages;
                if (table && (t & 31) == 0) pages = t + lane < item.tiles ? attn_page(p, item, item.tile_begin + t + lane) : 0;
                const int page = table ? __shfl_sync(0xffffffffu, pages, t & 31) : 0;
                const int key = (item.tile_begin + t) * kAttnTile;
                const int row = table ? key % seg.page_size : item.k_first + key;
                const int stage = ring % kStages;
                ok = wait(&sh.kv_empty[stage], ((ring / kStages) & 1) ^ 1);
                ++ring;
                if (ok && lane == 0) {
                    // a value tile that the guard has to look at reaches the issuer through the guard
                    const bool guarded = !key_tile && key + kAttnTile > l.first_visible;
                    uint64_t* full = guarded ? &sh.guard_full[stage] : &sh.kv_full[stage];
                    mbar_arrive_expect_tx(full, Shape::kTileBytes);
                    for (int c = 0; c < Shape::kChunks; ++c)
                        tma_load_4d(smem_kv + stage * Shape::kTileBytes + c * (kAttnTile * 128), key_tile ? map_k : map_v,
                                    full, c * 64, head, row, page);
                }
            }
        }
    } else if (warp == kAttnMmaWarp || warp == kAttnMmaWarp + 1) {
        // ============================================================ UMMA issuer of lane x
        // One warp per lane: while one waits for its weights the other keeps the tensor pipe fed.  A parity wait says
        // nothing about a barrier that is more than one phase behind, so BOTH issuers see every use of q_full and
        // kv_full, in the order of the loads, and each gives one of the two arrivals that free the buffer: a commit
        // behind its last read, or a plain arrival for what only the other lane reads.
        constexpr uint32_t kIdescS = umma_idesc_16bit(Element<T>::kBf16, kAttnHalf, false);
        constexpr uint32_t kIdescO = umma_idesc_16bit(Element<T>::kBf16, DIM, true);
        const int x = warp - kAttnMmaWarp;
        const uint32_t tmem_s = tmem + kAttnColumnS + x * 128, tmem_o = tmem + kAttnColumnO + x * 128;
        const uint32_t q_base = smem_u32(smem_q), kv_base = smem_u32(smem_kv);
        int ring = 0, items = 0, q_uses[2] = {0, 0};      // tiles seen so far; items of this lane; uses of the row tiles
        uint32_t p_phase = 0;               // parity of the next weights; both buffers' turn over with a tile
        auto release = [&](uint64_t* bar) {
            if (lane == 0) mbar_arrive(bar);
        };
        while (ok && take()) {
            done();
            const AttnLanes l = attn_lanes(item, p.tile_tokens);
            const bool pair = uniform(l.pair) != 0;
            const int tiles = uniform(item.tiles), mine = uniform(l.tiles[x]);
            if (tiles == 0) continue;
            const int q_tile = pair ? x : 0;
            for (int tile = 0; ok && tile < (pair ? 2 : 1); ++tile) {
                ok = wait(&sh.q_full[tile], q_uses[tile] & 1);
                ++q_uses[tile];
                if (ok && (tile != q_tile || mine == 0)) release(&sh.q_empty[tile]);
            }
            const uint64_t q_desc = umma_desc_sw128_kmajor(q_base + q_tile * Shape::kTileBytes);
            uint32_t k_tile = 0;
            int k_stage = 0;
            // the next tile of the ring, in shared memory
            auto arrive_tile = [&](int& stage) {
                stage = ring % kStages;
                ok = ok && wait(&sh.kv_full[stage], (ring / kStages) & 1);
                ++ring;
                return ok;
            };
            // tiles that only the other lane reads (split items)
            auto pass_tile = [&]() {
                int stage;
                if (arrive_tile(stage)) release(&sh.kv_empty[stage]);
            };
            // S for half h of the lane's tile j; the key tile is released when its last half has been issued
            auto scores = [&](int j, int h) {
                if (h == 0) {
                    if (!arrive_tile(k_stage)) return;
                    k_tile = kv_base + k_stage * Shape::kTileBytes;
                }
                if (!ok) return;
                const uint64_t b = umma_desc_sw128_kmajor(k_tile + h * (kAttnHalf * 128));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DIM / 16; ++k) {
                        constexpr int kChunkStep = (kAttnTile * 128) >> 4;
                        const int offset = (k / 4) * kChunkStep + (k % 4) * 2;      // 16-byte units: 32 bytes per K step
                        umma_16bit_ss(tmem_s + h * kAttnHalf, q_desc + offset, b + offset, kIdescS, k > 0);
                    }
                    umma_commit(&sh.s_full[x][h]);
                    if (h == 1) {
                        umma_commit(&sh.kv_empty[k_stage]);
                        // the last scores of the row tile: its rows may be replaced
                        if (j + 1 == mine) umma_commit(&sh.q_empty[q_tile]);
                    }
                }
                __syncwarp();
            };
            // Loads come as K0 V0 K1 V1 ... (pair) or K0 K1 V0 K2 V1 K3 ... (split, tile t being lane t % 2's)
            if (!pair && x == 1) pass_tile();
            if (mine > 0) {
                scores(0, 0);
                scores(0, 1);
            }
            if (!pair && x == 0 && tiles > 1) pass_tile();
            for (int t = 0; ok && t < tiles; ++t) {
                if (!pair && (t & 1) != x) {
                    pass_tile();
                    if (t + 2 < tiles) pass_tile();
                    continue;
                }
                const int j = pair ? t : t >> 1;
                int v_stage;
                if (!arrive_tile(v_stage)) break;
                const uint64_t v_desc = umma_desc_sw128_mnmajor(kv_base + v_stage * Shape::kTileBytes, kAttnTile * 128);
                if (j == 0) ok = wait(&sh.o_empty[x], (items & 1) ^ 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (ok) ok = wait(&sh.p_full[x][h], p_phase);
                    if (!ok) continue;
                    tcgen05_fence_after_sync();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kAttnHalf / 16; ++k)
                            umma_16bit_ts(tmem_o, tmem_s + h * kAttnHalf + k * 8, v_desc + (h * (kAttnHalf * 128) + k * 2048) / 16,
                                          kIdescO, j > 0 || h > 0 || k > 0);
                        umma_commit(&sh.pv_done[x]);
                        if (h == 1) {
                            if (j + 1 == mine) umma_commit(&sh.o_full[x]);
                            umma_commit(&sh.kv_empty[v_stage]);
                        }
                    }
                    __syncwarp();
                    if (j + 1 < mine) scores(j + 1, h);
                }
                p_phase ^= 1u;
            }
            if (mine > 0) ++items;
        }
    } else if (warp == kAttnGuardWarp) {
        // ============================================================ guard
        int ring = 0;
        uint32_t phases = 0;          // of guard_full: a stage's flips with every tile the guard takes from it
        while (ok && p.withhold_loads == 0 && take()) {
            done();
            const AttnLanes l = attn_lanes(item, p.tile_tokens);
            if (item.tiles == 0) continue;
            const int first = max(0, l.first_visible / kAttnTile - item.tile_begin);
            for (int t = first; ok && t < item.tiles; ++t) {
                const int at = ring + ring_value(l.pair, t, item.tiles);
                const int stage = at % kStages;
                ok = wait(&sh.guard_full[stage], (phases >> stage) & 1);
                phases ^= 1u << stage;
                if (!ok) break;
                const int base = (item.tile_begin + t) * kAttnTile;
                const int shared_rows = max(0, l.first_visible - base), end = min(kAttnTile, item.keys - base);
                uint8_t* tile = smem_kv + stage * Shape::kTileBytes;
                bool found = false;
                constexpr int kVectors = DIM / 8;
                for (int i = shared_rows * kVectors + lane; i < kAttnTile * kVectors; i += 32) {
                    const int row = i / kVectors, vector = i % kVectors;
                    uint4* place = reinterpret_cast<uint4*>(tile + (vector / 8) * (kAttnTile * 128) + row * 128 + (vector % 8) * 16);
                    if (row >= end) {
                        *place = make_uint4(0, 0, 0, 0);
                        continue;
                    }
                    uint4 v = *place;
                    uint32_t words[4] = {v.x, v.y, v.z, v.w};
                    bool hit = false;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        constexpr uint32_t kExp = Element<T>::kExponent;
                        if ((words[w] & kExp) == kExp) {
                            words[w] &= 0xffff0000u;
                            hit = true;
                        }
                        if ((words[w] & (kExp << 16)) == (kExp << 16)) {
                            words[w] &= 0x0000ffffu;
                            hit = true;
                        }
                    }
                    if (hit) *place = make_uint4(words[0], words[1], words[2], words[3]);
                    found |= hit;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                found = __any_sync(0xffffffffu, found) != 0;
                __syncwarp();            // orders all lanes' writes before the arrival, which a vote does not
                if (lane == 0) {
                    if (found) *reinterpret_cast<volatile int*>(&sh.poison[units % kAttnPoison]) = units;
                    mbar_arrive(&sh.kv_full[stage]);
                }
            }
            ring += 2 * item.tiles;
        }
    } else {
        // ============================================================ softmax
        const int x = warp >> 2;                      // lane A or B
        const uint32_t tmem_row = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t tmem_s = tmem_row + kAttnColumnS + x * 128;
        constexpr int kToO = kAttnColumnO - kAttnColumnS;
        const float scale = p.scale_log2;
        // What a row of the tile means in an item, worked out where it is needed: the loop over the keys has 64 scores in
        // registers, and what it had to spill would go to L2 (shared memory takes all of L1).
        struct Row {
            int token, head;       // of the item, of the key head's group
            bool valid;
            int visible;           // keys it sees
        };
        auto row_of = [&](const AttnItem& it, bool pair) {
            Row r;
            const int row = (warp & 3) * 32 + lane, token_of_row = row / p.group;
            r.head = row - token_of_row * p.group;
            r.token = token_of_row + (pair ? x * p.tile_tokens : 0);
            r.valid = token_of_row < p.tile_tokens && r.token < it.tokens;
            r.visible = max(0, min(it.keys, it.visible + it.slope * r.token));
            return r;
        };
        int steps = 0, items = 0;       // steps and items with keys of this lane
        while (ok && take()) {
            const bool pair = item.tokens > p.tile_tokens;
            const int tiles = pair ? item.tiles : (item.tiles + 1 - x) / 2, tile_begin = item.tile_begin;
            const Row mine = row_of(item, pair);
            const bool active = __any_sync(0xffffffffu, mine.valid) != 0;
            const int visible = mine.visible;
            float top = -INFINITY, base = 0.0f;           // raw maximum in use, the same scaled
            float2 total = make_float2(0.0f, 0.0f);       // sum of weights
            // step `at` of the lane's count works in buffer at % 2; an item has an even number of them
            int at = steps;
            steps += 2 * tiles;
            // keys from the step's first one on that the row sees, and that all rows of this warp see
            int left = visible - (tile_begin + (pair ? 0 : x)) * kAttnTile;
            int left_all = __reduce_min_sync(0xffffffffu, left);
            auto hand_over = [&]() {
                tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[x][at & 1]);
            };
            // What is taken off the scaled scores for a new maximum.  Rounded up as fp16, and `moves` below rounds down, so that
            // no rounding of large scores lifts a weight above 2^(kAttnLazy + kHeadroom): 2^16 would be infinite.
            auto base_of = [&](float maximum) {
                if constexpr (Element<T>::kHeadroom == 0.0f) return maximum * scale;
                return __fadd_ru(__fmul_ru(maximum, scale), -Element<T>::kHeadroom);
            };
            uint32_t s[2][32];
            float step_top = -INFINITY;
            // the scores of a step, which have arrived in s: masked where a row does not see all of them, and their maximum
            auto take_scores = [&]() {
                if (left_all < kAttnHalf) {
                    mask_scores(s[0], left);
                    mask_scores(s[1], left - 32);
                }
                step_top = fmaxf(top_of(s[0]), top_of(s[1]));
            };
            auto next_step = [&]() {
                const int on = !pair && (at & 1) != 0 ? kAttnHalf + kAttnTile : kAttnHalf;     // the other lane's tile is passed over
                left -= on;
                left_all -= on;
            };
            // the weights of 32 scores, rounded to the element type for the product; the sum takes them unrounded
            const float2 scale2 = make_float2(scale, scale);
            auto weigh = [&](const uint32_t (&part)[32], uint32_t (&packed)[16]) {
                const float2 base2 = make_float2(-base, -base);
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float2 z = fma2(make_float2(__uint_as_float(part[2 * k]), __uint_as_float(part[2 * k + 1])), scale2, base2);
                    const float2 w = k % kAttnPolynomial == kAttnPolynomial - 1 ? exp2_polynomial(z) : make_float2(exp2_fast(z.x), exp2_fast(z.y));
                    sum = add2(sum, w);
                    packed[k] = Element<T>::pack(w.x, w.y);
                }
                total = add2(total, sum);
            };
            if (!active) {
                for (; ok && at < steps; ++at) {
                    ok = wait(&sh.s_full[x][at & 1], (at >> 1) & 1);
                    if (ok) hand_over();
                }
            } else if (at < steps) {
                ok = wait(&sh.s_full[x][0], (at >> 1) & 1);
                if (!ok) break;
                tcgen05_fence_after_sync();
                tmem_load_32(tmem_s, s[0]);
                tmem_load_32(tmem_s + 32, s[1]);
                tmem_load_wait(s[0]);
                tmem_load_wait(s[1]);
                take_scores();
                top = step_top;
                base = top == -INFINITY ? 0.0f : base_of(top);
                for (;; ++at) {
                    const uint32_t here = tmem_s + (at & 1) * kAttnHalf, there = tmem_s + ((at + 1) & 1) * kAttnHalf;
                    const bool more = at + 1 < steps;
                    uint64_t* next_full = &sh.s_full[x][(at + 1) & 1];
                    const uint32_t next_phase = ((at + 1) >> 1) & 1;
                    // The next step's scores, when they are there by now, are loaded into the registers that this
                    // step's exponentials free: the loads, half of the maximum and the hand-over run behind the
                    // second half of those.
                    uint32_t packed[16];
                    weigh(s[0], packed);
                    tmem_store_16(here, packed);
                    const bool early = more && __all_sync(0xffffffffu, mbar_test_wait(next_full, next_phase));
                    if (early) {
                        tcgen05_fence_after_sync();
                        tmem_load_32(there, s[0]);
                        next_step();
                        weigh(s[1], packed);
                        tmem_load_wait(s[0]);
                        const float lower_top = top_of(s[0]);
                        tmem_store_16(here + 16, packed);
                        tmem_load_32(there + 32, s[1]);
                        tmem_store_wait();
                        hand_over();
                        tmem_load_wait(s[1]);
                        if (left_all < kAttnHalf)
                            take_scores();
                        else
                            step_top = fmaxf(lower_top, top_of(s[1]));
                    } else {
                        weigh(s[1], packed);
                        tmem_store_16(here + 16, packed);
                        tmem_store_wait();
                        hand_over();
                        if (!more) break;
                        ok = wait(next_full, next_phase);
                        if (!ok) break;
                        tcgen05_fence_after_sync();
                        tmem_load_32(there, s[0]);
                        tmem_load_32(there + 32, s[1]);
                        next_step();
                        tmem_load_wait(s[0]);
                        tmem_load_wait(s[1]);
                        take_scores();
                    }
                    const bool moves = step_top > __fadd_rd(top, p.lazy);
                    if (__any_sync(0xffffffffu, moves)) {
                        float shrink = 1.0f;
                        if (moves) {
                            const float new_base = base_of(step_top);
                            shrink = top == -INFINITY ? 0.0f : exp2_fast(base - new_base);
                            top = step_top;
                            base = new_base;
                            total.x *= shrink;
                            total.y *= shrink;
                        }
                        // O has to hold the steps up to this one (the next step's scores imply all but that); the
                        // next P V waits for the next step's weights
                        ok = wait(&sh.pv_done[x], at & 1);
                        if (!ok) break;
                        tcgen05_fence_after_sync();
#pragma unroll 1
                        for (int c = 0; c < DIM; c += 16) {      // in small pieces: the scores sit in 64 registers
                            uint32_t o[16];
                            tmem_load_16(tmem_s + kToO + c, o);
                            tmem_load_wait16(o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
                            tmem_store_16(tmem_s + kToO + c, o);
                        }
                    }
                }
            }
            if (!ok) break;

            // ------------------------------------------------------ epilogue
            if (tiles > 0) {
                ok = wait(&sh.o_full[x], items & 1);
                ++items;
                if (!ok) break;
                tcgen05_fence_after_sync();
            }
            const float sum = total.x + total.y;
            read_unit(units - 1);
            done();
            const AttnLanes l = attn_lanes(item, p.tile_tokens);
            const Row r = row_of(item, l.pair);
            const bool valid = r.valid, direct = item.partial < 0;
            // lane B of a split item has rows of its own only among partial results
            const bool writes = __any_sync(0xffffffffu, valid) != 0 && item.partial != -2 && (l.pair || x == 0 || (!direct && item.slots > 1));
            const int head_index = head * p.group + r.head;
            const long long out_token = item.q_first + r.token;
            const bool empty = sum == 0.0f;
            const float inverse = empty ? 0.0f : 1.0f / sum;
            long long partial_row = 0;
            bool stores = valid && writes;
            if (!direct) {
                const int rows = item.tokens * p.group;
                const int slot = item.slot + (l.pair ? 0 : x);
                // a split entry of a single tile has one slot: lane A's
                if (!l.pair && x == 1 && slot >= item.slots) stores = false;
                partial_row = item.partial + (static_cast<long long>(head) * item.slots + slot) * rows + r.token * p.group + r.head;
            }
            const bool poisoned = tiles > 0 && *reinterpret_cast<volatile int*>(&sh.poison[units % kAttnPoison]) == units;
            if (writes) {
#pragma unroll 1
                for (int c = 0; c < DIM / 32; ++c) {
                    uint32_t o[32];
                    if (tiles > 0) {
                        tmem_load_32(tmem_s + kToO + c * 32, o);
                        tmem_load_wait(o);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = empty ? 0u : __float_as_uint(__uint_as_float(o[i]) * inverse);
                    if (poisoned && valid) {
                        const int from = max(l.first_visible, item.tile_begin * kAttnTile);
                        const int to = min(r.visible, (item.tile_begin + item.tiles) * kAttnTile);
#pragma unroll 1
                        for (int key = from; key < to; ++key) {
                            if (!l.pair && (((key / kAttnTile - item.tile_begin) & 1) != x)) continue;
                            const uint32_t* source = reinterpret_cast<const uint32_t*>(attn_value_row<T>(p, item, head, key) + c * 32);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint32_t word = source[i];
                                constexpr uint32_t kExp = Element<T>::kExponent;
                                if ((word & kExp) == kExp) o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) + Element<T>::value(word & 0xffffu));
                                if ((word >> 16 & kExp) == kExp)
                                    o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) + Element<T>::value(word >> 16));
                            }
                        }
                    }
                    if (stores && direct) {
                        T* out = static_cast<T*>(p.a.out) + out_token * p.a.out_token_stride + head_index * p.a.out_head_stride + c * 32;
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = Element<T>::pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
                        if (p.out_sectors != 0) {
                            store_sector(out, &o[0]);
                            store_sector(out + 16, &o[8]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                reinterpret_cast<uint4*>(out)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    } else if (stores && !empty) {
                        float* out = p.w.partial_out + partial_row * DIM + c * 32;
#pragma unroll
                        for (int i = 0; i < 4; ++i) store_sector(out + 8 * i, &o[8 * i]);
                    }
                }
                if (stores) {
                    const float lse2 = empty ? -INFINITY : base + log2f(sum);
                    if (!direct) {
                        p.w.partial_lse[partial_row] = lse2;
                    } else if (p.a.lse != nullptr) {
                        p.a.lse[out_token * p.a.heads + head_index] = lse2 * kLn2;
                    }
                }
            }
            if (tiles > 0) {
                tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.o_empty[x]);
            }
        }
    }
    if (!ok && lane == 0) {
        sh.abort = 1;
        atomicOr(p.status, ITK_SERVING_WAIT_EXPIRED);
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == kAttnMmaWarp) {
        if (sh.abort != 0) {
            // a wait expired: copies and UMMAs issued before that may still be in flight; neither shared
            // memory nor TMEM is given up under them
            const uint64_t until = global_timer_ns() + 2000000ull;
            while (global_timer_ns() < until) {
            }
        }
        __syncwarp();
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem, kAttnTmemColumns);
    }
}

// ------------------------------------------------------------------ join

constexpr int kJoinThreads = 256;

// out = sum_c 2^(lse_c - lse) out_c over the slots of a row (own ones, then the prefix's), in slot order.  One warp
// per row, kFlight partial rows on their way at a time; also clears the rows of no request when asked to.
//
// Bound by the chain record - statistics - rows - store, about 3 us for one token over 8192 keys.  Small calls have fewer rows than
// the device has warps and take the time of a trip per kFlight slots: 32 (a call of 15.5 us took 1 us longer with 16).  Large ones
// have rows for all warps, and 32 cost occupancy (128 registers, 197 for 32; 64 rows over a prefix of 16384 keys 84.4 and 88.2 us).
template <typename T, int DIM, int kFlight>
__global__ void __launch_bounds__(kJoinThreads) itk_attention_join_kernel(const __grid_constant__ AttnParams p) {
    constexpr int kOwn = DIM / 32;
    constexpr int kGroup = 4;            // partial rows that are asked for together
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int span = 2 * p.tile_tokens;
    const int heads = p.a.kv_heads;
    grid_wait();
    AttnCounters counters;
    for (int work = blockIdx.x;; work += gridDim.x) {
        // (the record is read before it is known whether there is one: what this kernel takes is the chain of loads that
        // depend on one another)
        const int index = work / heads, head = work - index * heads;
        const int4* source = reinterpret_cast<const int4*>(p.w.combines + min(index, p.w.max_combines - 1));
        const int4 record = source[0];
        const int row_first = source[1].x;
        if (work == static_cast<int>(blockIdx.x)) counters = *p.w.counters;
        if (work >= counters.combines * heads) break;
        const AttnCombine entry{record.x, record.y, record.z, record.w, row_first, {}};
        const int rows = entry.tokens * p.group, row_end = min(rows, entry.row_first + kAttnCombineRows);
        for (int r = entry.row_first + warp; r < row_end; r += kJoinThreads / 32) {
            const int token = entry.q_first + r / p.group;
            const int head_index = head * p.group + r % p.group;
            // the row's own partial results, then the prefix's: two runs of rows
            int count = entry.slots, prefix_count = 0, prefix_rows = 0;
            const int first = entry.partial + head * entry.slots * rows + r;       // (partial rows are counted in 31 bits)
            int prefix_first = 0;
            if (p.a.prefix_keys > 0 && token < counters.rows_end) {
                const int e = token / span;
                const int2 slots = p.w.prefix_slots[e];
                prefix_rows = min(span, counters.rows_end - e * span) * p.group;
                prefix_first = slots.x + head * slots.y * prefix_rows + (token - e * span) * p.group + r % p.group;
                prefix_count = slots.y;
            }
            count += prefix_count;
            auto row_of = [&](int c) {
                return c < entry.slots ? first + c * rows : prefix_first + (c - entry.slots) * prefix_rows;
            };
            float top = -INFINITY, total = 0.0f, sums[kOwn] = {};
            bool broken = false;
            for (int base = 0; base < count; base += kFlight) {
                const int here = min(kFlight, count - base);
                const float lse = lane < here ? p.w.partial_lse[row_of(base + lane)] : -INFINITY;
                float held[kFlight][kOwn];
#pragma unroll
                for (int k = 0; k < kFlight; ++k) {
                    if (k % kGroup == 0 && k >= here) break;
                    const float* values = p.w.partial_out + static_cast<size_t>(row_of(base + min(k, here - 1))) * DIM + lane * kOwn;
                    if constexpr (kOwn == 4) {
                        *reinterpret_cast<float4*>(held[k]) = *reinterpret_cast<const float4*>(values);
                    } else {
                        *reinterpret_cast<float2*>(held[k]) = *reinterpret_cast<const float2*>(values);
                    }
                }
                broken |= __any_sync(0xffffffffu, lse != lse) != 0;
                float new_top = fmaxf(top, lse);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) new_top = fmaxf(new_top, __shfl_xor_sync(0xffffffffu, new_top, d));
                if (new_top == -INFINITY) continue;
                const float shrink = exp2_fast(top - new_top), weight = exp2_fast(lse - new_top);
                top = new_top;
                total *= shrink;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) sums[i] *= shrink;
#pragma unroll
                for (int k = 0; k < kFlight; ++k) {
                    if (k % kGroup == 0 && k >= here) break;
                    const float w = __shfl_sync(0xffffffffu, weight, k);
                    total += w;
#pragma unroll
                    for (int i = 0; i < kOwn; ++i) sums[i] = w != 0.0f ? fmaf(w, held[k][i], sums[i]) : sums[i];   // an empty slot holds no values
                }
            }
            const bool empty = total == 0.0f && !broken;
            const float nan = __int_as_float(0x7fffffff);
            const float inverse = broken ? nan : (empty ? 0.0f : 1.0f / total);
            uint32_t packed[kOwn / 2];
#pragma unroll
            for (int i = 0; i < kOwn / 2; ++i) packed[i] = Element<T>::pack(sums[2 * i] * inverse, sums[2 * i + 1] * inverse);
            T* out = static_cast<T*>(p.a.out) + token * p.a.out_token_stride + head_index * p.a.out_head_stride + lane * kOwn;
            if constexpr (kOwn == 4) {
                *reinterpret_cast<uint2*>(out) = make_uint2(packed[0], packed[1]);
            } else {
                *reinterpret_cast<uint32_t*>(out) = packed[0];
            }
            if (lane == 0 && p.a.lse != nullptr)
                p.a.lse[static_cast<long long>(token) * p.a.heads + head_index] = broken ? nan : (empty ? -INFINITY : (top + log2f(total)) * kLn2);
        }
    }
    const bool clear_out = (p.a.clear_tail & 1) != 0, clear_lse = (p.a.clear_tail & 2) != 0 && p.a.lse != nullptr;
    if (clear_out || clear_lse) {
        // rows in front of the first request and behind the last one
        const long long head_rows = static_cast<long long>(counters.rows_begin) * p.a.heads;
        const long long tail = static_cast<long long>(max(counters.rows_end, counters.rows_begin)) * p.a.heads;
        const long long all = head_rows + static_cast<long long>(p.a.tokens) * p.a.heads - tail;
        for (long long i = static_cast<long long>(blockIdx.x) * (kJoinThreads / 32) + warp; i < all;
             i += static_cast<long long>(gridDim.x) * (kJoinThreads / 32)) {
            const long long r = i < head_rows ? i : tail + i - head_rows;
            const long long token = r / p.a.heads, head = r - token * p.a.heads;
            T* out = static_cast<T*>(p.a.out) + token * p.a.out_token_stride + head * p.a.out_head_stride + lane * kOwn;
            if (clear_out) {
                if constexpr (kOwn == 4) {
                    *reinterpret_cast<uint2*>(out) = make_uint2(0u, 0u);
                } else {
                    *reinterpret_cast<uint32_t*>(out) = 0u;
                }
            }
            if (lane == 0 && clear_lse) p.a.lse[r] = -INFINITY;
        }
    }
}

}  // namespace itk
