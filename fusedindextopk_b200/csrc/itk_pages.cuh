// Page bookkeeping of a serving step: block tables and slot maps from request lengths, and the writing of a
// step's tokens into the key / value and index-key pools.
#pragma once

#include "../../include/itk_b200.h"
#include "itk_quantize.cuh"

namespace itk {

// ------------------------------------------------------------------ page plan

constexpr int kPlanThreads = 512;

// Inclusive prefix sums of three values over the block.
struct PlanSums {
    long long fresh;
    int need, after;
};

__device__ __forceinline__ PlanSums block_scan(PlanSums v, PlanSums* warp_totals) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
        const long long fresh = __shfl_up_sync(0xffffffffu, v.fresh, step);
        const int need = __shfl_up_sync(0xffffffffu, v.need, step);
        const int after = __shfl_up_sync(0xffffffffu, v.after, step);
        if (lane >= step) {
            v.fresh += fresh;
            v.need += need;
            v.after += after;
        }
    }
    if (lane == 31) warp_totals[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
        v.fresh += warp_totals[w].fresh;
        v.need += warp_totals[w].need;
        v.after += warp_totals[w].after;
    }
    return v;
}

struct PlanRequest {
    int old, before, after, length;
    long long fresh;
    bool clamped, no_room;
};

__device__ __forceinline__ PlanRequest plan_request(const itk_page_plan_args& p, int b) {
    PlanRequest r;
    const long long room = static_cast<long long>(p.table_pages) * p.page_size;
    const long long old = p.old[b], fresh = p.fresh[b];
    r.clamped = old < 0 || fresh < 0;
    r.no_room = max(old, 0ll) + max(fresh, 0ll) > room;
    r.old = static_cast<int>(min(max(old, 0ll), room));
    r.fresh = max(fresh, 0ll);
    r.length = static_cast<int>(min(r.old + r.fresh, room));
    r.before = (r.old + p.page_size - 1) / p.page_size;
    r.after = (r.length + p.page_size - 1) / p.page_size;
    return r;
}

// What every CTA knows of the requests: rows, free pages and flat entries before each.
struct PlanState {
    const int *cu, *taken, *first;
};

// Slots and key ranges, kRows neighbouring rows at a time.
template <int kRows>
__device__ __forceinline__ void plan_rows(const itk_page_plan_args& p, const PlanState& state, unsigned start, unsigned stride) {
    const int last = state.cu[p.requests];
    const unsigned units = (static_cast<unsigned>(p.rows) + kRows - 1) / kRows;
    for (unsigned unit = start; unit < units; unit += stride) {
        long long slots[kRows];
        int starts[kRows], ends[kRows];
        const unsigned base = unit * kRows;
        PlanRequest r{};
        int b = 0;
        unsigned until = base;                  // rows below it are of request b
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const unsigned row = base + i;
            slots[i] = -1;
            starts[i] = ends[i] = 0;
            if (row >= static_cast<unsigned>(last)) continue;
            if (row >= until) {
                int low = b, high = p.requests;     // cu[low] <= row < cu[high]
                while (high - low > 1) {
                    const int middle = (low + high) >> 1;
                    if (static_cast<unsigned>(state.cu[middle]) <= row) {
                        low = middle;
                    } else {
                        high = middle;
                    }
                }
                b = low;
                until = state.cu[b + 1];
                r = plan_request(p, b);
            }
            const long long position = static_cast<long long>(r.old) + row - state.cu[b];
            starts[i] = state.first[b] * p.page_size;
            ends[i] = starts[i] + static_cast<int>(min(position + 1, static_cast<long long>(r.length)));
            if (position < r.length) {
                const int column = static_cast<int>(position) / p.page_size;
                int page = -1;
                if (column < r.before) {
                    page = p.table[b * p.table_stride + column];
                } else {
                    const int next = state.taken[b] + column - r.before;
                    if (next < p.free_count) page = p.free_pages[next];
                }
                if (page >= 0) slots[i] = static_cast<long long>(page) * p.page_size + position % p.page_size;
            }
        }
        if constexpr (kRows == 4) {
            if (base + 4 <= static_cast<unsigned>(p.rows)) {
                *reinterpret_cast<longlong2*>(p.slots + base) = make_longlong2(slots[0], slots[1]);
                *reinterpret_cast<longlong2*>(p.slots + base + 2) = make_longlong2(slots[2], slots[3]);
                *reinterpret_cast<int4*>(p.k_start + base) = make_int4(starts[0], starts[1], starts[2], starts[3]);
                *reinterpret_cast<int4*>(p.k_end + base) = make_int4(ends[0], ends[1], ends[2], ends[3]);
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (base + i < static_cast<unsigned>(p.rows)) {
                p.slots[base + i] = slots[i];
                p.k_start[base + i] = starts[i];
                p.k_end[base + i] = ends[i];
            }
    }
}

// One launch.  Every CTA scans all requests itself (a few KB that sit in L2) and keeps the prefix sums in shared
// memory, so that table cells and rows can be filled by all CTAs with no second launch and no hand-off: the page of
// a position is either an old cell of the table, which no CTA writes, or free_pages[taken before + ...], which is
// computed, not read back.  Bound by latency for the batches of a decode step (8 requests: 4.3 us, of which the launch is
// 2.2), by the chain search - lengths - page - store for large ones (1024 requests, 300000 rows: 9.4 us for 8 MB; the
// writes alone, 16 B per row and 8 B per table cell, would take 1.2).
__global__ void __launch_bounds__(kPlanThreads) itk_plan_pages_kernel(const itk_page_plan_args p, int wide, int* status) {
    extern __shared__ int plan_smem[];
    int* cu = plan_smem;                        // [B + 1] rows before request b, clamped to the row buffer
    int* taken = plan_smem + p.requests + 1;    // [B] free pages handed out before request b
    int* first = taken + p.requests;            // [B] flat entries before request b
    __shared__ PlanSums warp_totals[kPlanThreads / 32];
    __shared__ int total_pages;

    const int per_thread = (p.requests + kPlanThreads - 1) / kPlanThreads;
    const int lo = min(static_cast<int>(threadIdx.x) * per_thread, p.requests);
    const int hi = min(lo + per_thread, p.requests);
    PlanSums mine{0, 0, 0};
    bool clamped = false, no_room = false;
    for (int b = lo; b < hi; ++b) {
        const PlanRequest r = plan_request(p, b);
        mine.fresh += r.fresh;
        mine.need += r.after - r.before;
        mine.after += r.after;
        clamped |= r.clamped;
        no_room |= r.no_room;
    }
    const PlanSums upto = block_scan(mine, warp_totals);
    PlanSums run{upto.fresh - mine.fresh, upto.need - mine.need, upto.after - mine.after};
    const long long rows = p.rows;
    for (int b = lo; b < hi; ++b) {
        const PlanRequest r = plan_request(p, b);
        cu[b] = static_cast<int>(min(run.fresh, rows));
        taken[b] = run.need;
        first[b] = run.after;
        if (blockIdx.x == 0) {
            p.cu_q[b] = cu[b];
            p.lengths[b] = r.length;
        }
        run.fresh += r.fresh;
        run.need += r.after - r.before;
        run.after += r.after;
    }
    if (threadIdx.x == kPlanThreads - 1) {
        cu[p.requests] = static_cast<int>(min(upto.fresh, rows));
        total_pages = upto.after;
        if (blockIdx.x == 0) {
            p.cu_q[p.requests] = cu[p.requests];
            p.pages_needed[0] = upto.need;
            if (upto.need > p.free_count) no_room = true;
            if (upto.fresh > rows) clamped = true;
        }
    }
    if (blockIdx.x == 0 && (clamped || no_room))
        atomicOr(status, (clamped ? ITK_SERVING_BAD_LENGTHS : 0) | (no_room ? ITK_SERVING_OUT_OF_PAGES : 0));
    __syncthreads();

    // counted unsigned: up to 2^31 - 1 cells or rows, and a step behind the last
    const unsigned stride = gridDim.x * kPlanThreads;
    const unsigned start = blockIdx.x * kPlanThreads + threadIdx.x;
    const unsigned cells = static_cast<unsigned>(p.requests) * static_cast<unsigned>(p.table_pages);
    for (unsigned cell = start; cell < cells; cell += stride) {
        const int b = static_cast<int>(cell / static_cast<unsigned>(p.table_pages));
        const int column = static_cast<int>(cell) - b * p.table_pages;
        const PlanRequest r = plan_request(p, b);
        int32_t* entry = p.table + b * p.table_stride + column;
        int page = -1;
        if (column < r.before) {
            page = *entry;
        } else {
            const int next = taken[b] + column - r.before;
            if (column < r.after && next < p.free_count) {
                page = p.free_pages[next];
                if (page < 0) atomicOr(status, ITK_SERVING_OUT_OF_PAGES);      // a free list padded to a fixed length
            }
            *entry = page;
        }
        if (column < r.after) p.flat[first[b] + column] = page;
    }
    for (unsigned entry = total_pages + start; entry < cells; entry += stride) p.flat[entry] = 0;

    // Four neighbouring rows a thread when one each is not enough: most are of one request, so that it is looked for once, and
    // their stores are wide (300000 rows of 1024 requests: 10.4 -> 9.4 us).  One each otherwise: four take longer than one
    // (8 requests: 4.3 us, 6.3 with four).
    const PlanState state{cu, taken, first};
    if (wide && static_cast<unsigned>(p.rows) > stride)
        plan_rows<4>(p, state, start, stride);
    else
        plan_rows<1>(p, state, start, stride);
}

// ------------------------------------------------------------------ append

constexpr int kAppendThreads = 128;

template <typename Source>
__device__ __forceinline__ void load_index_quad(const Source* row, int lane, float (&x)[4]);

template <>
__device__ __forceinline__ void load_index_quad<float>(const float* row, int lane, float (&x)[4]) {
    const float4 raw = reinterpret_cast<const float4*>(row)[lane];
    x[0] = raw.x;
    x[1] = raw.y;
    x[2] = raw.z;
    x[3] = raw.w;
}

template <>
__device__ __forceinline__ void load_index_quad<__nv_bfloat16>(const __nv_bfloat16* row, int lane, float (&x)[4]) {
    const uint2 raw = reinterpret_cast<const uint2*>(row)[lane];
    x[0] = __uint_as_float(raw.x << 16);
    x[1] = __uint_as_float(raw.x & 0xffff0000u);
    x[2] = __uint_as_float(raw.y << 16);
    x[3] = __uint_as_float(raw.y & 0xffff0000u);
}

// One warp per token: the slot is read once, keys and values move as 16-byte vectors with up to eight loads in
// flight per lane, and the index key (128 elements, four per lane) is quantised from registers.  Bound by HBM: 8191 tokens
// of 8 heads of 128 with bf16 index keys take 13.4 us, 5.2 TB/s or 0.79 of the copy rate; 64 tokens 3.2 us, a launch.
template <typename Source>
__global__ void __launch_bounds__(kAppendThreads) itk_append_tokens_kernel(const itk_append_args p, int* status) {
    const unsigned token = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (token >= static_cast<unsigned>(p.tokens)) return;
    const long long slot = p.slots[token];
    if (slot < 0) return;
    if (slot >= static_cast<long long>(p.pages) * p.page_size) {
        if (lane == 0) atomicOr(status, ITK_SERVING_BAD_PAGE);
        return;
    }
    const unsigned page = static_cast<unsigned>(slot) / static_cast<unsigned>(p.page_size);
    const unsigned row = static_cast<unsigned>(slot) - page * static_cast<unsigned>(p.page_size);

    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.index_source != nullptr)
        load_index_quad(static_cast<const Source*>(p.index_source) + token * p.index_stride, lane, x);

    const int head_shift = p.dim == 128 ? 4 : 3;     // 16-byte vectors per head: dim / 8
    const int vectors = p.kv_heads << head_shift;
    const uint16_t* k = static_cast<const uint16_t*>(p.k) + token * p.k_token_stride;
    const uint16_t* v = static_cast<const uint16_t*>(p.v) + token * p.v_token_stride;
    uint16_t* k_out = static_cast<uint16_t*>(p.k_pool) + page * p.k_page_stride + row * p.k_row_stride;
    uint16_t* v_out = static_cast<uint16_t*>(p.v_pool) + page * p.v_page_stride + row * p.v_row_stride;
    for (int base = 0; base < vectors; base += 128) {
        uint4 held[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int vector = base + i * 32 + lane;
            if (vector < vectors) {
                const int head = vector >> head_shift, column = (vector - (head << head_shift)) * 8;
                held[0][i] = load_stream16(k + head * p.k_head_stride + column);
                held[1][i] = load_stream16(v + head * p.v_head_stride + column);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int vector = base + i * 32 + lane;
            if (vector < vectors) {
                const int head = vector >> head_shift, column = (vector - (head << head_shift)) * 8;
                *reinterpret_cast<uint4*>(k_out + head * p.k_pool_head_stride + column) = held[0][i];
                *reinterpret_cast<uint4*>(v_out + head * p.v_pool_head_stride + column) = held[1][i];
            }
        }
    }
    if (p.index_source == nullptr) return;

    float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, step));
    const float scale = __fdiv_rn(fmaxf(amax, kQuantAmaxFloor), kE4m3Max);
    const RowDivisor divisor = make_row_divisor(scale);
    static_cast<uint32_t*>(p.index_pool)[slot * 32 + lane] = e4m3x4(
        divisor.quotient(x[0]), divisor.quotient(x[1]), divisor.quotient(x[2]), divisor.quotient(x[3]));
    if (lane == 0) p.index_scales[slot] = scale;
}

}  // namespace itk
