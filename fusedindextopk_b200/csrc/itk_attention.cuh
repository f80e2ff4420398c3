// Attention of packed, paged and shared-prefix batches.
//
//     s_j = scale * q . k_j,   m = max_j s_j,   l = sum_j exp(s_j - m),   out = sum_j exp(s_j - m) v_j / l
//
// over the prefix keys (all of them) and the request's own keys (the first min(N, N - Q + i + 1) of them for row i
// of Q when causal).  Scores, statistics and sums are fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/itk_b200.h"
#include "itk_ptx.cuh"

namespace itk {

constexpr int kRowsKernelThreads = 128;

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Lengths of one request, clamped to the buffers they index.
struct AttentionRequest {
    int q_first, q_count, k_first, k_count;
};

__device__ __forceinline__ AttentionRequest attention_request(const itk_attention_args& p, int b, int* status) {
    AttentionRequest r;
    const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1];
    r.q_first = min(max(q0, 0), p.tokens);
    r.q_count = max(min(max(q1, 0), p.tokens) - r.q_first, 0);
    bool bad = q0 != r.q_first || q1 != r.q_first + r.q_count;
    if (p.cu_k != nullptr) {
        const int k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
        r.k_first = min(max(k0, 0), p.own.page_size);
        r.k_count = max(min(max(k1, 0), p.own.page_size) - r.k_first, 0);
        bad |= k0 != r.k_first || k1 != r.k_first + r.k_count;
    } else {
        const int n = p.lens_k[b];
        const long long room = static_cast<long long>(p.own.table_pages) * p.own.page_size;
        r.k_first = 0;
        r.k_count = static_cast<int>(min(static_cast<long long>(max(n, 0)), room));
        bad |= n != r.k_count;
    }
    if (bad) atomicOr(status, ITK_SERVING_BAD_LENGTHS);
    return r;
}

// One warp per (row, head): the plainest form.  32 keys at a time, a lane scores one of them; the weighted values
// are added with every lane owning dim / 32 columns.
template <typename T, int DIM>
__global__ void __launch_bounds__(kRowsKernelThreads) itk_attention_rows_kernel(const itk_attention_args p, int* status) {
    constexpr int kOwn = DIM / 32;
    __shared__ float q_rows[kRowsKernelThreads / 32][DIM];
    const int lane = threadIdx.x & 31;
    float* q_row = q_rows[threadIdx.x >> 5];
    const long long work = static_cast<long long>(blockIdx.x) * (kRowsKernelThreads / 32) + (threadIdx.x >> 5);
    if (work >= static_cast<long long>(p.tokens) * p.heads) return;
    const int token = static_cast<int>(work / p.heads), head = static_cast<int>(work - static_cast<long long>(token) * p.heads);
    const int kv_head = head / (p.heads / p.kv_heads);
    T* out = static_cast<T*>(p.out) + token * p.out_token_stride + head * p.out_head_stride;

    int low = 0, high = p.requests;
    while (high - low > 1) {
        const int middle = (low + high) >> 1;
        if (p.cu_q[middle] <= token) {
            low = middle;
        } else {
            high = middle;
        }
    }
    const AttentionRequest r = attention_request(p, low, status);
    if (token < r.q_first || token >= r.q_first + r.q_count) {
        if (p.clear_tail) {
            for (int c = lane; c < DIM; c += 32) out[c] = from_float<T>(0.0f);
            if (lane == 0 && p.lse != nullptr) p.lse[work] = -INFINITY;
        }
        return;
    }
    const int visible = p.causal ? min(r.k_count, r.k_count - r.q_count + (token - r.q_first) + 1) : r.k_count;
    const T* q = static_cast<const T*>(p.q) + token * p.q_token_stride + head * p.q_head_stride;
    for (int c = lane; c < DIM; c += 32) q_row[c] = to_float<T>(q[c]);
    __syncwarp();

    float top = -INFINITY, total = 0.0f, sums[kOwn] = {};
    for (int part = 0; part < 2; ++part) {
        const itk_kv_segment& seg = part == 0 ? p.prefix : p.own;
        const int keys = part == 0 ? (p.prefix.k != nullptr ? p.prefix_keys : 0) : visible;
        const int first = part == 0 ? 0 : r.k_first;
        const int32_t* table = seg.table == nullptr ? nullptr : seg.table + (part == 0 ? 0 : low * seg.table_stride);
        for (int base = 0; base < keys; base += 32) {
            const int key = base + lane;
            float score = -INFINITY;
            const T* v_row = nullptr;
            if (key < keys) {
                long long page = 0, row = first + key;
                if (table != nullptr) {
                    page = table[key / seg.page_size];
                    row = key % seg.page_size;
                    if (page < 0 || page >= seg.pages) {
                        atomicOr(status, ITK_SERVING_BAD_PAGE);
                        page = page < 0 ? 0 : seg.pages - 1;
                    }
                }
                const T* k_row = static_cast<const T*>(seg.k) + page * seg.k_page_stride + row * seg.k_row_stride + kv_head * seg.k_head_stride;
                v_row = static_cast<const T*>(seg.v) + page * seg.v_page_stride + row * seg.v_row_stride + kv_head * seg.v_head_stride;
                float dot = 0.0f;
                for (int c = 0; c < DIM; c += 8) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(k_row + c);
                    const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dot = fmaf(q_row[c + i], to_float<T>(x[i]), dot);
                }
                score = dot * p.scale;
            }
            float tile_top = score;
            for (int step = 16; step > 0; step >>= 1) tile_top = fmaxf(tile_top, __shfl_xor_sync(0xffffffffu, tile_top, step));
            const float new_top = fmaxf(top, tile_top);
            const float base_top = new_top == -INFINITY ? 0.0f : new_top;
            const float shrink = expf(top - base_top);
            const float weight = key < keys ? expf(score - base_top) : 0.0f;
            top = new_top;
            total = total * shrink + weight;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) sums[i] *= shrink;
            const int count = min(32, keys - base);
            for (int j = 0; j < count; ++j) {
                const float w = __shfl_sync(0xffffffffu, weight, j);
                const T* row = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(v_row), j));
#pragma unroll
                for (int i = 0; i < kOwn; ++i) sums[i] = fmaf(w, to_float<T>(row[lane + 32 * i]), sums[i]);
            }
        }
    }
    for (int step = 16; step > 0; step >>= 1) total += __shfl_xor_sync(0xffffffffu, total, step);
    const bool empty = total == 0.0f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) out[lane + 32 * i] = from_float<T>(empty ? 0.0f : sums[i] / total);
    if (lane == 0 && p.lse != nullptr) p.lse[work] = empty ? -INFINITY : top + logf(total);
}

}  // namespace itk
