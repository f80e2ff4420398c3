// C-ABI entry points of the serving step around the operator: page plans, token appends and attention.
#include "itk_host.cuh"

#include <algorithm>
#include <initializer_list>

#include "itk_attention.cuh"
#include "itk_pages.cuh"

namespace {

using namespace itk;

// One status word per device context, part of the library image: every serving kernel reports into it, and no
// caller has to carry a buffer for it.
__device__ int g_serving_status;
__device__ int g_serving_taken;

// Reads the word, and clears it in the same step: a bit that another stream sets meanwhile is in this report or in the next.
__global__ void itk_take_status_kernel(int clear) { g_serving_taken = clear ? atomicExch(&g_serving_status, 0) : atomicOr(&g_serving_status, 0); }

constexpr int kMaxDevices = 64;

struct DeviceState {
    bool ready = false;
    int sm_count = 0;
    int* status = nullptr;
};
std::mutex g_device_mutex;
DeviceState g_devices[kMaxDevices];

template <typename Kernel>
cudaError_t raise_smem(Kernel kernel, int bytes) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

int current_device(DeviceState* state) {
    int device = 0;
    ITK_CUDA(cudaGetDevice(&device));
    if (device < 0 || device >= kMaxDevices) return fail(ITK_ERR_UNSUPPORTED, "device index %d out of range", device);
    std::lock_guard<std::mutex> lock(g_device_mutex);
    DeviceState& d = g_devices[device];
    if (!d.ready) {
        int major = 0;
        ITK_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
        if (major != 10) return fail(ITK_ERR_UNSUPPORTED, "device %d is not sm_100; this library is built for sm_100a only", device);
        ITK_CUDA(cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, device));
        void* address = nullptr;
        ITK_CUDA(cudaGetSymbolAddress(&address, g_serving_status));
        d.status = static_cast<int*>(address);
        ITK_CUDA(cudaFuncSetAttribute(itk_plan_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (3 * ITK_MAX_PLAN_REQUESTS + 1) * static_cast<int>(sizeof(int))));
        ITK_CUDA(raise_smem(itk_attention_kernel<__nv_bfloat16, 128>, AttnShape<128>::kSmemBytes));
        ITK_CUDA(raise_smem(itk_attention_kernel<__nv_bfloat16, 64>, AttnShape<64>::kSmemBytes));
        ITK_CUDA(raise_smem(itk_attention_kernel<__half, 128>, AttnShape<128>::kSmemBytes));
        ITK_CUDA(raise_smem(itk_attention_kernel<__half, 64>, AttnShape<64>::kSmemBytes));
        d.ready = true;
    }
    *state = d;
    return ITK_OK;
}

int launched(const char* what) {
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(ITK_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(status));
    return ITK_OK;
}

bool strides_ok(std::initializer_list<long long> strides) {
    for (const long long s : strides)
        if (s < 0 || s % 8 != 0) return false;
    return true;
}

struct Bytes {
    const void* first;
    size_t count;
};

bool overlap(const Bytes& x, const Bytes& y) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x.first), b = reinterpret_cast<uintptr_t>(y.first);
    return x.count > 0 && y.count > 0 && a < b + y.count && b < a + x.count;
}

// Rows of a pool are counted in 31 bits; addresses are formed in 64.
bool pool_rows_ok(long long pages, long long page_size) { return pages > 0 && page_size > 0 && pages * page_size < (1ll << 31); }

int check_segment(const itk_kv_segment& s, const void* k, const void* v, const int32_t* table, const char* what) {
    ITK_REQUIRE(k && v, "%s: keys and values must not be null", what);
    ITK_REQUIRE(aligned16(k) && aligned16(v), "%s: keys and values must be 16-byte aligned", what);
    ITK_REQUIRE(strides_ok({s.k_page_stride, s.k_row_stride, s.k_head_stride, s.v_page_stride, s.v_row_stride, s.v_head_stride}),
                "%s: strides must be multiples of 8 elements", what);
    ITK_REQUIRE(pool_rows_ok(s.pages, s.page_size), "%s: need 0 < pages * page_size < 2^31", what);
    if (table != nullptr) {
        ITK_REQUIRE(s.page_size % 128 == 0, "%s: page_size must be a multiple of 128", what);
        ITK_REQUIRE(s.table_pages >= 0 && s.table_stride >= 0, "%s: table sizes must not be negative", what);
    } else {
        ITK_REQUIRE(s.pages == 1, "%s: keys without a table are one page", what);
        ITK_REQUIRE(s.page_size <= ITK_MAX_ATTENTION_KEYS, "%s: need at most %d keys", what, ITK_MAX_ATTENTION_KEYS);
    }
    return ITK_OK;
}

int check_attention(const itk_attention_args& a) {
    ITK_REQUIRE(a.tokens >= 0 && a.requests >= 0 && a.prefix_keys >= 0, "sizes must not be negative");
    ITK_REQUIRE(a.heads > 0 && a.kv_heads > 0 && a.heads % a.kv_heads == 0 && a.heads / a.kv_heads <= 128,
                "heads must be a multiple of kv_heads, at most 128 times as many");
    ITK_REQUIRE(a.dim == 64 || a.dim == 128, "head dimension must be 64 or 128");
    ITK_REQUIRE(a.element == ITK_ELEMENT_BF16 || a.element == ITK_ELEMENT_FP16, "element must be bf16 or fp16");
    ITK_REQUIRE(static_cast<long long>(a.tokens) * a.heads < (1ll << 31), "tokens * heads must stay below 2^31");
    return ITK_OK;
}

// Tokens of a row tile: as many as fit.
int attention_tile_tokens(const itk_attention_args& a) { return kAttnTile / (a.heads / a.kv_heads); }

constexpr int kAttnMaxSms = 160;     // the workspace is sized for any device the library runs on

// Workspace of a call: what the plan kernel can write at most.  With T tokens, B requests and 2 TT tokens per entry
// there are at most T / (2 TT) + B own entries; the prefix has T / (2 TT) + 1.  A chunk costs at least a kAttnWaves-th of an
// SM's share of the work (less a hundredth: the share is rounded up, its part down), so that chunking adds at most
// kAttnWaves items per SM over all key heads.
// Partial rows.  Entries of up to TT tokens, at most one per request and 128 rows per key head each, have two lanes.  Without a
// prefix longer ones have partial results only when they are cut, which takes half a share of work each, so that there are two
// of them per SM at most; with one every own row and every prefix row has a result, the last prefix entry two.  An added chunk has
// one result for each of up to 256 rows or two for each of up to 128, and no row has more of them than there are for one key head.
//
// 64 tokens of 64/8 heads of 128 ask for 135 MB, of which the added chunks' part, 128 MB at dimension 128, is the same for every larger
// call (the lengths are not known here, and one long entry among short ones can take all of them); 4096 rows of one request ask
// for 172 MB, 8192 rows of 64 heads behind a prefix for 674, two results in fp32 per row.
int attention_workspace(const itk_attention_args& a, AttnWorkspace* w, size_t* bytes) {
    const long long span = 2 * attention_tile_tokens(a);
    const long long rows = static_cast<long long>(a.tokens) * a.heads;
    const long long own = a.tokens / span + a.requests, prefix = a.prefix_keys > 0 ? a.tokens / span + 1 : 0;
    constexpr long long kAdded = kAttnMaxSms * kAttnWaves * 101ll / 100 + 1, kCut = kAttnMaxSms * 2 * 101ll / 100 + 1;
    const long long short_rows = std::min(rows, static_cast<long long>(a.requests) * kAttnTile * a.kv_heads);
    long long partial = std::min(kAdded * 2 * kAttnTile, 2 * rows * (kAdded / a.kv_heads));
    if (prefix > 0)
        partial += rows + short_rows + rows + static_cast<long long>(kAttnTile) * a.kv_heads;
    else
        partial += 2 * short_rows + std::min(rows, kCut * 2 * kAttnTile);
    ITK_REQUIRE(partial < (1ll << 31) - 1 && own < kAttnMostEntries && (own + prefix + kAdded) * a.kv_heads < (1ll << 31),
                "the batch is too large for one call");
    size_t at = 0;
    auto take = [&](size_t size) {
        const size_t offset = at;
        at += (size + 255) / 256 * 256;
        return static_cast<char*>(a.workspace) + offset;
    };
    const long long combines = (rows / a.kv_heads + kAttnCombineRows - 1) / kAttnCombineRows + own;
    ITK_REQUIRE(combines * a.kv_heads < (1ll << 31), "the batch is too large for one call");
    w->max_entries = static_cast<int>(own);
    w->max_combines = static_cast<int>(combines);
    w->max_items = static_cast<int>(own + prefix + kAdded);
    w->max_partial_rows = static_cast<int>(partial);
    w->counters = reinterpret_cast<AttnCounters*>(take(sizeof(AttnCounters)));
    w->entry_first = reinterpret_cast<int*>(take((static_cast<size_t>(a.requests) + 1) * sizeof(int)));
    w->prefix_slots = reinterpret_cast<int2*>(take(static_cast<size_t>(prefix) * sizeof(int2)));
    w->items = reinterpret_cast<AttnItem*>(take(static_cast<size_t>(w->max_items) * sizeof(AttnItem)));
    w->combines = reinterpret_cast<AttnCombine*>(take(static_cast<size_t>(combines) * sizeof(AttnCombine)));
    w->partial_lse = reinterpret_cast<float*>(take(static_cast<size_t>(partial) * sizeof(float)));
    w->partial_out = reinterpret_cast<float*>(take(static_cast<size_t>(partial) * a.dim * sizeof(float)));
    *bytes = at;
    return ITK_OK;
}

int encode_map(CUtensorMap* map, int element, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
               const cuuint32_t* box) {
    EncodeTiled encode = encode_tiled_entry();
    if (encode == nullptr) return fail(ITK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    const CUresult result = encode(
        map, element == ITK_ELEMENT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
        static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS) return fail(ITK_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", int(result));
    return ITK_OK;
}

// Bytes between the entries of a dimension; one with a single entry may carry any stride, which nothing steps over.
cuuint64_t map_stride(long long elements, long long count) { return count > 1 || elements > 0 ? elements * 2 : 16; }

// [pages, page_size, kv_heads, dim] in any order of strides; a box is 128 rows of 64 columns of one head.
int segment_map(CUtensorMap* map, const itk_attention_args& a, const itk_kv_segment& s, const void* base, long long page_stride,
                long long row_stride, long long head_stride) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.kv_heads),
                                static_cast<cuuint64_t>(s.page_size), static_cast<cuuint64_t>(s.pages)};
    const cuuint64_t strides[3] = {map_stride(head_stride, a.kv_heads), map_stride(row_stride, s.page_size), map_stride(page_stride, s.pages)};
    const cuuint32_t box[4] = {64, 1, kAttnTile, 1};
    return encode_map(map, a.element, 4, base, dims, strides, box);
}

// A launch whose prologue may overlap the kernel before it on the stream.
template <typename Kernel, typename Params>
cudaError_t launch_after(Kernel kernel, int grid, int threads, size_t smem, cudaStream_t stream, const Params& params) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, params);
}

template <typename T, int DIM>
int launch_attention(const AttnParams& params, cudaStream_t stream) {
    if (params.small_plan) {
        itk_attention_kernel<T, DIM><<<params.sm_count, kAttnThreads, AttnShape<DIM>::kSmemBytes, stream>>>(params);
    } else {
        // barriers of a small block cost a third of a large one's; the large one is for batches with more entries than threads
        if (params.w.max_entries <= 256)
            itk_attention_plan_kernel<256><<<1, 256, 0, stream>>>(params);
        else
            itk_attention_plan_kernel<1024><<<1, 1024, 0, stream>>>(params);
        ITK_CUDA(launch_after(itk_attention_kernel<T, DIM>, params.sm_count, kAttnThreads, AttnShape<DIM>::kSmemBytes, stream, params));
    }
    if (params.small_plan)
        ITK_CUDA(launch_after(itk_attention_join_kernel<T, DIM, 32>, 4 * params.sm_count, kJoinThreads, 0, stream, params));
    else
        ITK_CUDA(launch_after(itk_attention_join_kernel<T, DIM, 16>, 4 * params.sm_count, kJoinThreads, 0, stream, params));
    return launched("itk_attention_kernel");
}

}  // namespace

extern "C" {

int itk_serving_status(int* status, int clear) {
    ITK_REQUIRE(status != nullptr, "status must not be null");
    DeviceState device;
    const int rc = current_device(&device);
    if (rc != ITK_OK) return rc;
    static std::mutex taking;                  // of the word in between
    std::lock_guard<std::mutex> lock(taking);
    ITK_CUDA(cudaDeviceSynchronize());
    itk_take_status_kernel<<<1, 1>>>(clear);
    ITK_CUDA(cudaGetLastError());
    ITK_CUDA(cudaMemcpyFromSymbol(status, g_serving_taken, sizeof(int)));
    return ITK_OK;
}

int itk_plan_pages(const itk_page_plan_args* args, itk_stream_t stream) {
    ITK_REQUIRE(args != nullptr, "args must not be null");
    const itk_page_plan_args& a = *args;
    ITK_REQUIRE(a.requests > 0 && a.requests <= ITK_MAX_PLAN_REQUESTS, "need 0 < requests <= %d", ITK_MAX_PLAN_REQUESTS);
    ITK_REQUIRE(a.rows >= 0 && a.free_count >= 0, "sizes must not be negative");
    ITK_REQUIRE(a.table_pages > 0 && a.page_size > 0 && a.table_stride >= a.table_pages &&
                    static_cast<long long>(a.requests) * a.table_pages < (1ll << 31) / a.page_size,
                "need 0 < requests * table_pages * page_size < 2^31 and a row stride of at least table_pages");
    ITK_REQUIRE(a.table && a.old && a.fresh && a.cu_q && a.lengths && a.flat && a.pages_needed &&
                    (a.free_pages || a.free_count == 0) && ((a.slots && a.k_start && a.k_end) || a.rows == 0),
                "page plan pointers must not be null");
    // Every CTA reads the lengths and the free list for itself while others write: a plan's lengths, for one, cannot be the
    // next plan's old lengths in the same buffers.
    {
        const size_t word = sizeof(int32_t), requests = a.requests, rows = a.rows;
        const Bytes reads[] = {{a.old, requests * word}, {a.fresh, requests * word}, {a.free_pages, a.free_count * word}};
        const Bytes writes[] = {{a.table, ((requests - 1) * a.table_stride + a.table_pages) * word},
                                {a.slots, rows * sizeof(long long)},
                                {a.cu_q, (requests + 1) * word},
                                {a.lengths, requests * word},
                                {a.flat, requests * a.table_pages * word},
                                {a.k_start, rows * word},
                                {a.k_end, rows * word},
                                {a.pages_needed, word}};
        for (const Bytes& written : writes)
            for (const Bytes& read : reads)
                ITK_REQUIRE(!overlap(written, read), "the request lengths and the free list must not share memory with the table or the plan");
        for (const Bytes& written : writes)
            for (const Bytes* other = writes; other != &written; ++other)
                ITK_REQUIRE(!overlap(written, *other), "the table and the plan's buffers must not share memory with one another");
    }
    DeviceState device;
    const int rc = current_device(&device);
    if (rc != ITK_OK) return rc;
    const long long work = std::max(static_cast<long long>(a.requests) * a.table_pages, static_cast<long long>(a.rows));
    const int grid = static_cast<int>(std::min<long long>(2 * device.sm_count, (work + 2 * kPlanThreads - 1) / (2 * kPlanThreads)));
    const int wide = aligned16(a.slots) && aligned16(a.k_start) && aligned16(a.k_end);
    const size_t smem = (3 * static_cast<size_t>(a.requests) + 1) * sizeof(int);
    itk_plan_pages_kernel<<<grid, kPlanThreads, smem, stream>>>(a, wide, device.status);
    return launched("itk_plan_pages_kernel");
}

int itk_append_tokens(const itk_append_args* args, itk_stream_t stream) {
    ITK_REQUIRE(args != nullptr, "args must not be null");
    const itk_append_args& a = *args;
    ITK_REQUIRE(a.tokens >= 0 && a.kv_heads > 0, "need tokens >= 0 and kv_heads > 0");
    ITK_REQUIRE(a.dim == 64 || a.dim == 128, "head dimension must be 64 or 128");
    ITK_REQUIRE(pool_rows_ok(a.pages, a.page_size), "need 0 < pages * page_size < 2^31");
    if (a.tokens == 0) return ITK_OK;
    ITK_REQUIRE(a.slots && a.k && a.v && a.k_pool && a.v_pool, "append pointers must not be null");
    ITK_REQUIRE(aligned16(a.k) && aligned16(a.v) && aligned16(a.k_pool) && aligned16(a.v_pool),
                "keys, values and their pools must be 16-byte aligned");
    ITK_REQUIRE(strides_ok({a.k_token_stride, a.k_head_stride, a.v_token_stride, a.v_head_stride, a.k_page_stride, a.k_row_stride,
                            a.k_pool_head_stride, a.v_page_stride, a.v_row_stride, a.v_pool_head_stride}),
                "strides must be multiples of 8 elements");
    if (a.index_source != nullptr) {
        ITK_REQUIRE(a.index_pool && a.index_scales, "index keys need an index pool and its scales");
        ITK_REQUIRE(a.index_dtype == ITK_SOURCE_F32 || a.index_dtype == ITK_SOURCE_BF16,
                    "index_dtype must be ITK_SOURCE_F32 or ITK_SOURCE_BF16");
        ITK_REQUIRE(aligned16(a.index_source) && aligned16(a.index_pool) && a.index_stride >= 0 && a.index_stride % 8 == 0,
                    "index keys and their pool must be 16-byte aligned");
    }
    DeviceState device;
    const int rc = current_device(&device);
    if (rc != ITK_OK) return rc;
    constexpr unsigned kTokensPerBlock = kAppendThreads / 32;
    const unsigned grid = (static_cast<unsigned>(a.tokens) + kTokensPerBlock - 1) / kTokensPerBlock;
    if (a.index_source != nullptr && a.index_dtype == ITK_SOURCE_BF16)
        itk_append_tokens_kernel<__nv_bfloat16><<<grid, kAppendThreads, 0, stream>>>(a, device.status);
    else
        itk_append_tokens_kernel<float><<<grid, kAppendThreads, 0, stream>>>(a, device.status);
    return launched("itk_append_tokens_kernel");
}

int itk_attention_workspace_bytes(const itk_attention_args* args, size_t* bytes) {
    ITK_REQUIRE(args != nullptr && bytes != nullptr, "args and bytes must not be null");
    const int rc = check_attention(*args);
    if (rc != ITK_OK) return rc;
    AttnWorkspace ignored;
    return attention_workspace(*args, &ignored, bytes);
}

int itk_attention(const itk_attention_args* args, itk_stream_t stream) {
    ITK_REQUIRE(args != nullptr, "args must not be null");
    const itk_attention_args& a = *args;
    int rc = check_attention(a);
    if (rc != ITK_OK) return rc;
    if (a.tokens == 0) return ITK_OK;
    ITK_REQUIRE(a.requests > 0, "need at least one request");
    ITK_REQUIRE(a.q && a.out && a.cu_q, "q, out and cu_q must not be null");
    ITK_REQUIRE((a.cu_k != nullptr) != (a.lens_k != nullptr), "own keys need either cu_k (packed) or lens_k (paged)");
    ITK_REQUIRE((a.lens_k != nullptr) == (a.table != nullptr), "paged own keys need a block table, packed ones have none");
    ITK_REQUIRE(aligned16(a.q) && aligned16(a.out), "q and out must be 16-byte aligned");
    ITK_REQUIRE(strides_ok({a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride}),
                "strides must be multiples of 8 elements");
    // packed batches may have no own key at all (every key is in the prefix): then there is nothing to point at
    if (a.k == nullptr)
        ITK_REQUIRE(a.cu_k != nullptr && a.own.page_size == 0, "own keys: keys and values must not be null");
    else if ((rc = check_segment(a.own, a.k, a.v, a.table, "own keys")) != ITK_OK)
        return rc;
    if (a.k_prefix != nullptr) {
        if ((rc = check_segment(a.prefix, a.k_prefix, a.v_prefix, a.prefix_table, "prefix keys")) != ITK_OK) return rc;
        const long long room = a.prefix_table != nullptr ? static_cast<long long>(a.prefix.table_pages) * a.prefix.page_size : a.prefix.page_size;
        ITK_REQUIRE(a.prefix_keys <= room, "prefix_keys exceeds the prefix");
        ITK_REQUIRE(a.prefix_keys <= ITK_MAX_ATTENTION_KEYS, "need at most %d prefix keys", ITK_MAX_ATTENTION_KEYS);
    } else {
        ITK_REQUIRE(a.prefix_keys == 0, "prefix keys: keys and values must not be null");
    }
    ITK_REQUIRE(a.scale > 0.0f && a.scale * kLog2e <= 3.0e38f, "scale must be positive and finite");
    DeviceState device;
    if ((rc = current_device(&device)) != ITK_OK) return rc;
    AttnParams params;
    size_t needed = 0;
    if ((rc = attention_workspace(a, &params.w, &needed)) != ITK_OK) return rc;
    ITK_REQUIRE(a.workspace != nullptr && (reinterpret_cast<uintptr_t>(a.workspace) & 255u) == 0 && a.workspace_bytes >= needed,
                "the workspace must be 256-byte aligned and hold %zu bytes", needed);
    params.a = a;
    params.status = device.status;
    params.group = a.heads / a.kv_heads;
    params.tile_tokens = attention_tile_tokens(a);
    params.sm_count = std::min(device.sm_count, kAttnMaxSms);
    params.withhold_loads = a.withhold_loads;
    const long long entries = params.w.max_entries + (a.prefix_keys > 0 ? a.tokens / (2 * params.tile_tokens) + 1 : 0);
    params.small_plan = entries <= kAttnSmallEntries && entries * a.kv_heads <= params.sm_count && a.requests <= kAttnSmallEntries;
    params.inverse_sms = 1.0f / static_cast<float>(params.sm_count);
    params.out_sectors = (reinterpret_cast<uintptr_t>(a.out) & 31u) == 0 && a.out_token_stride % 16 == 0 && a.out_head_stride % 16 == 0;
    params.scale_log2 = a.scale * kLog2e;
    params.lazy = kAttnLazy / params.scale_log2;
    params.wait_polls = static_cast<uint32_t>(std::min(std::max((a.wait_limit_ns != 0 ? a.wait_limit_ns : kWaitLimitNs) / 1000, 1ull), 1ull << 31));
    {
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.heads), static_cast<cuuint64_t>(a.tokens)};
        const cuuint64_t strides[2] = {map_stride(a.q_head_stride, a.heads), map_stride(a.q_token_stride, a.tokens)};
        cuuint32_t box[3] = {64, static_cast<cuuint32_t>(params.group), static_cast<cuuint32_t>(std::min(params.tile_tokens, a.tokens))};
        const int token_bytes = a.dim * 2 * params.group;
        if ((rc = encode_map(&params.map_q, a.element, 3, a.q, dims, strides, box)) != ITK_OK) return rc;
        params.q_bytes = token_bytes * static_cast<int>(box[2]);
        params.map_q_one = params.map_q;
        params.q_bytes_one = params.q_bytes;
        if (!params.small_plan && box[2] > 1) {       // (a small call is too short for power to matter)
            box[2] = 1;
            if ((rc = encode_map(&params.map_q_one, a.element, 3, a.q, dims, strides, box)) != ITK_OK) return rc;
            params.q_bytes_one = token_bytes;
        }
    }
    if (a.k != nullptr) {
        const itk_kv_segment& s = a.own;
        if ((rc = segment_map(&params.map_k, a, s, a.k, s.k_page_stride, s.k_row_stride, s.k_head_stride)) != ITK_OK) return rc;
        if ((rc = segment_map(&params.map_v, a, s, a.v, s.v_page_stride, s.v_row_stride, s.v_head_stride)) != ITK_OK) return rc;
    } else {        // no own key: no item loads through these
        params.map_k = params.map_v = params.map_q;
    }
    if (a.prefix_keys > 0) {
        const itk_kv_segment& s = a.prefix;
        if ((rc = segment_map(&params.map_k_prefix, a, s, a.k_prefix, s.k_page_stride, s.k_row_stride, s.k_head_stride)) != ITK_OK) return rc;
        if ((rc = segment_map(&params.map_v_prefix, a, s, a.v_prefix, s.v_page_stride, s.v_row_stride, s.v_head_stride)) != ITK_OK) return rc;
    } else {
        params.map_k_prefix = params.map_k;
        params.map_v_prefix = params.map_v;
    }
    if (a.element == ITK_ELEMENT_BF16)
        return a.dim == 128 ? launch_attention<__nv_bfloat16, 128>(params, stream) : launch_attention<__nv_bfloat16, 64>(params, stream);
    return a.dim == 128 ? launch_attention<__half, 128>(params, stream) : launch_attention<__half, 64>(params, stream);
}

}  // extern "C"
