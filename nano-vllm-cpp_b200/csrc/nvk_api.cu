// extern "C" entry points declared in include/nvk.h: argument validation (the checks the
// reference performs in src/kernels/kvcache.cu:146-190, src/kernels/attention.cu:679-681 and
// src/kernels/kernel_types.cu:24-110) and dispatch to the kernels of this library.
#include "nvk_internal.cuh"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

namespace nvk {

namespace {
thread_local std::string g_last_error;
}

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

int check_launch(const char* what) {
    const cudaError_t e = cudaPeekAtLastError();
    if (e == cudaSuccess) return NVK_OK;
    return fail(NVK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

namespace {

bool is_compute_dtype(int dtype) { return dtype == NVK_F16 || dtype == NVK_BF16 || dtype == NVK_F32; }
bool is_index_dtype(int dtype) { return dtype == NVK_I32 || dtype == NVK_I64; }
IndexArray index_array(const void* p, int dtype) { return IndexArray(p, dtype == NVK_I64 ? 1 : 0); }

// What the calls over a 4-bit cache have in common: its types and its shape.
int check_int4(const char* what, int dtype, int num_kv_heads, int head_dim) {
    if (dtype != NVK_F16 && dtype != NVK_BF16) return fail(NVK_ERR_UNSUPPORTED, "%s: needs F16 or BF16", what);
    if (num_kv_heads <= 0 || head_dim <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: sizes must be positive", what);
    if (head_dim != 128) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", what, head_dim);
    return NVK_OK;
}
int check_decode_sizes(int64_t batch, int64_t max_blocks, int64_t num_cache_blocks, int num_heads, int num_kv_heads, int head_dim, int block_size) {
    if (batch < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "attention dimensions must be positive");
    if (num_heads % num_kv_heads != 0) return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    return NVK_OK;
}
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
    return x < y + b_bytes && y < x + a_bytes;
}
// Two arrays of `rows` x `heads` x `keys` weights that are neither the same nor apart.
bool weights_overlap(const float* old_weights, const float* new_weights, int64_t rows, int heads, int64_t keys) {
    const int64_t bytes = rows * heads * keys * static_cast<int64_t>(sizeof(float));
    return old_weights != nullptr && old_weights != new_weights && overlap(old_weights, bytes, new_weights, bytes);
}
int64_t index_bytes(int dtype) { return dtype == NVK_I64 ? 8 : 4; }
// What the calls over a cache with block scales have in common.
int check_blocks8(const char* what, int dtype, int cache_dtype, int num_kv_heads, int head_dim) {
    if (cache_dtype != NVK_I8 && cache_dtype != NVK_E4M3) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: cache elements are int8 or e4m3", what);
    return check_int4(what, dtype, num_kv_heads, head_dim);
}
constexpr int64_t kMostBytes = 1LL << 60;   // of a tensor: sizes are held below it before they are multiplied
// Neither the same nor apart.
bool partly(const void* a, const void* b, int64_t bytes) { return a != b && overlap(a, bytes, b, bytes); }
// Memory that a call writes, or only reads.
struct Range { const void* at; int64_t bytes; };
// Whether something that is written overlaps with anything else.
bool written_twice(std::initializer_list<Range> written, std::initializer_list<Range> read) {
    for (const Range* a = written.begin(); a != written.end(); ++a) {
        if (a->at == nullptr || a->bytes <= 0) continue;
        auto hits = [&](const Range& b) { return b.at != nullptr && b.bytes > 0 && overlap(a->at, a->bytes, b.at, b.bytes); };
        for (const Range* b = a + 1; b != written.end(); ++b)
            if (hits(*b)) return true;
        for (const Range& b : read)
            if (hits(b)) return true;
    }
    return false;
}
// `rows` rows of `row` bytes, `stride` bytes from each to the next.  Whether two such share a byte: told apart by their ends, and with one stride by the columns that they take.
struct Rows { const void* at; int64_t stride, row, rows; };
bool rows_overlap(const Rows& a, const Rows& b) {
    if (a.at == nullptr || b.at == nullptr) return false;
    if (!overlap(a.at, (a.rows - 1) * a.stride + a.row, b.at, (b.rows - 1) * b.stride + b.row)) return false;
    if (a.stride != b.stride) return true;
    const int64_t apart = static_cast<const char*>(b.at) - static_cast<const char*>(a.at), column = (apart % a.stride + a.stride) % a.stride;   // where b's columns begin after a's
    return column < a.row || column + b.row > a.stride;
}
// What the calls over the tables of requests have in common.
int check_requests(const char* what, const void* lens, const void* blocks, const void* free_blocks, const void* count, const void* new_lens, const void* new_count,
                   int64_t batch, int64_t rows, int64_t row_blocks, int64_t num_free, int block_size, const void* request_rows, int index_dtype) {
    if (!lens || !blocks || !free_blocks || !count || !new_lens || !new_count) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: lengths, blocks and counts must be defined", what);
    if (!is_index_dtype(index_dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: index tensors must be int32 or int64", what);
    if (batch < 0 || rows <= 0 || row_blocks <= 0 || num_free <= 0 || block_size <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: sizes must be positive", what);
    if (rows > (1LL << 40) / row_blocks || num_free > (1LL << 40)) return fail(NVK_ERR_UNSUPPORTED, "%s: too many requests or blocks", what);
    if (!request_rows && rows < batch) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: without request_rows there has to be a row for every request", what);
    const int64_t wide = index_bytes(index_dtype);
    for (const void* p : {lens, blocks, free_blocks, count, new_lens, new_count, request_rows})
        if (!aligned_to(p, static_cast<size_t>(wide))) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: misaligned tensor", what);
    if (partly(lens, new_lens, rows * wide) || partly(count, new_count, wide))
        return fail(NVK_ERR_INVALID_ARGUMENT, "%s: new lengths and count are the old ones' memory or do not overlap with it", what);
    return NVK_OK;
}

int launch_prefill(const PrefillArgs& a) {
    if (prefill_tc_supported(a) && !prefill_takes_tiles(a)) return launch_prefill_tc(a);
    if (prefill_mma_supported(a)) return launch_prefill_mma(a);
    return launch_rowwise_prefill(a);
}

}  // namespace
}  // namespace nvk

using namespace nvk;

extern "C" {

int nvk_abi_version(void) { return 2; }

const char* nvk_last_error(void) { return g_last_error.c_str(); }

int nvk_store_kvcache(const void* key, const void* value, void* k_cache, void* v_cache,
                      const void* slot_mapping, int slot_dtype, int64_t num_tokens, int64_t row_elems,
                      int64_t cache_rows, int dtype, void* stream) {
    if (!key || !value || !k_cache || !v_cache || !slot_mapping)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache: key, value, k_cache, v_cache and slot_mapping must be defined");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "key must be float16, bfloat16, or float32");
    if (slot_dtype != NVK_I32 && slot_dtype != NVK_I64)
        return fail(NVK_ERR_INVALID_ARGUMENT, "slot_mapping must be int32 or int64");
    if (num_tokens <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "slot_mapping must contain at least one element");
    if (row_elems <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "key cannot be flattened by the provided leading count");
    if (cache_rows <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "k_cache does not contain an integer number of cache rows");
    return launch_store_kvcache(key, value, k_cache, v_cache, slot_mapping, slot_dtype == NVK_I64, num_tokens,
                                row_elems * static_cast<int64_t>(dtype_size(dtype)), cache_rows,
                                static_cast<cudaStream_t>(stream));
}

int nvk_fused_split_norm_rope_store(const void* qkv, const int32_t* positions, const void* q_norm_weight,
                                    const void* k_norm_weight, float norm_eps, const float* cos_sin_cache,
                                    int64_t max_positions, const int32_t* slot_mapping, void* k_cache,
                                    void* v_cache, int64_t cache_rows, int64_t rows, int num_q_heads,
                                    int num_kv_heads, int head_dim, void* q_out, int dtype, void* stream) {
    if (dtype != NVK_F16 && dtype != NVK_BF16)
        return fail(NVK_ERR_INVALID_ARGUMENT, "fused_split_norm_rope_store only supports bf16/fp16");
    if (!qkv || !positions || !cos_sin_cache || !k_cache || !v_cache || !q_out)
        return fail(NVK_ERR_INVALID_ARGUMENT, "fused_split_norm_rope_store: all tensors must be defined");
    if ((q_norm_weight == nullptr) != (k_norm_weight == nullptr))
        return fail(NVK_ERR_INVALID_ARGUMENT, "fused_split_norm_rope_store: q_norm_weight and k_norm_weight go together");
    if (rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || max_positions <= 0 || cache_rows <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "fused_split_norm_rope_store: sizes must be positive");
    if (rows == 0) return NVK_OK;
    if (!aligned_to(qkv, 16) || !aligned_to(q_out, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) ||
        !aligned_to(q_norm_weight, 16) || !aligned_to(k_norm_weight, 16) || !aligned_to(cos_sin_cache, 16))
        return fail(NVK_ERR_UNSUPPORTED, "fused_split_norm_rope_store: tensors must be 16-byte aligned");
    return launch_fused_prologue(qkv, positions, q_norm_weight, k_norm_weight, norm_eps, cos_sin_cache,
                                 max_positions, slot_mapping, k_cache, v_cache, cache_rows, rows, num_q_heads,
                                 num_kv_heads, head_dim, q_out, dtype, static_cast<cudaStream_t>(stream));
}

size_t nvk_decode_attention_workspace_bytes(int64_t batch, int num_heads, int num_kv_heads, int head_dim,
                                            int64_t max_blocks, int block_size) {
    return decode_mma_workspace_bytes(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
}

int nvk_decode_attention_paged(const void* query, const void* k_cache, const void* v_cache,
                               const void* context_lens, int context_lens_dtype, const void* block_tables,
                               int block_tables_dtype, int64_t batch, int64_t max_blocks, int64_t num_cache_blocks,
                               int num_heads, int num_kv_heads, int head_dim, int block_size, float scale,
                               void* output, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !context_lens || !block_tables || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention requires KV cache, context_lens, and block_tables");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens and block_tables must be int32 or int64");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "unsupported dtype for decode_attention_paged");
    if (batch < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        head_dim <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "attention dimensions must be positive");
    if (num_heads % num_kv_heads != 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    if (batch == 0) return NVK_OK;
    DecodeArgs a{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype),
                 index_array(block_tables, block_tables_dtype), output, batch, max_blocks, num_cache_blocks,
                 num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                 static_cast<cudaStream_t>(stream)};
    if (decode_mma_supported(a)) {
        if (workspace != nullptr) {
            const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
            if (workspace_bytes < need)
                return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention: workspace of %zu bytes given, %zu needed",
                            workspace_bytes, need);
            if (!aligned_to(workspace, 16))
                return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention: workspace must be 16-byte aligned");
        }
        return launch_decode_mma(a);
    }
    if (decode_simt_supported(a)) return launch_decode_simt(a);
    return launch_rowwise_decode(a);
}

int nvk_store_kvcache_int8(const void* key, const void* value, void* k_cache, void* v_cache, void* k_scale,
                           void* v_scale, const int32_t* slot_mapping, int64_t num_tokens, int num_kv_heads,
                           int head_dim, int64_t cache_rows, int dtype, void* stream) {
    if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int8: every tensor must be defined");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "unsupported input dtype for store_kvcache_int8");
    if (num_kv_heads <= 0 || head_dim <= 0 || cache_rows <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int8: dimensions must be positive");
    if (num_tokens <= 0) return NVK_OK;   // the reference returns without a launch (kvcache.cu:327)
    if (!aligned_to(key, dtype == NVK_F32 ? 4 : 16) || !aligned_to(value, dtype == NVK_F32 ? 4 : 16) ||
        !aligned_to(k_cache, 8) || !aligned_to(v_cache, 8) || !aligned_to(k_scale, 2) || !aligned_to(v_scale, 2))
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int8: misaligned tensor");
    return launch_store_int8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, num_tokens, num_kv_heads,
                             head_dim, cache_rows, dtype, static_cast<cudaStream_t>(stream));
}

int nvk_decode_attention_paged_int8(const void* query, const void* k_cache, const void* v_cache, const void* k_scale,
                                    const void* v_scale, const void* context_lens, int context_lens_dtype,
                                    const void* block_tables, int block_tables_dtype, int64_t batch, int64_t max_blocks,
                                    int64_t num_cache_blocks, int num_heads, int num_kv_heads, int head_dim,
                                    int block_size, float scale, void* output, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !k_scale || !v_scale || !context_lens || !block_tables || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int8) requires KV cache, scales, context_lens, and block_tables");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens and block_tables must be int32 or int64");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "unsupported query dtype for decode_attention_paged_int8");
    if (batch < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        head_dim <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "attention dimensions must be positive");
    if (num_heads % num_kv_heads != 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    if (batch == 0) return NVK_OK;
    DecodeInt8Args a{{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype),
                      index_array(block_tables, block_tables_dtype), output, batch, max_blocks, num_cache_blocks,
                      num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                      static_cast<cudaStream_t>(stream)},
                     k_scale, v_scale};
    if (decode_int8_mma_supported(a)) {
        if (workspace != nullptr) {
            const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
            if (workspace_bytes < need)
                return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int8): workspace of %zu bytes given, %zu needed",
                            workspace_bytes, need);
            if (!aligned_to(workspace, 16))
                return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int8): workspace must be 16-byte aligned");
        }
        return launch_decode_int8_mma(a);
    }
    return launch_rowwise_decode_int8(a);
}

int nvk_store_kvcache_fp8(const void* key, const void* value, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                          const int32_t* slot_mapping, int64_t num_tokens, int num_kv_heads, int head_dim, int64_t cache_rows,
                          int dtype, void* stream) {
    if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !slot_mapping)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_fp8 requires key, value, caches, scales and slot_mapping");
    if (dtype != NVK_F16 && dtype != NVK_BF16) return fail(NVK_ERR_UNSUPPORTED, "store_kvcache_fp8: key / value must be F16 or BF16");
    if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || cache_rows <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_fp8: sizes must be positive");
    if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_cache, 8) || !aligned_to(v_cache, 8))
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_fp8: key / value must be 16-byte aligned, the caches 8-byte aligned");
    if (num_tokens == 0) return NVK_OK;
    return launch_store_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping, num_tokens, num_kv_heads, head_dim,
                            cache_rows, dtype, static_cast<cudaStream_t>(stream));
}

int nvk_decode_attention_paged_fp8(const void* query, const void* k_cache, const void* v_cache, const void* k_scale,
                                   const void* v_scale, const void* context_lens, int context_lens_dtype,
                                   const void* block_tables, int block_tables_dtype, int64_t batch, int64_t max_blocks,
                                   int64_t num_cache_blocks, int num_heads, int num_kv_heads, int head_dim,
                                   int block_size, float scale, void* output, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !k_scale || !v_scale || !context_lens || !block_tables || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (fp8) requires KV cache, scales, context_lens, and block_tables");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens and block_tables must be int32 or int64");
    if (batch < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || num_heads <= 0 || num_kv_heads <= 0 ||
        head_dim <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "attention dimensions must be positive");
    if (num_heads % num_kv_heads != 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    if (batch == 0) return NVK_OK;
    DecodeInt8Args a{{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype),
                      index_array(block_tables, block_tables_dtype), output, batch, max_blocks, num_cache_blocks,
                      num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                      static_cast<cudaStream_t>(stream)},
                     k_scale, v_scale, true};
    if (!decode_int8_mma_supported(a))
        return fail(NVK_ERR_UNSUPPORTED, "decode attention (fp8): F16 / BF16 queries, head_dim 128, at most 8 query heads per KV head, "
                                         "block_size a multiple of 16");
    if (workspace != nullptr) {
        const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
        if (workspace_bytes < need)
            return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (fp8): workspace of %zu bytes given, %zu needed", workspace_bytes, need);
        if (!aligned_to(workspace, 16)) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (fp8): workspace must be 16-byte aligned");
    }
    return launch_decode_int8_mma(a);
}

int nvk_store_kvcache_int4(const void* key, const void* value, void* k_cache, void* v_cache, void* k_params, void* v_params,
                           const void* slot_mapping, int slot_dtype, int64_t num_tokens, int num_kv_heads, int head_dim, int64_t cache_rows,
                           int dtype, void* stream) {
    if (!key || !value || !k_cache || !v_cache || !k_params || !v_params || !slot_mapping)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int4: every tensor must be defined");
    if (const int rc = check_int4("store_kvcache_int4", dtype, num_kv_heads, head_dim); rc != NVK_OK) return rc;
    if (!is_index_dtype(slot_dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "slot_mapping must be int32 or int64");
    if (num_tokens < 0 || cache_rows <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int4: sizes must be positive");
    if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) || !aligned_to(k_params, 4) ||
        !aligned_to(v_params, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int4: key, value and the caches must be 16-byte aligned, the params 4-byte aligned");
    if (num_tokens == 0) return NVK_OK;
    return launch_store_int4(key, value, k_cache, v_cache, k_params, v_params, index_array(slot_mapping, slot_dtype), num_tokens, num_kv_heads, cache_rows,
                             dtype, static_cast<cudaStream_t>(stream));
}

int nvk_gather_kvcache_int4(const void* k_cache, const void* v_cache, const void* k_params, const void* v_params, const void* cu_seqlens_k,
                            int cu_seqlens_k_dtype, const void* block_tables, int block_tables_dtype, int64_t num_seqs, int64_t total_k,
                            int64_t max_blocks, int64_t num_cache_blocks, int num_kv_heads, int head_dim, int block_size, void* key, void* value,
                            int dtype, void* stream) {
    if (!k_cache || !v_cache || !k_params || !v_params || !cu_seqlens_k || !block_tables || !key || !value)
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_int4: every tensor must be defined");
    if (const int rc = check_int4("gather_kvcache_int4", dtype, num_kv_heads, head_dim); rc != NVK_OK) return rc;
    if (!is_index_dtype(cu_seqlens_k_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "cu_seqlens_k and block_tables must be int32 or int64");
    if (num_seqs <= 0 || total_k < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_int4: sizes must be positive");
    if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) || !aligned_to(k_params, 4) ||
        !aligned_to(v_params, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_int4: key, value and the caches must be 16-byte aligned, the params 4-byte aligned");
    if (total_k == 0) return NVK_OK;
    return launch_gather_int4(k_cache, v_cache, k_params, v_params, index_array(cu_seqlens_k, cu_seqlens_k_dtype), index_array(block_tables, block_tables_dtype),
                              num_seqs, total_k, max_blocks, num_cache_blocks, num_kv_heads, block_size, key, value, dtype, static_cast<cudaStream_t>(stream));
}

int nvk_decode_attention_paged_int4(const void* query, const void* k_cache, const void* v_cache, const void* k_params, const void* v_params,
                                    const void* context_lens, int context_lens_dtype, const void* block_tables, int block_tables_dtype,
                                    int64_t batch, int64_t max_blocks, int64_t num_cache_blocks, int num_heads, int num_kv_heads,
                                    int head_dim, int block_size, float scale, void* output, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !k_params || !v_params || !context_lens || !block_tables || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int4) requires KV cache, params, context_lens, and block_tables");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens and block_tables must be int32 or int64");
    if (const int rc = check_decode_sizes(batch, max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size); rc != NVK_OK) return rc;
    if (batch == 0) return NVK_OK;
    const DecodeArgs a{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype), index_array(block_tables, block_tables_dtype), output, batch,
                       max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream)};
    if (!decode_int4_supported(a, k_params, v_params))
        return fail(NVK_ERR_UNSUPPORTED, "decode attention (int4): F16 / BF16 queries, head_dim 128, at most 8 query heads per KV head, block_size a multiple "
                                         "of 16; query and caches 16-byte aligned, params 4-byte and output 8-byte aligned");
    if (workspace != nullptr) {
        const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
        if (workspace_bytes < need)
            return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int4): workspace of %zu bytes given, %zu needed", workspace_bytes, need);
        if (!aligned_to(workspace, 16)) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (int4): workspace must be 16-byte aligned");
    }
    return launch_decode_int4(a, k_params, v_params);
}

int nvk_store_kvcache_blocks8(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride, void* k_cache, void* v_cache,
                              float* k_scale, float* v_scale, int cache_dtype, const void* cu_seqlens_q, int cu_seqlens_q_dtype,
                              const void* context_lens, int context_lens_dtype, const void* block_tables, int block_tables_dtype, int64_t num_seqs,
                              int64_t total_q, int64_t max_blocks, int64_t num_cache_blocks, int num_kv_heads, int head_dim, int block_size, int dtype,
                              void* stream) {
    if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !context_lens || !block_tables)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: key, value, caches, scales, context_lens and block_tables must be defined");
    if (const int rc = check_blocks8("store_kvcache_blocks8", dtype, cache_dtype, num_kv_heads, head_dim); rc != NVK_OK) return rc;
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype) || (cu_seqlens_q && !is_index_dtype(cu_seqlens_q_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "cu_seqlens_q, context_lens and block_tables must be int32 or int64");
    if (num_seqs < 0 || total_q < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: sizes must be positive");
    if (!cu_seqlens_q && total_q != num_seqs)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: without cu_seqlens_q there has to be one row for every sequence");
    const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
    if (key_row_stride < row || value_row_stride < row || key_row_stride % 8 != 0 || value_row_stride % 8 != 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: row strides must be multiples of 8 elements, and no less than a row");
    if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) || !aligned_to(k_scale, 4) || !aligned_to(v_scale, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: key, value and the caches must be 16-byte aligned, the scales 4-byte aligned");
    if (num_seqs > (1LL << 30) / num_kv_heads || total_q >= (1LL << 31) - block_size || max_blocks > ((1LL << 31) - 1) / block_size || num_kv_heads > (1 << 24))
        return fail(NVK_ERR_UNSUPPORTED, "store_kvcache_blocks8: too many sequences, tokens, heads or blocks");
    if (num_seqs == 0 || total_q == 0) return NVK_OK;
    if (num_cache_blocks > kMostBytes / row / block_size || num_seqs > kMostBytes / 8 / max_blocks || key_row_stride > kMostBytes / 2 / total_q || value_row_stride > kMostBytes / 2 / total_q)
        return fail(NVK_ERR_UNSUPPORTED, "store_kvcache_blocks8: too many cache blocks or table entries, or rows too far apart");
    const int64_t cache = num_cache_blocks * block_size * row, scales = num_cache_blocks * num_kv_heads * 4;
    if (written_twice({{k_cache, cache}, {v_cache, cache}, {k_scale, scales}, {v_scale, scales}},
                      {{key, ((total_q - 1) * key_row_stride + row) * 2}, {value, ((total_q - 1) * value_row_stride + row) * 2},
                       {cu_seqlens_q, (num_seqs + 1) * index_bytes(cu_seqlens_q_dtype)}, {context_lens, num_seqs * index_bytes(context_lens_dtype)},
                       {block_tables, num_seqs * max_blocks * index_bytes(block_tables_dtype)}}))
        return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_blocks8: a cache or its scales overlap with another tensor");
    return launch_store_blocks8(Blocks8StoreArgs{key, value, k_cache, v_cache, k_scale, v_scale, index_array(cu_seqlens_q, cu_seqlens_q_dtype),
                                                 index_array(context_lens, context_lens_dtype), index_array(block_tables, block_tables_dtype), num_seqs, total_q,
                                                 max_blocks, num_cache_blocks, key_row_stride, value_row_stride, num_kv_heads, block_size,
                                                 cache_dtype == NVK_E4M3, dtype, static_cast<cudaStream_t>(stream)});
}

int nvk_gather_kvcache_blocks8(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, int cache_dtype,
                               const void* cu_seqlens_k, int cu_seqlens_k_dtype, const void* block_tables, int block_tables_dtype, int64_t num_seqs,
                               int64_t total_k, int64_t max_blocks, int64_t num_cache_blocks, int num_kv_heads, int head_dim, int block_size, void* key,
                               void* value, int dtype, void* stream) {
    if (!k_cache || !v_cache || !k_scale || !v_scale || !cu_seqlens_k || !block_tables || !key || !value)
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_blocks8: every tensor must be defined");
    if (const int rc = check_blocks8("gather_kvcache_blocks8", dtype, cache_dtype, num_kv_heads, head_dim); rc != NVK_OK) return rc;
    if (!is_index_dtype(cu_seqlens_k_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "cu_seqlens_k and block_tables must be int32 or int64");
    if (num_seqs <= 0 || total_k < 0 || max_blocks <= 0 || num_cache_blocks <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_blocks8: sizes must be positive");
    if (!aligned_to(key, 16) || !aligned_to(value, 16) || !aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) || !aligned_to(k_scale, 4) || !aligned_to(v_scale, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_blocks8: key, value and the caches must be 16-byte aligned, the scales 4-byte aligned");
    if (max_blocks > ((1LL << 31) - 1) / block_size) return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_blocks8: too many blocks");
    const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
    if (total_k == 0) return NVK_OK;
    if (total_k > (1LL << 38) || total_k > kMostBytes / 2 / row) return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_blocks8: too many rows");
    if (num_cache_blocks > kMostBytes / row / block_size || num_seqs > kMostBytes / 8 / max_blocks)
        return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_blocks8: too many cache blocks or table entries");
    const int64_t cache = num_cache_blocks * block_size * row, scales = num_cache_blocks * num_kv_heads * 4;
    if (written_twice({{key, total_k * row * 2}, {value, total_k * row * 2}},
                      {{k_cache, cache}, {v_cache, cache}, {k_scale, scales}, {v_scale, scales}, {cu_seqlens_k, (num_seqs + 1) * index_bytes(cu_seqlens_k_dtype)},
                       {block_tables, num_seqs * max_blocks * index_bytes(block_tables_dtype)}}))
        return fail(NVK_ERR_INVALID_ARGUMENT, "gather_kvcache_blocks8: key or value overlaps with another tensor");
    return launch_gather_blocks8(Blocks8GatherArgs{k_cache, v_cache, k_scale, v_scale, index_array(cu_seqlens_k, cu_seqlens_k_dtype),
                                                   index_array(block_tables, block_tables_dtype), num_seqs, total_k, max_blocks, num_cache_blocks, num_kv_heads,
                                                   block_size, cache_dtype == NVK_E4M3, key, value, dtype, static_cast<cudaStream_t>(stream)});
}

int nvk_decode_attention_paged_blocks8(const void* query, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                                       int cache_dtype, const void* context_lens, int context_lens_dtype, const void* block_tables,
                                       int block_tables_dtype, int64_t batch, int64_t max_blocks, int64_t num_cache_blocks, int num_heads,
                                       int num_kv_heads, int head_dim, int block_size, float scale, void* output, int dtype, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !k_scale || !v_scale || !context_lens || !block_tables || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8) requires KV cache, scales, context_lens, and block_tables");
    if (cache_dtype != NVK_I8 && cache_dtype != NVK_E4M3) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8): cache elements are int8 or e4m3");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens and block_tables must be int32 or int64");
    if (const int rc = check_decode_sizes(batch, max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size); rc != NVK_OK) return rc;
    if (!std::isfinite(scale)) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8): scale must be finite");
    if (batch == 0) return NVK_OK;
    const DecodeArgs a{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype), index_array(block_tables, block_tables_dtype), output, batch,
                       max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream)};
    if (!decode_blocks8_supported(a, k_scale, v_scale))
        return fail(NVK_ERR_UNSUPPORTED, "decode attention (blocks8): F16 / BF16 queries, head_dim 128, at most 8 query heads per KV head, block_size a multiple "
                                         "of 16; query and caches 16-byte aligned, output 8-byte and scales 4-byte aligned");
    if (workspace != nullptr) {
        const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, max_blocks, block_size);
        if (workspace_bytes < need)
            return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8): workspace of %zu bytes given, %zu needed", workspace_bytes, need);
        if (!aligned_to(workspace, 16)) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8): workspace must be 16-byte aligned");
    }
    if (batch < (1LL << 28) / num_heads) {   // (the launch refuses more; the output may be the query: a head's is written when all have read it)
        const int64_t rows = batch * num_heads * head_dim * 2, room = static_cast<int64_t>(std::min<size_t>(workspace_bytes, kMostBytes)), cache = num_cache_blocks * block_size * num_kv_heads * head_dim, scales = num_cache_blocks * num_kv_heads * 4;
        const Range lens{context_lens, batch * index_bytes(context_lens_dtype)}, tables{block_tables, batch * max_blocks * index_bytes(block_tables_dtype)};
        const Range q{query, query == output ? 0 : rows};
        if (written_twice({{output, rows}, {workspace, room}}, {q, {k_cache, cache}, {v_cache, cache}, {k_scale, scales}, {v_scale, scales}, lens, tables}) ||
            (workspace != nullptr && overlap(workspace, room, query, rows)))
            return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (blocks8): output or workspace overlaps with another tensor");
    }
    return launch_decode_blocks8(a, k_scale, v_scale, cache_dtype == NVK_E4M3);
}

int nvk_step_metadata(const void* new_lens, const void* request_rows, const void* request_lens, void* request_blocks, const void* free_blocks,
                      const void* free_count, int64_t batch, int64_t num_request_rows, int64_t request_max_blocks, int64_t num_free_blocks,
                      int64_t num_cache_blocks, int block_size, void* block_tables, int64_t max_blocks, void* context_lens, void* cu_seqlens_q,
                      void* cu_seqlens_k, void* positions, void* slot_mapping, int64_t num_tokens, void* new_request_lens, void* new_free_count,
                      int index_dtype, void* stream) {
    if (!new_lens || !block_tables || !context_lens) return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: new_lens, block_tables and context_lens must be defined");
    if (const int rc = check_requests("step_metadata", request_lens, request_blocks, free_blocks, free_count, new_request_lens, new_free_count, batch,
                                      num_request_rows, request_max_blocks, num_free_blocks, block_size, request_rows, index_dtype); rc != NVK_OK)
        return rc;
    if (batch == 0 || max_blocks <= 0 || num_cache_blocks <= 0 || num_tokens < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: sizes must be positive");
    if (num_tokens > 0 && (!positions || !slot_mapping)) return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: positions and slot_mapping must be defined");
    for (const void* p : {new_lens, static_cast<const void*>(block_tables), static_cast<const void*>(context_lens), static_cast<const void*>(cu_seqlens_q),
                          static_cast<const void*>(cu_seqlens_k), static_cast<const void*>(positions), static_cast<const void*>(slot_mapping)})
        if (!aligned_to(p, static_cast<size_t>(index_bytes(index_dtype)))) return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: misaligned tensor");
    if (index_dtype == NVK_I32 && num_cache_blocks > ((1LL << 31) - 1) / block_size)
        return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: slots of that many blocks need int64");
    if (batch > (1LL << 40) / max_blocks || num_tokens > (1LL << 40) || num_cache_blocks > (1LL << 40)) return fail(NVK_ERR_UNSUPPORTED, "step_metadata: too many requests or table entries");
    {
        const int64_t w = index_bytes(index_dtype);
        const Range lens{request_lens == new_request_lens ? nullptr : request_lens, num_request_rows * w}, count{free_count == new_free_count ? nullptr : free_count, w};
        if (written_twice({{request_blocks, num_request_rows * request_max_blocks * w}, {block_tables, batch * max_blocks * w}, {context_lens, batch * w},
                           {cu_seqlens_q, (batch + 1) * w}, {cu_seqlens_k, (batch + 1) * w}, {positions, num_tokens * w}, {slot_mapping, num_tokens * w},
                           {new_request_lens, num_request_rows * w}, {new_free_count, w}},
                          {{new_lens, batch * w}, {request_rows, batch * w}, {free_blocks, num_free_blocks * w}, lens, count}))
            return fail(NVK_ERR_INVALID_ARGUMENT, "step_metadata: an output overlaps with another tensor (lengths and count may be updated in place)");
    }
    StepArgs a{};
    auto index = [&](const void* p) { return index_array(p, index_dtype); };
    a.new_lens = index(new_lens); a.rows = index(request_rows); a.lens = index(request_lens); a.free_count = index(free_count);
    a.request_blocks = request_blocks; a.free_blocks = const_cast<void*>(free_blocks);
    a.block_tables = block_tables; a.context_lens = context_lens; a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k;
    a.positions = positions; a.slots = slot_mapping; a.new_request_lens = new_request_lens; a.new_free_count = new_free_count;
    a.batch = batch; a.num_rows = num_request_rows; a.row_blocks = request_max_blocks; a.num_free = num_free_blocks;
    a.num_cache_blocks = num_cache_blocks; a.max_blocks = max_blocks; a.num_tokens = num_tokens;
    a.block_size = block_size; a.wide = index_dtype == NVK_I64 ? 1 : 0;
    a.stream = static_cast<cudaStream_t>(stream);
    return launch_step_metadata(a);
}

int nvk_release_blocks(const void* request_rows, const void* first_blocks, const void* request_lens, const void* request_blocks, void* free_blocks,
                       const void* free_count, int64_t batch, int64_t num_request_rows, int64_t request_max_blocks, int64_t num_free_blocks,
                       int block_size, void* new_request_lens, void* new_free_count, int index_dtype, void* stream) {
    if (const int rc = check_requests("release_blocks", request_lens, request_blocks, free_blocks, free_count, new_request_lens, new_free_count, batch,
                                      num_request_rows, request_max_blocks, num_free_blocks, block_size, request_rows, index_dtype); rc != NVK_OK)
        return rc;
    if (!aligned_to(first_blocks, static_cast<size_t>(index_bytes(index_dtype)))) return fail(NVK_ERR_INVALID_ARGUMENT, "release_blocks: misaligned tensor");
    {
        const int64_t w = index_bytes(index_dtype);
        const Range lens{request_lens == new_request_lens ? nullptr : request_lens, num_request_rows * w}, count{free_count == new_free_count ? nullptr : free_count, w};
        if (written_twice({{free_blocks, num_free_blocks * w}, {new_request_lens, num_request_rows * w}, {new_free_count, w}},
                          {{request_rows, batch * w}, {first_blocks, batch * w}, {request_blocks, num_request_rows * request_max_blocks * w}, lens, count}))
            return fail(NVK_ERR_INVALID_ARGUMENT, "release_blocks: an output overlaps with another tensor (lengths and count may be updated in place)");
    }
    StepArgs a{};
    auto index = [&](const void* p) { return index_array(p, index_dtype); };
    a.rows = index(request_rows); a.first_blocks = index(first_blocks); a.lens = index(request_lens); a.free_count = index(free_count);
    a.request_blocks = const_cast<void*>(request_blocks); a.free_blocks = free_blocks;
    a.new_request_lens = new_request_lens; a.new_free_count = new_free_count;
    a.batch = batch; a.num_rows = num_request_rows; a.row_blocks = request_max_blocks; a.num_free = num_free_blocks;
    a.block_size = block_size; a.wide = index_dtype == NVK_I64 ? 1 : 0;
    a.stream = static_cast<cudaStream_t>(stream);
    return launch_release_blocks(a);
}

int nvk_rotary_embedding(const void* query, const void* key, const void* positions, int positions_dtype, const float* inv_freq, float attention_factor,
                         int64_t rows, int num_q_heads, int num_kv_heads, int head_dim, int rotary_dim, int interleaved, int64_t query_row_stride,
                         int64_t key_row_stride, void* query_out, void* key_out, int64_t query_out_row_stride, int64_t key_out_row_stride, int dtype,
                         void* stream) {
    if (!query || !query_out || !positions || !inv_freq) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: query, query_out, positions and inv_freq must be defined");
    if ((key == nullptr) != (key_out == nullptr)) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: key and key_out go together");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: query must be float16, bfloat16, or float32");
    if (!is_index_dtype(positions_dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: positions must be int32 or int64");
    if (rows < 0 || num_q_heads <= 0 || (key && num_kv_heads <= 0) || head_dim <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: sizes must be positive");
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: rotary_dim must be even, positive and at most head_dim");
    if (head_dim > 1024) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: head_dim must be at most 1024 (got %d)", head_dim);
    if (num_q_heads > (1 << 19) || (key && num_kv_heads > (1 << 19))) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: too many heads");
    const int64_t size = static_cast<int64_t>(dtype_size(dtype));
    auto check = [&](const void* at, int64_t stride, int heads) -> int {
        if (stride < static_cast<int64_t>(heads) * head_dim) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: a row stride is less than a row");
        if (!aligned_to(at, static_cast<size_t>(size))) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: misaligned tensor");
        if (stride > (1LL << 40) || rows > (1LL << 56) / stride) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: too many rows");
        return NVK_OK;
    };
    if (const int rc = check(query, query_row_stride, num_q_heads); rc != NVK_OK) return rc;
    if (const int rc = check(query_out, query_out_row_stride, num_q_heads); rc != NVK_OK) return rc;
    if (key) {
        if (const int rc = check(key, key_row_stride, num_kv_heads); rc != NVK_OK) return rc;
        if (const int rc = check(key_out, key_out_row_stride, num_kv_heads); rc != NVK_OK) return rc;
    }
    if (!aligned_to(positions, static_cast<size_t>(index_bytes(positions_dtype))) || !aligned_to(inv_freq, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: misaligned tensor");
    if (rows == 0) return NVK_OK;
    {   // an output may be its own input, row for row, and a part of the packed rows that its input is another part of
        const int64_t q_row = static_cast<int64_t>(num_q_heads) * head_dim * size, k_row = key ? static_cast<int64_t>(num_kv_heads) * head_dim * size : 0;
        const Rows q{query, query_row_stride * size, q_row, rows}, k{key, key_row_stride * size, k_row, rows};
        const Rows q_out{query_out, query_out_row_stride * size, q_row, rows}, k_out{key_out, key_out_row_stride * size, k_row, rows};
        const int64_t positions_bytes = rows * index_bytes(positions_dtype), freq_bytes = rotary_dim / 2 * static_cast<int64_t>(sizeof(float));
        const Rows pos{positions, positions_bytes, positions_bytes, 1}, freq{inv_freq, freq_bytes, freq_bytes, 1};
        auto same = [](const Rows& a, const Rows& b) { return a.at == b.at && (a.stride == b.stride || a.rows == 1); };
        if ((!same(q, q_out) && rows_overlap(q, q_out)) || (!same(k, k_out) && rows_overlap(k, k_out)) || rows_overlap(q_out, k) || rows_overlap(k_out, q) ||
            rows_overlap(q_out, k_out) || rows_overlap(q_out, pos) || rows_overlap(k_out, pos) || rows_overlap(q_out, freq) || rows_overlap(k_out, freq))
            return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_embedding: an output is its input, with its stride, or does not overlap with any tensor of the call");
    }
    return launch_rotary(RotaryArgs{query, key, query_out, key_out, query_row_stride, key_row_stride, query_out_row_stride, key_out_row_stride,
                                    index_array(positions, positions_dtype), inv_freq, attention_factor, rows, num_q_heads, num_kv_heads, head_dim, rotary_dim,
                                    interleaved != 0, dtype, static_cast<cudaStream_t>(stream)});
}

int nvk_rotary_inv_freq(float* inv_freq, float* attention_factor, int rotary_dim, double base, int scaling, double factor, double original_positions,
                        double low_turns, double high_turns) {
    if (!inv_freq || !attention_factor) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: inv_freq and attention_factor must be defined");
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || !(base > 0.0) || !std::isfinite(base)) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: rotary_dim must be even, base positive");
    if (scaling < NVK_ROPE_PLAIN || scaling > NVK_ROPE_YARN) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: no such scaling (%d)", scaling);
    if (scaling != NVK_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: factor must be at least 1");
    if (scaling == NVK_ROPE_BASE && rotary_dim <= 2) return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: a scaled base needs more than one pair");
    const bool parts = scaling == NVK_ROPE_PARTS || scaling == NVK_ROPE_YARN;
    if (parts && (!(original_positions > 0.0) || !(high_turns > low_turns)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "rotary_inv_freq: original_positions must be positive, high_turns above low_turns");
    if (scaling == NVK_ROPE_BASE) base *= std::pow(factor, static_cast<double>(rotary_dim) / (rotary_dim - 2));
    for (int i = 0; i < rotary_dim / 2; ++i) {
        const double theta = std::pow(base, -2.0 * i / rotary_dim);
        double f = theta;
        if (scaling == NVK_ROPE_LINEAR) f = theta / factor;
        if (parts) {
            const double turns = original_positions * theta / 6.283185307179586;
            const double g = std::fmin(std::fmax((turns - low_turns) / (high_turns - low_turns), 0.0), 1.0);
            f = (1.0 - g) * theta / factor + g * theta;
        }
        inv_freq[i] = static_cast<float>(f);
    }
    *attention_factor = scaling == NVK_ROPE_YARN ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
    return NVK_OK;
}

size_t nvk_decode_attention_weights_workspace_bytes(int64_t batch, int num_heads, int num_kv_heads, int head_dim, int64_t max_blocks, int block_size) {
    return head_dim > 0 ? decode_weights_workspace_bytes(batch, num_heads, num_kv_heads, max_blocks, block_size) : 0;
}

int nvk_decode_attention_paged_weights(const void* query, const void* k_cache, const void* v_cache, const void* k_params, const void* v_params,
                                       const void* context_lens, int context_lens_dtype, const void* block_tables, int block_tables_dtype,
                                       int64_t batch, int64_t max_blocks, int64_t num_cache_blocks, int num_heads, int num_kv_heads,
                                       int head_dim, int block_size, float scale, const float* key_weights, const void* weight_rows,
                                       int weight_rows_dtype, int64_t num_weight_rows, int64_t weight_row_keys, float* new_key_weights,
                                       void* output, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (!query || !k_cache || !v_cache || !context_lens || !block_tables || !new_key_weights || !output)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights) requires KV cache, context_lens, block_tables, new_key_weights and output");
    if ((k_params == nullptr) != (v_params == nullptr)) return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): k_params and v_params go together");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype) || (weight_rows && !is_index_dtype(weight_rows_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens, block_tables and weight_rows must be int32 or int64");
    if (const int rc = check_decode_sizes(batch, max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size); rc != NVK_OK) return rc;
    if (num_weight_rows <= 0 || weight_row_keys <= 0 || weight_row_keys / block_size < max_blocks)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): a row of weights has to hold max_blocks * block_size keys");
    if (!weight_rows && num_weight_rows < batch)
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): without weight_rows there has to be a row of weights for every sequence");
    if (batch == 0) return NVK_OK;
    const DecodeArgs a{query, k_cache, v_cache, index_array(context_lens, context_lens_dtype), index_array(block_tables, block_tables_dtype), output, batch,
                       max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream)};
    if (k_params ? !decode_int4_supported(a, k_params, v_params) : !decode_mma_supported(a))
        return fail(NVK_ERR_UNSUPPORTED, "decode attention (weights): F16 / BF16 queries, head_dim 128, at most 8 query heads per KV head, block_size a "
                                         "multiple of 16; caches (4-bit ones: query too) 16-byte aligned, params 4-byte and output 8-byte aligned");
    if (!aligned_to(key_weights, 4) || !aligned_to(new_key_weights, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): weights must be 4-byte aligned");
    if (weights_overlap(key_weights, new_key_weights, num_weight_rows, num_kv_heads, weight_row_keys))
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): new_key_weights must be key_weights or not overlap with it");
    const size_t need = decode_weights_workspace_bytes(batch, num_heads, num_kv_heads, max_blocks, block_size);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(NVK_ERR_INVALID_ARGUMENT, "decode attention (weights): a 16-byte aligned workspace of %zu bytes is needed "
                                              "(nvk_decode_attention_weights_workspace_bytes)", need);
    return launch_decode_weights(a, k_params, v_params,
                                 KeyWeights{key_weights, new_key_weights, index_array(weight_rows, weight_rows_dtype), num_weight_rows, weight_row_keys});
}

int nvk_evict_kvcache(void* k_cache, void* v_cache, void* k_params, void* v_params, const float* key_weights, const void* weight_rows,
                      int weight_rows_dtype, int64_t num_weight_rows, int64_t weight_row_keys, const void* context_lens, int context_lens_dtype,
                      const void* block_tables, int block_tables_dtype, int64_t batch, int64_t max_blocks, int64_t num_cache_blocks,
                      float* new_key_weights, const void* new_block_tables, int new_block_tables_dtype, int64_t new_max_blocks,
                      void* new_context_lens, int num_kv_heads, int head_dim, int block_size, int64_t budget, int64_t sinks, int64_t recent,
                      int dtype, void* stream) {
    if (!k_cache || !v_cache || !key_weights || !context_lens || !block_tables || !new_key_weights || !new_block_tables || !new_context_lens)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: the caches, weights, context lengths and block tables must be defined");
    if ((k_params == nullptr) != (v_params == nullptr)) return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: k_params and v_params go together");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(block_tables_dtype) || !is_index_dtype(new_block_tables_dtype) ||
        (weight_rows && !is_index_dtype(weight_rows_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "context_lens, block_tables, new_block_tables and weight_rows must be int32 or int64");
    if (const int rc = check_int4("evict_kvcache", dtype, num_kv_heads, head_dim); rc != NVK_OK) return rc;
    if (batch < 0 || max_blocks <= 0 || new_max_blocks <= 0 || num_cache_blocks <= 0 || block_size <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: sizes must be positive");
    if (sinks < 0 || recent < 0 || budget <= 0 || sinks > budget || recent > budget - sinks)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: budget must be positive, sinks and recent not negative and no more than it together");
    if (num_weight_rows <= 0 || weight_row_keys <= 0 || weight_row_keys / block_size < max_blocks)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: a row of weights has to hold max_blocks * block_size keys");
    if (!weight_rows && num_weight_rows < batch)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: without weight_rows there has to be a row of weights for every sequence");
    if (new_max_blocks < max_blocks && new_max_blocks < (budget + block_size - 1) / block_size)
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: new_block_tables has to hold the budget, or as many blocks as block_tables");
    if (!aligned_to(k_cache, 16) || !aligned_to(v_cache, 16) || !aligned_to(k_params, 4) || !aligned_to(v_params, 4) || !aligned_to(key_weights, 4) ||
        !aligned_to(new_key_weights, 4))
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: the caches must be 16-byte aligned, params and weights 4-byte aligned");
    if (batch == 0) return NVK_OK;
    if (overlap(new_context_lens, batch * index_bytes(context_lens_dtype), context_lens, batch * index_bytes(context_lens_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: new_context_lens must not be context_lens");
    if (weights_overlap(key_weights, new_key_weights, num_weight_rows, num_kv_heads, weight_row_keys))
        return fail(NVK_ERR_INVALID_ARGUMENT, "evict_kvcache: new_key_weights must be key_weights or not overlap with it");
    return launch_evict(EvictArgs{k_cache, v_cache, k_params, v_params, key_weights, new_key_weights, index_array(weight_rows, weight_rows_dtype),
                                  index_array(context_lens, context_lens_dtype), index_array(block_tables, block_tables_dtype),
                                  index_array(new_block_tables, new_block_tables_dtype), new_context_lens, batch, num_weight_rows, weight_row_keys, max_blocks,
                                  new_max_blocks, num_cache_blocks, budget, sinks, recent, num_kv_heads, block_size, static_cast<cudaStream_t>(stream)});
}

int nvk_prefill_attention_varlen(const void* query, const void* key, const void* value, const void* k_cache,
                                 const void* v_cache, const void* cu_seqlens_q, int cu_seqlens_q_dtype,
                                 const void* cu_seqlens_k, int cu_seqlens_k_dtype, const void* block_tables,
                                 int block_tables_dtype, int64_t num_seqs, int64_t total_q, int64_t total_k,
                                 int64_t max_blocks, int64_t num_cache_blocks, int max_seqlen_q, int num_heads,
                                 int num_kv_heads, int head_dim, int block_size, float scale, void* output,
                                 int dtype, void* stream) {
    if (!query || !output) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: query and output must be defined");
    if (!is_compute_dtype(dtype)) return fail(NVK_ERR_INVALID_ARGUMENT, "unsupported dtype for prefill attention");
    if (num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || total_q < 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "attention dimensions must be positive");
    if (num_heads % num_kv_heads != 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    if ((cu_seqlens_q && !is_index_dtype(cu_seqlens_q_dtype)) || (cu_seqlens_k && !is_index_dtype(cu_seqlens_k_dtype)) ||
        (block_tables && !is_index_dtype(block_tables_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "cu_seqlens and block_tables must be int32 or int64");
    const bool paged = block_tables != nullptr;
    if (paged) {
        if (!cu_seqlens_q || !cu_seqlens_k)
            return fail(NVK_ERR_INVALID_ARGUMENT, "paged prefill attention requires cu_seqlens_q and cu_seqlens_k");
        if (!k_cache || !v_cache) return fail(NVK_ERR_INVALID_ARGUMENT, "paged prefill attention requires k_cache and v_cache");
        if (max_blocks <= 0 || num_cache_blocks <= 0 || block_size <= 0)
            return fail(NVK_ERR_INVALID_ARGUMENT, "paged prefill attention: block sizes must be positive");
    } else {
        if (!key || !value) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: key and value must be defined");
        if (total_k < 0) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: total_k must be non-negative");
        if ((cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr)) { cu_seqlens_q = nullptr; cu_seqlens_k = nullptr; }
    }
    if (cu_seqlens_q && num_seqs <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: num_seqs must be positive");
    if (total_q == 0) return NVK_OK;
    PrefillArgs a{query, key, value, k_cache, v_cache, index_array(cu_seqlens_q, cu_seqlens_q_dtype),
                  index_array(cu_seqlens_k, cu_seqlens_k_dtype), index_array(block_tables, block_tables_dtype), output, num_seqs,
                  total_q, total_k, max_blocks, num_cache_blocks, max_seqlen_q, num_heads, num_kv_heads, head_dim,
                  block_size, scale, dtype, static_cast<cudaStream_t>(stream)};
    return launch_prefill(a);
}

int nvk_attention_mixed_step(const void* p_query, const void* p_key, const void* p_value, const void* k_cache, const void* v_cache,
                             const void* cu_seqlens_q, int cu_seqlens_q_dtype, const void* cu_seqlens_k, int cu_seqlens_k_dtype,
                             const void* p_block_tables, int p_block_tables_dtype, int64_t num_seqs, int64_t total_q,
                             int64_t total_k, int64_t p_max_blocks, int max_seqlen_q, void* p_output, const void* d_query,
                             const void* context_lens, int context_lens_dtype, const void* d_block_tables,
                             int d_block_tables_dtype, int64_t batch, int64_t d_max_blocks, void* d_output,
                             int64_t num_cache_blocks, int num_heads, int num_kv_heads, int head_dim, int block_size, float scale,
                             int dtype, void* workspace, size_t workspace_bytes, int prefill_blocks, void* stream) {
    if (!p_query || !p_output || !d_query || !d_output || !k_cache || !v_cache || !context_lens || !d_block_tables)
        return fail(NVK_ERR_INVALID_ARGUMENT, "mixed step: queries, outputs, the KV cache, context_lens and the decode block tables must be defined");
    if (!is_index_dtype(context_lens_dtype) || !is_index_dtype(d_block_tables_dtype) || (cu_seqlens_q && !is_index_dtype(cu_seqlens_q_dtype)) ||
        (cu_seqlens_k && !is_index_dtype(cu_seqlens_k_dtype)) || (p_block_tables && !is_index_dtype(p_block_tables_dtype)))
        return fail(NVK_ERR_INVALID_ARGUMENT, "mixed step: index tensors must be int32 or int64");
    if (num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_cache_blocks <= 0 || total_q <= 0 || batch <= 0 ||
        d_max_blocks <= 0)
        return fail(NVK_ERR_INVALID_ARGUMENT, "mixed step: sizes must be positive (a step without prefill rows or without decode rows takes the single-purpose entry point)");
    if (num_heads % num_kv_heads != 0) return fail(NVK_ERR_INVALID_ARGUMENT, "num_heads must be divisible by num_kv_heads");
    const bool paged = p_block_tables != nullptr;
    if (paged && (!cu_seqlens_q || !cu_seqlens_k || p_max_blocks <= 0))
        return fail(NVK_ERR_INVALID_ARGUMENT, "paged prefill attention requires cu_seqlens_q and cu_seqlens_k");
    if (!paged && (!p_key || !p_value)) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: key and value must be defined");
    if ((cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr)) { cu_seqlens_q = nullptr; cu_seqlens_k = nullptr; }
    if (cu_seqlens_q && num_seqs <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "prefill attention: num_seqs must be positive");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    PrefillArgs pa{p_query, p_key, p_value, k_cache, v_cache, index_array(cu_seqlens_q, cu_seqlens_q_dtype),
                   index_array(cu_seqlens_k, cu_seqlens_k_dtype), index_array(p_block_tables, p_block_tables_dtype), p_output, num_seqs,
                   total_q, total_k, p_max_blocks, num_cache_blocks, max_seqlen_q, num_heads, num_kv_heads, head_dim, block_size, scale,
                   dtype, st};
    DecodeArgs da{d_query, k_cache, v_cache, index_array(context_lens, context_lens_dtype), index_array(d_block_tables, d_block_tables_dtype),
                  d_output, batch, d_max_blocks, num_cache_blocks, num_heads, num_kv_heads, head_dim, block_size, scale, dtype, workspace,
                  workspace_bytes, st};
    const size_t need = decode_mma_workspace_needed(batch, num_heads, num_kv_heads, head_dim, d_max_blocks, block_size);
    if (workspace == nullptr || workspace_bytes < need || !aligned_to(workspace, 16))
        return fail(NVK_ERR_INVALID_ARGUMENT, "mixed step: a 16-byte aligned workspace of %zu bytes is needed (nvk_decode_attention_workspace_bytes)", need);
    if (!mixed_step_supported(pa, da))
        return fail(NVK_ERR_UNSUPPORTED, "mixed step: needs F16 / BF16, head_dim 128, an even number of query heads per KV head, at most 8, and "
                                         "paged block sizes that are multiples of 128; call the prefill and decode entry points instead");
    // A scale that is not positive: the prefill rows take another kernel.  So do few of them, and the decode kernel runs beside that one (us a step as
    // one launch / as these: 1 prompt of 670 tokens, 5 decode rows of 400 keys, 4 / 1 heads, 22.7 / 15.0; 3 of 109 to 136, 9 of up to 1929, 16 / 4
    // heads, 20.1 / 16.2; 1 of 300, 60 of up to 4096, 4 / 1 heads, 31.6 / 27.4).
    // More decode rows than the decode kernel's grid has room for stay in one launch, or are refused before anything is launched.
    const bool one_launch = prefill_tc_supported(pa), small = one_launch && prefill_takes_tiles(pa);
    if (small || !one_launch) {
        int rc = check_decode_mma(da);
        if (rc == NVK_OK) {
            rc = launch_prefill(pa);
            da.beside = small;
            return rc != NVK_OK ? rc : launch_decode_mma(da);
        }
        if (!one_launch) return rc;
    }
    return launch_mixed_step(pa, da, prefill_blocks);
}

}  // extern "C"
