// Operator wrappers: the reference's C++ kernel API (include/kernels/*.h of nano-vllm-cpp) implemented
// as argument checks + one call into the C ABI of libnvk.so (include/nvk.h).  Error behaviour follows
// the reference: std::invalid_argument for bad operands (src/kernels/kvcache.cu:146-190,
// src/kernels/kernel_types.cu:24-110), std::runtime_error for CUDA failures.
#include "kernels/attention.h"
#include "kernels/flash_attn.h"
#include "kernels/kernel_types.h"
#include "engine/step_metadata.h"
#include "kernels/kvcache.h"
#include "kernels/rotary.h"
#include "kernels/split_qkv.h"

#include "nvk.h"

#include "../../csrc/decode_sizes.h"

#include <cmath>
#include <stdexcept>
#include <string>

namespace nano_vllm {

// ---- checks -----------------------------------------------------------------------------------------
void ensure_cuda_tensor(const char* name, const Tensor& tensor) {
    if (!tensor.defined()) throw std::invalid_argument(std::string(name) + " must be defined");
    if (tensor.device().type != DeviceType::kCUDA) throw std::invalid_argument(std::string(name) + " must live on CUDA");
    if (!tensor.is_contiguous()) throw std::invalid_argument(std::string(name) + " must be contiguous");
}

void ensure_same_device(const char* lhs_name, const Tensor& lhs, const char* rhs_name, const Tensor& rhs) {
    if (lhs.device() != rhs.device())
        throw std::invalid_argument(std::string(lhs_name) + " and " + rhs_name + " must be on the same device");
}

void ensure_same_shape(const char* lhs_name, const Tensor& lhs, const char* rhs_name, const Tensor& rhs) {
    if (lhs.sizes() != rhs.sizes())
        throw std::invalid_argument(std::string(lhs_name) + " and " + rhs_name + " must have the same shape");
}

void ensure_same_dtype(const char* lhs_name, const Tensor& lhs, const char* rhs_name, const Tensor& rhs) {
    if (lhs.dtype() != rhs.dtype())
        throw std::invalid_argument(std::string(lhs_name) + " and " + rhs_name + " must have the same dtype");
}

void validate_supported_dtype(const char* name, ScalarType dtype) {
    if (dtype != ScalarType::kFloat16 && dtype != ScalarType::kBFloat16 && dtype != ScalarType::kFloat32)
        throw std::invalid_argument(std::string(name) + " must be float16, bfloat16, or float32");
}

MatrixShape flatten_by_leading_count(const char* name, const Tensor& tensor, int64_t leading_count) {
    if (leading_count <= 0) throw std::invalid_argument(std::string(name) + " must have a positive leading count");
    const int64_t total = static_cast<int64_t>(tensor.numel());
    const int64_t cols = total / leading_count;
    if (cols <= 0 || cols * leading_count != total)
        throw std::invalid_argument(std::string(name) + " cannot be flattened by the provided leading count");
    return {leading_count, cols};
}

int64_t cache_rows_from_tensor(const char* name, const Tensor& tensor, int64_t row_width) {
    if (row_width <= 0) throw std::invalid_argument(std::string(name) + " row width must be positive");
    const int64_t total = static_cast<int64_t>(tensor.numel());
    const int64_t rows = total / row_width;
    if (rows <= 0 || rows * row_width != total)
        throw std::invalid_argument(std::string(name) + " does not contain an integer number of cache rows");
    return rows;
}

void throw_on_nvk_status(int status) {
    if (status == NVK_OK) return;
    if (status == NVK_ERR_CUDA) throw std::runtime_error(nvk_last_error());
    throw std::invalid_argument(nvk_last_error());
}

namespace {

int code(ScalarType t) { return static_cast<int>(t); }

const int32_t* int32_data(const char* name, const Tensor& t) {
    ensure_cuda_tensor(name, t);
    if (t.dtype() != ScalarType::kInt32) throw std::invalid_argument(std::string(name) + " must be int32");
    return t.data_as<int32_t>();
}

// An index tensor of either width (the reference's attention kernels take int32 or int64 for each of cu_seqlens_q,
// cu_seqlens_k, context_lens and block_tables on its own, src/kernels/attention.cu:644-660, :708-735).
struct IndexRef { const void* ptr; int dtype; };
IndexRef index_data(const char* name, const Tensor& t) {
    ensure_cuda_tensor(name, t);
    if (t.dtype() != ScalarType::kInt32 && t.dtype() != ScalarType::kInt64)
        throw std::invalid_argument(std::string(name) + " must be int32 or int64");
    return {t.data(), code(t.dtype())};
}

int64_t cache_blocks(const Tensor& cache, int block_size, int num_kv_heads, int head_dim) {
    const int64_t per_block = static_cast<int64_t>(block_size) * num_kv_heads * head_dim;
    if (per_block <= 0) throw std::invalid_argument("attention dimensions must be positive");
    return static_cast<int64_t>(cache.numel()) / per_block;
}

void check_qo(const Tensor& query, const Tensor& output) {
    ensure_cuda_tensor("query", query);
    ensure_cuda_tensor("output", output);
    ensure_same_device("query", query, "output", output);
    ensure_same_dtype("query", query, "output", output);
    ensure_same_shape("query", query, "output", output);
    if (query.dim() != 3) throw std::invalid_argument("attention expects [tokens, heads, head_dim] tensors");
}

}  // namespace

// ---- store_kvcache ----------------------------------------------------------------------------------
void store_kvcache(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, const Tensor& slot_mapping,
                   cudaStream_t stream) {
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_cuda_tensor("slot_mapping", slot_mapping);
    ensure_same_device("key", key, "value", value);
    ensure_same_device("key", key, "k_cache", k_cache);
    ensure_same_device("key", key, "v_cache", v_cache);
    ensure_same_device("key", key, "slot_mapping", slot_mapping);
    ensure_same_dtype("key", key, "value", value);
    ensure_same_dtype("key", key, "k_cache", k_cache);
    ensure_same_dtype("key", key, "v_cache", v_cache);
    validate_supported_dtype("key", key.dtype());
    if (slot_mapping.dtype() != ScalarType::kInt32 && slot_mapping.dtype() != ScalarType::kInt64)
        throw std::invalid_argument("slot_mapping must be int32 or int64");
    const int64_t tokens = static_cast<int64_t>(slot_mapping.numel());
    if (tokens <= 0) throw std::invalid_argument("slot_mapping must contain at least one element");
    const MatrixShape k = flatten_by_leading_count("key", key, tokens);
    const MatrixShape v = flatten_by_leading_count("value", value, tokens);
    if (k.cols != v.cols) throw std::invalid_argument("key and value must have the same flattened row width");
    const int64_t k_rows = cache_rows_from_tensor("k_cache", k_cache, k.cols);
    const int64_t v_rows = cache_rows_from_tensor("v_cache", v_cache, k.cols);
    if (k_rows != v_rows) throw std::invalid_argument("k_cache and v_cache must contain the same number of slots");
    throw_on_nvk_status(nvk_store_kvcache(key.data(), value.data(), k_cache.data(), v_cache.data(), slot_mapping.data(),
                                          code(slot_mapping.dtype()), tokens, k.cols, k_rows, code(key.dtype()), stream));
}

void store_kvcache_int8(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_scale,
                        Tensor& v_scale, const Tensor& slot_mapping, cudaStream_t stream) {
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_cuda_tensor("k_scale", k_scale);
    ensure_cuda_tensor("v_scale", v_scale);
    ensure_cuda_tensor("slot_mapping", slot_mapping);
    validate_supported_dtype("key", key.dtype());
    ensure_same_dtype("key", key, "value", value);
    if (k_cache.dtype() != ScalarType::kInt8 || v_cache.dtype() != ScalarType::kInt8)
        throw std::invalid_argument("store_kvcache_int8 requires int8 caches");
    if (k_scale.dtype() != ScalarType::kFloat16 || v_scale.dtype() != ScalarType::kFloat16)
        throw std::invalid_argument("store_kvcache_int8 requires float16 scales");
    if (slot_mapping.dtype() != ScalarType::kInt32) throw std::invalid_argument("slot_mapping must be int32 for the int8 store");
    const int64_t tokens = static_cast<int64_t>(slot_mapping.numel());
    if (tokens <= 0) return;   // the reference returns without a launch
    if (key.dim() != 3) throw std::invalid_argument("key must be rank-3 for int8 store");
    ensure_same_shape("key", key, "value", value);
    if (key.sizes()[0] != tokens) throw std::invalid_argument("key rows must match slot_mapping");
    const int heads = static_cast<int>(key.sizes()[1]);
    const int head_dim = static_cast<int>(key.sizes()[2]);
    const int64_t row = static_cast<int64_t>(heads) * head_dim;
    const int64_t rows = cache_rows_from_tensor("k_cache", k_cache, row);
    if (cache_rows_from_tensor("v_cache", v_cache, row) != rows)
        throw std::invalid_argument("k_cache and v_cache must contain the same number of slots");
    if (static_cast<int64_t>(k_scale.numel()) != rows * heads || static_cast<int64_t>(v_scale.numel()) != rows * heads)
        throw std::invalid_argument("k_scale and v_scale must hold one value per cache row and KV head");
    throw_on_nvk_status(nvk_store_kvcache_int8(key.data(), value.data(), k_cache.data(), v_cache.data(), k_scale.data(),
                                               v_scale.data(), static_cast<const int32_t*>(slot_mapping.data()), tokens, heads,
                                               head_dim, rows, code(key.dtype()), stream));
}

// ---- 4-bit cache, eviction --------------------------------------------------------------------------
namespace {

// Caches and params of a 4-bit cache agree with one another and with `type`; its rows.
int64_t int4_rows(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_params, const Tensor& v_params, ScalarType type, int heads, int head_dim) {
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_cuda_tensor("k_params", k_params);
    ensure_cuda_tensor("v_params", v_params);
    ensure_same_device("k_cache", k_cache, "v_cache", v_cache);
    ensure_same_device("k_cache", k_cache, "k_params", k_params);
    ensure_same_device("k_cache", k_cache, "v_params", v_params);
    if (k_cache.dtype() != ScalarType::kInt8 || v_cache.dtype() != ScalarType::kInt8)
        throw std::invalid_argument("4-bit caches must be byte (int8) tensors");
    if (type != ScalarType::kFloat16 && type != ScalarType::kBFloat16) throw std::invalid_argument("a 4-bit cache needs float16 or bfloat16");
    if (k_params.dtype() != type || v_params.dtype() != type) throw std::invalid_argument("k_params and v_params must have the type of the keys");
    if (head_dim != 128) throw std::invalid_argument("a 4-bit cache needs head_dim 128");
    const int64_t row = static_cast<int64_t>(heads) * (head_dim / 2), rows = cache_rows_from_tensor("k_cache", k_cache, row);
    if (cache_rows_from_tensor("v_cache", v_cache, row) != rows) throw std::invalid_argument("k_cache and v_cache must contain the same number of slots");
    if (static_cast<int64_t>(k_params.numel()) != 2 * rows * heads || static_cast<int64_t>(v_params.numel()) != 2 * rows * heads)
        throw std::invalid_argument("k_params and v_params must hold a pair per cache row and KV head");
    return rows;
}

void ensure_rows(const char* name, const Tensor& t, int64_t rows) {
    if (t.sizes().empty() || t.sizes()[0] != rows) throw std::invalid_argument(std::string(name) + " must have a row for every sequence");
}

}  // namespace

void store_kvcache_int4(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_params,
                        Tensor& v_params, const Tensor& slot_mapping, cudaStream_t stream) {
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_same_dtype("key", key, "value", value);
    ensure_same_shape("key", key, "value", value);
    ensure_same_device("key", key, "value", value);
    const IndexRef slots = index_data("slot_mapping", slot_mapping);
    ensure_same_device("key", key, "slot_mapping", slot_mapping);
    if (key.dim() != 3 || key.sizes()[0] != static_cast<int64_t>(slot_mapping.numel()))
        throw std::invalid_argument("key must be [tokens, num_kv_heads, head_dim] with a slot for every token");
    const int heads = static_cast<int>(key.sizes()[1]), head_dim = static_cast<int>(key.sizes()[2]);
    const int64_t rows = int4_rows(k_cache, v_cache, k_params, v_params, key.dtype(), heads, head_dim);
    ensure_same_device("key", key, "k_cache", k_cache);
    throw_on_nvk_status(nvk_store_kvcache_int4(key.data(), value.data(), k_cache.data(), v_cache.data(), k_params.data(), v_params.data(), slots.ptr, slots.dtype,
                                               key.sizes()[0], heads, head_dim, rows, code(key.dtype()), stream));
}

void gather_kvcache_int4(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_params, const Tensor& v_params,
                         const Tensor& cu_seqlens_k, const Tensor& block_tables, int num_kv_heads, int head_dim,
                         int block_size, Tensor& key, Tensor& value, cudaStream_t stream) {
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_same_dtype("key", key, "value", value);
    ensure_same_shape("key", key, "value", value);
    const IndexRef starts = index_data("cu_seqlens_k", cu_seqlens_k), tables = index_data("block_tables", block_tables);
    const int64_t rows = int4_rows(k_cache, v_cache, k_params, v_params, key.dtype(), num_kv_heads, head_dim);
    ensure_same_device("key", key, "k_cache", k_cache);
    ensure_same_device("key", key, "value", value);
    ensure_same_device("key", key, "cu_seqlens_k", cu_seqlens_k);
    ensure_same_device("key", key, "block_tables", block_tables);
    if (key.dim() != 3 || key.sizes()[1] != num_kv_heads || key.sizes()[2] != head_dim)
        throw std::invalid_argument("key must be [total_k, num_kv_heads, head_dim]");
    const int64_t seqs = static_cast<int64_t>(cu_seqlens_k.numel()) - 1;
    if (block_tables.dim() != 2 || block_size <= 0) throw std::invalid_argument("block_tables must be [num_seqs, max_blocks], block_size positive");
    ensure_rows("block_tables", block_tables, seqs);
    throw_on_nvk_status(nvk_gather_kvcache_int4(k_cache.data(), v_cache.data(), k_params.data(), v_params.data(), starts.ptr, starts.dtype, tables.ptr,
                                                tables.dtype, seqs, key.sizes()[0], block_tables.sizes()[1], rows / block_size, num_kv_heads, head_dim,
                                                block_size, key.data(), value.data(), code(key.dtype()), stream));
}

// ---- 8-bit cache with block scales --------------------------------------------------------------------
namespace {

struct Blocks8 {   // caches and scales that agree
    int64_t blocks;
    int block_size, heads, head_dim, type;
    Blocks8(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale, bool e4m3) : type(e4m3 ? NVK_E4M3 : NVK_I8) {
        ensure_cuda_tensor("k_cache", k_cache);
        ensure_cuda_tensor("v_cache", v_cache);
        ensure_cuda_tensor("k_scale", k_scale);
        ensure_cuda_tensor("v_scale", v_scale);
        ensure_same_device("k_cache", k_cache, "v_cache", v_cache);
        ensure_same_device("k_cache", k_cache, "k_scale", k_scale);
        ensure_same_device("k_cache", k_cache, "v_scale", v_scale);
        ensure_same_shape("k_cache", k_cache, "v_cache", v_cache);
        if (k_cache.dtype() != ScalarType::kInt8 || v_cache.dtype() != ScalarType::kInt8) throw std::invalid_argument("8-bit caches must be byte (int8) tensors");
        if (k_cache.dim() != 4) throw std::invalid_argument("k_cache must be [blocks, block_size, num_kv_heads, head_dim]");
        if (k_cache.numel() == 0) throw std::invalid_argument("k_cache must contain at least one cache block");
        if (k_scale.dtype() != ScalarType::kFloat32 || v_scale.dtype() != ScalarType::kFloat32) throw std::invalid_argument("k_scale and v_scale must be float32");
        blocks = k_cache.sizes()[0];
        block_size = static_cast<int>(k_cache.sizes()[1]);
        heads = static_cast<int>(k_cache.sizes()[2]);
        head_dim = static_cast<int>(k_cache.sizes()[3]);
        if (static_cast<int64_t>(k_scale.numel()) != blocks * heads || k_scale.numel() != v_scale.numel())
            throw std::invalid_argument("k_scale and v_scale must hold one value per cache block and KV head");
    }
};

// Rows [rows, heads, head_dim], or [rows, heads * head_dim] that may be slices of wider ones; the elements from one to the next.
int64_t packed_rows(const char* name, const Tensor& t, int heads, int head_dim) {
    const std::string n(name);
    if (!t.defined()) throw std::invalid_argument(n + " must be defined");
    if (t.device().type != DeviceType::kCUDA) throw std::invalid_argument(n + " must live on CUDA");
    const int64_t row = static_cast<int64_t>(heads) * head_dim;
    if (t.dim() == 3 ? t.sizes()[1] != heads || t.sizes()[2] != head_dim || !t.is_contiguous() : t.dim() != 2 || t.sizes()[1] != row || t.strides()[1] != 1)
        throw std::invalid_argument(n + " must be [rows, heads, head_dim], or rows of heads * head_dim elements");
    return t.sizes()[0] > 1 && t.dim() == 2 ? t.strides()[0] : row;
}

}  // namespace

void store_kvcache_blocks8(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_scale,
                           Tensor& v_scale, const Tensor& cu_seqlens_q, const Tensor& context_lens, const Tensor& block_tables, bool e4m3,
                           cudaStream_t stream) {
    const Blocks8 c(k_cache, v_cache, k_scale, v_scale, e4m3);
    const int64_t key_stride = packed_rows("key", key, c.heads, c.head_dim), value_stride = packed_rows("value", value, c.heads, c.head_dim);
    ensure_same_dtype("key", key, "value", value);
    if (key.sizes()[0] != value.sizes()[0]) throw std::invalid_argument("key and value must have the same number of rows");
    ensure_same_device("key", key, "value", value);
    ensure_same_device("key", key, "k_cache", k_cache);
    const IndexRef lens = index_data("context_lens", context_lens), tables = index_data("block_tables", block_tables);
    const IndexRef starts = cu_seqlens_q.defined() ? index_data("cu_seqlens_q", cu_seqlens_q) : IndexRef{nullptr, NVK_I32};
    ensure_same_device("key", key, "context_lens", context_lens);
    ensure_same_device("key", key, "block_tables", block_tables);
    if (cu_seqlens_q.defined()) ensure_same_device("key", key, "cu_seqlens_q", cu_seqlens_q);
    const int64_t seqs = static_cast<int64_t>(context_lens.numel());
    if (cu_seqlens_q.defined() ? static_cast<int64_t>(cu_seqlens_q.numel()) != seqs + 1 : key.sizes()[0] != seqs)
        throw std::invalid_argument("cu_seqlens_q, or key, must have a sequence for every context length");
    if (block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [num_seqs, max_blocks]");
    ensure_rows("block_tables", block_tables, seqs);
    throw_on_nvk_status(nvk_store_kvcache_blocks8(key.data(), value.data(), key_stride, value_stride, k_cache.data(), v_cache.data(), k_scale.data_as<float>(),
                                                  v_scale.data_as<float>(), c.type, starts.ptr, starts.dtype, lens.ptr, lens.dtype, tables.ptr, tables.dtype, seqs,
                                                  key.sizes()[0], block_tables.sizes()[1], c.blocks, c.heads, c.head_dim, c.block_size, code(key.dtype()), stream));
}

void gather_kvcache_blocks8(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                            const Tensor& cu_seqlens_k, const Tensor& block_tables, Tensor& key, Tensor& value, bool e4m3, cudaStream_t stream) {
    const Blocks8 c(k_cache, v_cache, k_scale, v_scale, e4m3);
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_same_dtype("key", key, "value", value);
    ensure_same_shape("key", key, "value", value);
    const IndexRef starts = index_data("cu_seqlens_k", cu_seqlens_k), tables = index_data("block_tables", block_tables);
    ensure_same_device("key", key, "k_cache", k_cache);
    ensure_same_device("key", key, "value", value);
    ensure_same_device("key", key, "cu_seqlens_k", cu_seqlens_k);
    ensure_same_device("key", key, "block_tables", block_tables);
    if (key.dim() != 3 || key.sizes()[1] != c.heads || key.sizes()[2] != c.head_dim) throw std::invalid_argument("key must be [total_k, num_kv_heads, head_dim]");
    const int64_t seqs = static_cast<int64_t>(cu_seqlens_k.numel()) - 1;
    if (block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [num_seqs, max_blocks]");
    ensure_rows("block_tables", block_tables, seqs);
    throw_on_nvk_status(nvk_gather_kvcache_blocks8(k_cache.data(), v_cache.data(), k_scale.data_as<float>(), v_scale.data_as<float>(), c.type, starts.ptr,
                                                   starts.dtype, tables.ptr, tables.dtype, seqs, key.sizes()[0], block_tables.sizes()[1], c.blocks, c.heads,
                                                   c.head_dim, c.block_size, key.data(), value.data(), code(key.dtype()), stream));
}

// ---- rotary positions ---------------------------------------------------------------------------------
void rotary_embedding(const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& inv_freq, int num_q_heads,
                      int num_kv_heads, int head_dim, bool interleaved, float attention_factor, Tensor& query_out, Tensor& key_out,
                      cudaStream_t stream) {
    if (num_q_heads <= 0 || head_dim <= 0) throw std::invalid_argument("attention dimensions must be positive");
    const int64_t q_stride = packed_rows("query", query, num_q_heads, head_dim), qo_stride = packed_rows("query_out", query_out, num_q_heads, head_dim);
    const IndexRef pos = index_data("positions", positions);
    ensure_cuda_tensor("inv_freq", inv_freq);
    if (inv_freq.dtype() != ScalarType::kFloat32) throw std::invalid_argument("inv_freq must be float32");
    const int64_t rows = query.sizes()[0];
    auto alike = [&](const char* name, const Tensor& t) {
        if (t.sizes()[0] != rows) throw std::invalid_argument(std::string(name) + " must have the rows of query");
        ensure_same_dtype("query", query, name, t);
        ensure_same_device("query", query, name, t);
    };
    alike("query_out", query_out);
    if (key.defined() != key_out.defined()) throw std::invalid_argument("key and key_out go together");
    int64_t k_stride = 0, ko_stride = 0;
    if (key.defined()) {
        k_stride = packed_rows("key", key, num_kv_heads, head_dim);
        ko_stride = packed_rows("key_out", key_out, num_kv_heads, head_dim);
        alike("key", key);
        alike("key_out", key_out);
    }
    ensure_same_device("query", query, "positions", positions);
    ensure_same_device("query", query, "inv_freq", inv_freq);
    if (static_cast<int64_t>(positions.numel()) != rows) throw std::invalid_argument("positions must have an element for every row");
    if (static_cast<int64_t>(inv_freq.numel()) > head_dim / 2) throw std::invalid_argument("inv_freq must have an element for every pair, at most head_dim / 2");
    throw_on_nvk_status(nvk_rotary_embedding(query.data(), key.defined() ? key.data() : nullptr, pos.ptr, pos.dtype, inv_freq.data_as<float>(), attention_factor, rows,
                                             num_q_heads, num_kv_heads, head_dim, static_cast<int>(2 * inv_freq.numel()), interleaved ? 1 : 0, q_stride, k_stride,
                                             query_out.data(), key_out.defined() ? key_out.data() : nullptr, qo_stride, ko_stride, code(query.dtype()), stream));
}

RotaryFrequencies rotary_inv_freq(int rotary_dim, double base, RopeScaling scaling, double factor, double original_positions, double low_turns,
                                  double high_turns) {
    RotaryFrequencies f;
    f.inv_freq.resize(static_cast<size_t>(rotary_dim > 1 ? rotary_dim / 2 : 1));
    throw_on_nvk_status(nvk_rotary_inv_freq(f.inv_freq.data(), &f.attention_factor, rotary_dim, base, static_cast<int>(scaling), factor, original_positions, low_turns,
                                            high_turns));
    return f;
}

// ---- metadata of a step on the device -----------------------------------------------------------------
namespace {

// The tables of requests agree with one another; the width of their elements.
int check_tables(const RequestTables& t) {
    const IndexRef lens = index_data("lens", t.lens);
    struct { const char* name; const Tensor& t; } others[] = {{"blocks", t.blocks}, {"free_blocks", t.free_blocks}, {"free_count", t.free_count}};
    for (const auto& o : others) {
        if (index_data(o.name, o.t).dtype != lens.dtype) throw std::invalid_argument(std::string(o.name) + " must have the dtype of the other index tensors");
        ensure_same_device("lens", t.lens, o.name, o.t);
    }
    if (t.blocks.dim() != 2 || t.blocks.sizes()[0] != static_cast<int64_t>(t.lens.numel())) throw std::invalid_argument("blocks must have a row for every length");
    if (t.free_count.numel() != 1) throw std::invalid_argument("free_count must have one element");
    return lens.dtype;
}
const void* step_index(const char* name, const Tensor& x, const RequestTables& t, int dtype, int64_t elements) {
    if (index_data(name, x).dtype != dtype) throw std::invalid_argument(std::string(name) + " must have the dtype of the other index tensors");
    ensure_same_device("lens", t.lens, name, x);
    if (elements >= 0 && static_cast<int64_t>(x.numel()) != elements) throw std::invalid_argument(std::string(name) + " has the wrong size");
    return x.data();
}
void* step_output(const char* name, const Tensor& x, const RequestTables& t, int dtype, int64_t elements) {
    return x.defined() ? const_cast<void*>(step_index(name, x, t, dtype, elements)) : nullptr;
}

}  // namespace

void build_step(const Tensor& new_lens, const Tensor& rows, RequestTables& tables, DeviceStep& step, cudaStream_t stream) {
    const int dtype = check_tables(tables);
    const int64_t batch = new_lens.defined() ? static_cast<int64_t>(new_lens.numel()) : 0;
    const void* n = step_index("new_lens", new_lens, tables, dtype, batch);
    const void* r = rows.defined() ? step_index("rows", rows, tables, dtype, batch) : nullptr;
    if (!step.block_tables.defined() || step.block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [batch, max_blocks]");
    ensure_rows("block_tables", step.block_tables, batch);
    void* bt = step_output("block_tables", step.block_tables, tables, dtype, -1);
    if (!step.context_lens.defined()) throw std::invalid_argument("context_lens must be defined");
    void* ctx = step_output("context_lens", step.context_lens, tables, dtype, batch);
    void *cu_q = step_output("cu_seqlens_q", step.cu_seqlens_q, tables, dtype, batch + 1), *cu_k = step_output("cu_seqlens_k", step.cu_seqlens_k, tables, dtype, batch + 1);
    if (step.positions.defined() != step.slot_mapping.defined()) throw std::invalid_argument("positions and slot_mapping go together");
    const int64_t tokens = step.positions.defined() ? static_cast<int64_t>(step.positions.numel()) : 0;
    void *pos = step_output("positions", step.positions, tables, dtype, tokens), *slots = step_output("slot_mapping", step.slot_mapping, tables, dtype, tokens);
    throw_on_nvk_status(nvk_step_metadata(n, r, tables.lens.data(), tables.blocks.data(), tables.free_blocks.data(), tables.free_count.data(), batch,
                                          static_cast<int64_t>(tables.lens.numel()), tables.blocks.sizes()[1], static_cast<int64_t>(tables.free_blocks.numel()),
                                          tables.num_cache_blocks, tables.block_size, bt, step.block_tables.sizes()[1], ctx, cu_q, cu_k, pos, slots, tokens,
                                          tables.lens.data(), tables.free_count.data(), dtype, stream));
}

void release_blocks(const Tensor& rows, const Tensor& first_blocks, RequestTables& tables, cudaStream_t stream) {
    const int dtype = check_tables(tables);
    const int64_t batch = static_cast<int64_t>(rows.defined() ? rows.numel() : tables.lens.numel());
    const void* r = rows.defined() ? step_index("rows", rows, tables, dtype, batch) : nullptr;
    const void* f = first_blocks.defined() ? step_index("first_blocks", first_blocks, tables, dtype, batch) : nullptr;
    throw_on_nvk_status(nvk_release_blocks(r, f, tables.lens.data(), tables.blocks.data(), tables.free_blocks.data(), tables.free_count.data(), batch,
                                           static_cast<int64_t>(tables.lens.numel()), tables.blocks.sizes()[1], static_cast<int64_t>(tables.free_blocks.numel()),
                                           tables.block_size, tables.lens.data(), tables.free_count.data(), dtype, stream));
}

void evict_kvcache(Tensor& k_cache, Tensor& v_cache, Tensor& k_params, Tensor& v_params, const Tensor& key_weights,
                   const Tensor& weight_rows, const Tensor& context_lens, const Tensor& block_tables, Tensor& new_key_weights,
                   const Tensor& new_block_tables, Tensor& new_context_lens, int num_kv_heads, int head_dim, int block_size,
                   int64_t budget, int64_t sinks, int64_t recent, cudaStream_t stream) {
    const bool four = k_params.defined() || v_params.defined();
    if (num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0) throw std::invalid_argument("attention dimensions must be positive");
    int64_t blocks = 0;
    if (four) {
        blocks = int4_rows(k_cache, v_cache, k_params, v_params, k_params.defined() ? k_params.dtype() : v_params.dtype(), num_kv_heads, head_dim) / block_size;
    } else {
        ensure_cuda_tensor("k_cache", k_cache);
        ensure_cuda_tensor("v_cache", v_cache);
        ensure_same_dtype("k_cache", k_cache, "v_cache", v_cache);
        ensure_same_device("k_cache", k_cache, "v_cache", v_cache);
        if (k_cache.numel() != v_cache.numel()) throw std::invalid_argument("k_cache and v_cache must contain the same number of slots");
        blocks = cache_blocks(k_cache, block_size, num_kv_heads, head_dim);
    }
    ensure_cuda_tensor("key_weights", key_weights);
    ensure_cuda_tensor("new_key_weights", new_key_weights);
    ensure_same_shape("key_weights", key_weights, "new_key_weights", new_key_weights);
    if (key_weights.dtype() != ScalarType::kFloat32 || new_key_weights.dtype() != ScalarType::kFloat32 || key_weights.dim() != 3 ||
        key_weights.sizes()[1] != num_kv_heads)
        throw std::invalid_argument("key_weights and new_key_weights must be float32 [rows, num_kv_heads, keys]");
    const IndexRef lens = index_data("context_lens", context_lens), tables = index_data("block_tables", block_tables),
                   new_tables = index_data("new_block_tables", new_block_tables), new_lens = index_data("new_context_lens", new_context_lens);
    const IndexRef rows = weight_rows.defined() ? index_data("weight_rows", weight_rows) : IndexRef{nullptr, NVK_I32};
    const int64_t batch = static_cast<int64_t>(context_lens.numel());
    if (new_lens.dtype != lens.dtype || static_cast<int64_t>(new_context_lens.numel()) != batch)
        throw std::invalid_argument("new_context_lens must be like context_lens");
    if (block_tables.dim() != 2 || new_block_tables.dim() != 2) throw std::invalid_argument("block tables must be [batch, max_blocks]");
    ensure_rows("block_tables", block_tables, batch);
    ensure_rows("new_block_tables", new_block_tables, batch);
    if (weight_rows.defined()) ensure_rows("weight_rows", weight_rows, batch);
    for (const Tensor* t : {&key_weights, static_cast<const Tensor*>(&new_key_weights), &context_lens, &block_tables, &new_block_tables,
                            static_cast<const Tensor*>(&new_context_lens)})
        ensure_same_device("k_cache", k_cache, "every other tensor", *t);
    if (weight_rows.defined()) ensure_same_device("k_cache", k_cache, "weight_rows", weight_rows);
    throw_on_nvk_status(nvk_evict_kvcache(k_cache.data(), v_cache.data(), four ? k_params.data() : nullptr, four ? v_params.data() : nullptr,
                                          key_weights.data_as<float>(), rows.ptr, rows.dtype, key_weights.sizes()[0], key_weights.sizes()[2], lens.ptr,
                                          lens.dtype, tables.ptr, tables.dtype, batch, block_tables.sizes()[1], blocks, new_key_weights.data_as<float>(),
                                          new_tables.ptr, new_tables.dtype, new_block_tables.sizes()[1], new_context_lens.data(), num_kv_heads, head_dim,
                                          block_size, budget, sinks, recent, code(four ? k_params.dtype() : k_cache.dtype()), stream));
}

// ---- fused decode prologue ---------------------------------------------------------------------------
void fused_split_norm_rope_store(const Tensor& qkv, const Tensor& positions, const Tensor& q_norm_weight,
                                 const Tensor& k_norm_weight, float norm_eps, const Tensor& cos_sin_cache,
                                 const Tensor& slot_mapping, Tensor& k_cache, Tensor& v_cache, int num_q_heads,
                                 int num_kv_heads, int head_dim, Tensor& q_out, cudaStream_t stream) {
    if (qkv.defined() && qkv.dtype() != ScalarType::kBFloat16 && qkv.dtype() != ScalarType::kFloat16)
        throw std::invalid_argument("fused_split_norm_rope_store only supports bf16/fp16");
    ensure_cuda_tensor("qkv", qkv);
    ensure_cuda_tensor("q_norm_weight", q_norm_weight);
    ensure_cuda_tensor("k_norm_weight", k_norm_weight);
    ensure_cuda_tensor("cos_sin_cache", cos_sin_cache);
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_cuda_tensor("q_out", q_out);
    if (cos_sin_cache.dtype() != ScalarType::kFloat32 || cos_sin_cache.dim() != 2)
        throw std::invalid_argument("cos_sin_cache must be a [max_positions, head_dim] float32 tensor");
    const int64_t row_width = static_cast<int64_t>(num_kv_heads) * head_dim;
    throw_on_nvk_status(nvk_fused_split_norm_rope_store(
        qkv.data(), int32_data("positions", positions), q_norm_weight.data(), k_norm_weight.data(), norm_eps,
        cos_sin_cache.data_as<float>(), cos_sin_cache.sizes()[0], int32_data("slot_mapping", slot_mapping),
        k_cache.data(), v_cache.data(), cache_rows_from_tensor("k_cache", k_cache, row_width), qkv.sizes()[0],
        num_q_heads, num_kv_heads, head_dim, q_out.data(), code(qkv.dtype()), stream));
}

// ---- decode -------------------------------------------------------------------------------------------
namespace {

void decode_common(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache, const Tensor& context_lens,
                   const Tensor& block_tables, int num_kv_heads, int head_dim, int block_size, float scale,
                   Tensor& output, DeviceAllocator* allocator, cudaStream_t stream) {
    check_qo(query, output);
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_same_dtype("query", query, "k_cache", k_cache);
    ensure_same_dtype("query", query, "v_cache", v_cache);
    const IndexRef lens = index_data("context_lens", context_lens);
    const IndexRef tables = index_data("block_tables", block_tables);
    if (block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [batch, max_blocks]");
    const int64_t batch = query.sizes()[0];
    const int heads = static_cast<int>(query.sizes()[1]);
    const int64_t max_blocks = block_tables.sizes()[1];
    const int64_t blocks = cache_blocks(k_cache, block_size, num_kv_heads, head_dim);
    if (allocator != nullptr) {
        const size_t need = nvk::decode_mma_workspace_needed(batch, heads, num_kv_heads, head_dim, max_blocks, block_size);
        Memory::Ptr scratch = need > 0 ? allocator->allocate_on(need, query.device(), stream) : nullptr;
        throw_on_nvk_status(nvk_decode_attention_paged(query.data(), k_cache.data(), v_cache.data(), lens.ptr, lens.dtype,
                                                       tables.ptr, tables.dtype, batch, max_blocks, blocks, heads,
                                                       num_kv_heads, head_dim, block_size, scale, output.data(),
                                                       code(query.dtype()), scratch ? scratch->data() : nullptr, need, stream));
        return;   // the scratch goes to later calls on this stream, whose order keeps it valid for this launch
    }
    const size_t need = nvk::decode_mma_workspace_needed(batch, heads, num_kv_heads, head_dim, max_blocks, block_size);
    if (need > 0 && need <= nvk_decode_attention_static_scratch_bytes()) {
        throw_on_nvk_status(nvk_decode_attention_paged_static(query.data(), k_cache.data(), v_cache.data(), lens.ptr,
                                                              lens.dtype, tables.ptr, tables.dtype, batch, max_blocks,
                                                              blocks, heads, num_kv_heads, head_dim, block_size, scale,
                                                              output.data(), code(query.dtype()), stream));
        return;
    }
    throw_on_nvk_status(nvk_decode_attention_paged(query.data(), k_cache.data(), v_cache.data(), lens.ptr, lens.dtype,
                                                   tables.ptr, tables.dtype, batch, max_blocks, blocks, heads, num_kv_heads,
                                                   head_dim, block_size, scale, output.data(), code(query.dtype()), nullptr,
                                                   0, stream));
}

}  // namespace

void launch_decode_attention_paged(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                                   const Tensor& context_lens, const Tensor& block_tables, int num_kv_heads, int head_dim,
                                   int block_size, float scale, Tensor& output, cudaStream_t stream) {
    decode_common(query, k_cache, v_cache, context_lens, block_tables, num_kv_heads, head_dim, block_size, scale, output,
                  nullptr, stream);
}

void flash_attn_decode_kvcache(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                               const Tensor& context_lens, const Tensor& block_tables, int num_kv_heads, int head_dim,
                               int block_size, float scale, Tensor& output, DeviceAllocator& allocator,
                               cudaStream_t stream) {
    decode_common(query, k_cache, v_cache, context_lens, block_tables, num_kv_heads, head_dim, block_size, scale, output,
                  &allocator, stream);
}

void launch_decode_attention_paged_int8(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                                        const Tensor& k_scale, const Tensor& v_scale, const Tensor& context_lens,
                                        const Tensor& block_tables, int num_kv_heads, int head_dim, int block_size,
                                        float scale, Tensor& output, cudaStream_t stream) {
    check_qo(query, output);
    validate_supported_dtype("query", query.dtype());
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_cuda_tensor("k_scale", k_scale);
    ensure_cuda_tensor("v_scale", v_scale);
    ensure_cuda_tensor("context_lens", context_lens);
    ensure_cuda_tensor("block_tables", block_tables);
    if (k_cache.dtype() != ScalarType::kInt8 || v_cache.dtype() != ScalarType::kInt8)
        throw std::invalid_argument("int8 decode attention requires int8 caches");
    if (k_scale.dtype() != ScalarType::kFloat16 || v_scale.dtype() != ScalarType::kFloat16)
        throw std::invalid_argument("int8 decode attention requires float16 scales");
    const IndexRef lens = index_data("context_lens", context_lens);
    const IndexRef tables = index_data("block_tables", block_tables);
    if (block_tables.dim() != 2 || block_tables.sizes()[0] != query.sizes()[0])
        throw std::invalid_argument("block_tables must be [batch, max_blocks]");
    if (static_cast<int64_t>(context_lens.numel()) != query.sizes()[0])
        throw std::invalid_argument("context_lens must hold one entry per sequence");
    if (query.sizes()[2] != head_dim) throw std::invalid_argument("query head_dim does not match head_dim");
    const int64_t batch = query.sizes()[0];
    const int heads = static_cast<int>(query.sizes()[1]);
    const int64_t max_blocks = block_tables.sizes()[1];
    const int64_t per_block = static_cast<int64_t>(block_size) * num_kv_heads * head_dim;
    if (per_block <= 0 || static_cast<int64_t>(k_cache.numel()) % per_block != 0 || k_cache.numel() != v_cache.numel())
        throw std::invalid_argument("int8 caches do not hold a whole number of blocks");
    const int64_t blocks = static_cast<int64_t>(k_cache.numel()) / per_block;
    if (static_cast<int64_t>(k_scale.numel()) != blocks * block_size * num_kv_heads || k_scale.numel() != v_scale.numel())
        throw std::invalid_argument("k_scale and v_scale must hold one value per cache row and KV head");
    // no allocator in this signature (as in the reference): the call runs without split-K scratch
    throw_on_nvk_status(nvk_decode_attention_paged_int8(
        query.data(), k_cache.data(), v_cache.data(), k_scale.data(), v_scale.data(), lens.ptr, lens.dtype, tables.ptr,
        tables.dtype, batch, max_blocks, blocks, heads, num_kv_heads, head_dim, block_size, scale, output.data(), code(query.dtype()), nullptr, 0, stream));
}

namespace {

// The tensors that a decode step over a 16-bit or 4-bit cache has.
struct Step {
    IndexRef lens, tables;
    int64_t batch, max_blocks, blocks;
    int heads;
    Step(const Tensor& query, const Tensor& output, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_params, const Tensor& v_params, bool four,
         const Tensor& context_lens, const Tensor& block_tables, int num_kv_heads, int head_dim, int block_size)
        : lens(index_data("context_lens", context_lens)), tables(index_data("block_tables", block_tables)) {
        check_qo(query, output);
        if (num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0) throw std::invalid_argument("attention dimensions must be positive");
        batch = query.sizes()[0];
        heads = static_cast<int>(query.sizes()[1]);
        if (query.sizes()[2] != head_dim) throw std::invalid_argument("query head_dim does not match head_dim");
        if (block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [batch, max_blocks]");
        ensure_rows("block_tables", block_tables, batch);
        if (static_cast<int64_t>(context_lens.numel()) != batch) throw std::invalid_argument("context_lens must hold one entry per sequence");
        max_blocks = block_tables.sizes()[1];
        if (four) {
            blocks = int4_rows(k_cache, v_cache, k_params, v_params, query.dtype(), num_kv_heads, head_dim) / block_size;
        } else {
            ensure_cuda_tensor("k_cache", k_cache);
            ensure_cuda_tensor("v_cache", v_cache);
            ensure_same_dtype("query", query, "k_cache", k_cache);
            ensure_same_dtype("query", query, "v_cache", v_cache);
            if (k_cache.numel() != v_cache.numel()) throw std::invalid_argument("k_cache and v_cache must contain the same number of slots");
            blocks = cache_blocks(k_cache, block_size, num_kv_heads, head_dim);
        }
        ensure_same_device("query", query, "k_cache", k_cache);
        ensure_same_device("query", query, "v_cache", v_cache);
        ensure_same_device("query", query, "context_lens", context_lens);
        ensure_same_device("query", query, "block_tables", block_tables);
    }
};

}  // namespace

void launch_decode_attention_paged_int4(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                                        const Tensor& k_params, const Tensor& v_params, const Tensor& context_lens,
                                        const Tensor& block_tables, int num_kv_heads, int head_dim, int block_size,
                                        float scale, Tensor& output, DeviceAllocator& allocator, cudaStream_t stream) {
    const Step s(query, output, k_cache, v_cache, k_params, v_params, true, context_lens, block_tables, num_kv_heads, head_dim, block_size);
    const size_t need = nvk::decode_mma_workspace_needed(s.batch, s.heads, num_kv_heads, head_dim, s.max_blocks, block_size);
    Memory::Ptr scratch = need > 0 ? allocator.allocate_on(need, query.device(), stream) : nullptr;
    throw_on_nvk_status(nvk_decode_attention_paged_int4(query.data(), k_cache.data(), v_cache.data(), k_params.data(), v_params.data(), s.lens.ptr, s.lens.dtype,
                                                        s.tables.ptr, s.tables.dtype, s.batch, s.max_blocks, s.blocks, s.heads, num_kv_heads, head_dim,
                                                        block_size, scale, output.data(), code(query.dtype()), scratch ? scratch->data() : nullptr, need, stream));
}

void launch_decode_attention_paged_blocks8(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                                           const Tensor& k_scale, const Tensor& v_scale, const Tensor& context_lens,
                                           const Tensor& block_tables, float scale, Tensor& output, DeviceAllocator& allocator, bool e4m3,
                                           cudaStream_t stream) {
    const Blocks8 c(k_cache, v_cache, k_scale, v_scale, e4m3);
    check_qo(query, output);
    const IndexRef lens = index_data("context_lens", context_lens), tables = index_data("block_tables", block_tables);
    const int64_t batch = query.sizes()[0];
    const int heads = static_cast<int>(query.sizes()[1]);
    if (query.sizes()[2] != c.head_dim) throw std::invalid_argument("query head_dim does not match that of the cache");
    if (heads % c.heads != 0 || heads / c.heads > 8) throw std::invalid_argument("num_heads must be divisible by num_kv_heads, and at most 8 times as many");
    if (!std::isfinite(scale)) throw std::invalid_argument("scale must be finite");
    if (block_tables.dim() != 2) throw std::invalid_argument("block_tables must be [batch, max_blocks]");
    ensure_rows("block_tables", block_tables, batch);
    if (static_cast<int64_t>(context_lens.numel()) != batch) throw std::invalid_argument("context_lens must hold one entry per sequence");
    ensure_same_device("query", query, "k_cache", k_cache);
    ensure_same_device("query", query, "context_lens", context_lens);
    ensure_same_device("query", query, "block_tables", block_tables);
    const int64_t max_blocks = block_tables.sizes()[1];
    // (more than this call needs: with room for them, contexts go into shorter parts)
    const size_t room = nvk_decode_attention_workspace_bytes(batch, heads, c.heads, c.head_dim, max_blocks, c.block_size);
    Memory::Ptr scratch = room > 0 ? allocator.allocate_on(room, query.device(), stream) : nullptr;
    throw_on_nvk_status(nvk_decode_attention_paged_blocks8(query.data(), k_cache.data(), v_cache.data(), k_scale.data_as<float>(), v_scale.data_as<float>(), c.type,
                                                           lens.ptr, lens.dtype, tables.ptr, tables.dtype, batch, max_blocks, c.blocks, heads, c.heads, c.head_dim,
                                                           c.block_size, scale, output.data(), code(query.dtype()), scratch ? scratch->data() : nullptr, room, stream));
}

void launch_decode_attention_paged_weights(const Tensor& query, const Tensor& k_cache, const Tensor& v_cache,
                                           const Tensor& k_params, const Tensor& v_params, const Tensor& context_lens,
                                           const Tensor& block_tables, int num_kv_heads, int head_dim, int block_size,
                                           float scale, const Tensor& key_weights, const Tensor& weight_rows,
                                           Tensor& new_key_weights, Tensor& output, DeviceAllocator& allocator,
                                           cudaStream_t stream) {
    const bool four = k_params.defined() || v_params.defined();
    const Step s(query, output, k_cache, v_cache, k_params, v_params, four, context_lens, block_tables, num_kv_heads, head_dim, block_size);
    ensure_cuda_tensor("new_key_weights", new_key_weights);
    if (new_key_weights.dtype() != ScalarType::kFloat32 || new_key_weights.dim() != 3 || new_key_weights.sizes()[1] != num_kv_heads)
        throw std::invalid_argument("new_key_weights must be float32 [rows, num_kv_heads, keys]");
    if (key_weights.defined()) {
        ensure_cuda_tensor("key_weights", key_weights);
        ensure_same_dtype("key_weights", key_weights, "new_key_weights", new_key_weights);
        ensure_same_shape("key_weights", key_weights, "new_key_weights", new_key_weights);
        ensure_same_device("query", query, "key_weights", key_weights);
    }
    ensure_same_device("query", query, "new_key_weights", new_key_weights);
    const IndexRef rows = weight_rows.defined() ? index_data("weight_rows", weight_rows) : IndexRef{nullptr, NVK_I32};
    if (weight_rows.defined()) {
        ensure_rows("weight_rows", weight_rows, s.batch);
        ensure_same_device("query", query, "weight_rows", weight_rows);
    }
    const size_t need = nvk_decode_attention_weights_workspace_bytes(s.batch, s.heads, num_kv_heads, head_dim, s.max_blocks, block_size);
    Memory::Ptr scratch = need > 0 ? allocator.allocate_on(need, query.device(), stream) : nullptr;
    throw_on_nvk_status(nvk_decode_attention_paged_weights(
        query.data(), k_cache.data(), v_cache.data(), four ? k_params.data() : nullptr, four ? v_params.data() : nullptr, s.lens.ptr, s.lens.dtype, s.tables.ptr,
        s.tables.dtype, s.batch, s.max_blocks, s.blocks, s.heads, num_kv_heads, head_dim, block_size, scale,
        key_weights.defined() ? key_weights.data_as<float>() : nullptr, rows.ptr, rows.dtype, new_key_weights.sizes()[0], new_key_weights.sizes()[2],
        new_key_weights.data_as<float>(), output.data(), code(query.dtype()), scratch ? scratch->data() : nullptr, need, stream));
}

// ---- prefill ------------------------------------------------------------------------------------------
void launch_prefill_attention_dense(const Tensor& query, const Tensor* cu_seqlens_q, const Tensor& key,
                                    const Tensor& value, const Tensor* cu_seqlens_k, int num_kv_heads, int head_dim,
                                    float scale, Tensor& output, cudaStream_t stream, int max_seqlen_q) {
    check_qo(query, output);
    ensure_cuda_tensor("key", key);
    ensure_cuda_tensor("value", value);
    ensure_same_dtype("query", query, "key", key);
    ensure_same_dtype("query", query, "value", value);
    const bool varlen = cu_seqlens_q != nullptr && cu_seqlens_k != nullptr;   // either missing: one sequence
    const IndexRef cq = varlen ? index_data("cu_seqlens_q", *cu_seqlens_q) : IndexRef{nullptr, NVK_I32};
    const IndexRef ck = varlen ? index_data("cu_seqlens_k", *cu_seqlens_k) : IndexRef{nullptr, NVK_I32};
    const int64_t seqs = varlen ? static_cast<int64_t>(cu_seqlens_q->numel()) - 1 : 1;
    throw_on_nvk_status(nvk_prefill_attention_varlen(query.data(), key.data(), value.data(), nullptr, nullptr, cq.ptr,
                                                     cq.dtype, ck.ptr, ck.dtype, nullptr, NVK_I32, seqs, query.sizes()[0],
                                                     key.sizes()[0], 0, 0, max_seqlen_q,
                                                     static_cast<int>(query.sizes()[1]), num_kv_heads, head_dim, 1, scale,
                                                     output.data(), code(query.dtype()), stream));
}

void launch_prefill_attention_dense(const Tensor& query, const Tensor* cu_seqlens_q, const Tensor& key,
                                    const Tensor& value, const Tensor* cu_seqlens_k, int num_kv_heads, int head_dim,
                                    float scale, Tensor& output, cudaStream_t stream) {
    launch_prefill_attention_dense(query, cu_seqlens_q, key, value, cu_seqlens_k, num_kv_heads, head_dim, scale, output, stream, 0);
}

void launch_prefill_attention_paged(const Tensor& query, const Tensor* cu_seqlens_q, const Tensor& k_cache,
                                    const Tensor& v_cache, const Tensor* cu_seqlens_k, const Tensor& block_tables,
                                    int num_kv_heads, int head_dim, int block_size, float scale, Tensor& output,
                                    cudaStream_t stream, int max_seqlen_q) {
    if (cu_seqlens_q == nullptr || cu_seqlens_k == nullptr)
        throw std::invalid_argument("paged prefill attention requires cu_seqlens_q and cu_seqlens_k");
    check_qo(query, output);
    ensure_cuda_tensor("k_cache", k_cache);
    ensure_cuda_tensor("v_cache", v_cache);
    ensure_same_dtype("query", query, "k_cache", k_cache);
    if (block_tables.defined() && block_tables.dim() != 2)
        throw std::invalid_argument("block_tables must be [num_seqs, max_blocks]");
    const IndexRef tables = index_data("block_tables", block_tables);
    const IndexRef cq = index_data("cu_seqlens_q", *cu_seqlens_q), ck = index_data("cu_seqlens_k", *cu_seqlens_k);
    throw_on_nvk_status(nvk_prefill_attention_varlen(
        query.data(), nullptr, nullptr, k_cache.data(), v_cache.data(), cq.ptr, cq.dtype, ck.ptr, ck.dtype, tables.ptr,
        tables.dtype, static_cast<int64_t>(cu_seqlens_q->numel()) - 1,
        query.sizes()[0], 0, block_tables.sizes()[1], cache_blocks(k_cache, block_size, num_kv_heads, head_dim), max_seqlen_q,
        static_cast<int>(query.sizes()[1]), num_kv_heads, head_dim, block_size, scale, output.data(),
        code(query.dtype()), stream));
}

void launch_prefill_attention_paged(const Tensor& query, const Tensor* cu_seqlens_q, const Tensor& k_cache,
                                    const Tensor& v_cache, const Tensor* cu_seqlens_k, const Tensor& block_tables,
                                    int num_kv_heads, int head_dim, int block_size, float scale, Tensor& output,
                                    cudaStream_t stream) {
    launch_prefill_attention_paged(query, cu_seqlens_q, k_cache, v_cache, cu_seqlens_k, block_tables, num_kv_heads, head_dim, block_size, scale,
                                   output, stream, 0);
}

void throw_if_prefill_error(cudaStream_t stream) {
    int word = 0;
    throw_on_nvk_status(nvk_prefill_status(stream, &word));
    if (word != 0)
        throw std::runtime_error("prefill attention: a bounded wait inside the tensor-core kernel ran out (code " +
                                 std::to_string(word) + "); output rows of that launch are incomplete");
}

bool flash_attn_available() { return true; }

void flash_attn_varlen_fwd(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& cu_seqlens_q,
                           const Tensor& cu_seqlens_k, int max_seqlen_q, int /*max_seqlen_k*/, float scale,
                           bool is_causal, Tensor& output, DeviceAllocator& /*allocator*/, cudaStream_t stream) {
    if (!is_causal) throw std::invalid_argument("unsupported: non-causal varlen attention");
    const int num_kv_heads = key.defined() && key.dim() == 3 ? static_cast<int>(key.sizes()[1]) : 0;
    const int head_dim = query.defined() && query.dim() == 3 ? static_cast<int>(query.sizes()[2]) : 0;
    launch_prefill_attention_dense(query, &cu_seqlens_q, key, value, &cu_seqlens_k, num_kv_heads, head_dim, scale, output,
                                   stream, max_seqlen_q);
}

}  // namespace nano_vllm
