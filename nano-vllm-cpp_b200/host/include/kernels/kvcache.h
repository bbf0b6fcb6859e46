// store_kvcache operator (signature of include/kernels/kvcache.h:7-12 of the reference).
#pragma once

#include "utils/tensor.h"

namespace nano_vllm {

// cache row slot_mapping[t] <- key / value row t; slots < 0 or beyond the cache are skipped.
void store_kvcache(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache,
                   const Tensor& slot_mapping, cudaStream_t stream = nullptr);

// int8 KV cache (include/kernels/kvcache.h:14-24 of the reference): key / value [tokens, Hkv, D] are quantised per
// (token, KV head) into int8 caches [.., Hkv, D] with one fp16 scale each in k_scale / v_scale [.., Hkv].
void store_kvcache_int8(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_scale,
                        Tensor& v_scale, const Tensor& slot_mapping, cudaStream_t stream = nullptr);

// 4-bit KV cache (not in the reference): key / value [tokens, Hkv, 128], F16 / BF16, are quantised per (token, KV head) into byte caches
// (int8 tensors) [.., Hkv, 64] with a pair (step, low) each in k_params / v_params [.., Hkv, 2] of the keys' type.
void store_kvcache_int4(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_params,
                        Tensor& v_params, const Tensor& slot_mapping, cudaStream_t stream = nullptr);
// Whole contexts of a 4-bit cache as dense rows: key / value [total_k, Hkv, 128], sequence after sequence by cu_seqlens_k; rows behind the
// last one become zeros.
void gather_kvcache_int4(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_params, const Tensor& v_params,
                         const Tensor& cu_seqlens_k, const Tensor& block_tables, int num_kv_heads, int head_dim,
                         int block_size, Tensor& key, Tensor& value, cudaStream_t stream = nullptr);

// 8-bit KV cache with one scale for each cache block and KV head (not in the reference): byte caches (int8 tensors; `e4m3`: their elements are e4m3) [blocks, block_size, Hkv, 128]
// with float32 scales [blocks, Hkv].  The store goes by sequences: rows cu_seqlens_q[s] on of key / value [tokens, Hkv, 128], F16 / BF16, are the last of the context_lens[s]
// positions of sequence s; cu_seqlens_q undefined: one row for every sequence.  key and value may be parts of packed rows (slices of the last dimension, [tokens, Hkv * 128]).
void store_kvcache_blocks8(const Tensor& key, const Tensor& value, Tensor& k_cache, Tensor& v_cache, Tensor& k_scale,
                           Tensor& v_scale, const Tensor& cu_seqlens_q, const Tensor& context_lens,
                           const Tensor& block_tables, bool e4m3 = false, cudaStream_t stream = nullptr);
// Whole contexts of such a cache as dense rows, as gather_kvcache_int4.
void gather_kvcache_blocks8(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                            const Tensor& cu_seqlens_k, const Tensor& block_tables, Tensor& key, Tensor& value,
                            bool e4m3 = false, cudaStream_t stream = nullptr);

// Eviction by accumulated attention weight (not in the reference): of every sequence and KV head the first `sinks` keys, the last `recent` and the
// heaviest between them stay, `budget` in all, and close up in the blocks of new_block_tables (which may be block_tables).  Undefined k_params / v_params: a
// 16-bit cache; undefined weight_rows: sequence b has row b of key_weights [rows, Hkv, keys] (float32; new_key_weights may be the same tensor).
void evict_kvcache(Tensor& k_cache, Tensor& v_cache, Tensor& k_params, Tensor& v_params, const Tensor& key_weights,
                   const Tensor& weight_rows, const Tensor& context_lens, const Tensor& block_tables, Tensor& new_key_weights,
                   const Tensor& new_block_tables, Tensor& new_context_lens, int num_kv_heads, int head_dim, int block_size,
                   int64_t budget, int64_t sinks, int64_t recent, cudaStream_t stream = nullptr);

}  // namespace nano_vllm
