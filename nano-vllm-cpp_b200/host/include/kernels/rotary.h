// Rotary positions (not in the reference, whose rotation is part of the fused prologue: include/kernels/split_qkv.h).
#pragma once

#include "utils/tensor.h"

#include <vector>

namespace nano_vllm {

// The first 2 * inv_freq.numel() elements of every head: pairs of halves, or of neighbours if `interleaved`; the others are copied.  query and key (undefined: queries
// alone) are [rows, heads, head_dim], or rows [rows, heads * head_dim] that may be slices of packed ones; query_out and key_out likewise, and may be their inputs.
// inv_freq: float32 on the device; positions: int32 / int64, any.
void rotary_embedding(const Tensor& query, const Tensor& key, const Tensor& positions, const Tensor& inv_freq, int num_q_heads,
                      int num_kv_heads, int head_dim, bool interleaved, float attention_factor, Tensor& query_out,
                      Tensor& key_out, cudaStream_t stream = nullptr);

enum class RopeScaling { kPlain, kLinear, kBase, kParts, kYarn };   // (the order of NVK_ROPE_*)

struct RotaryFrequencies {
    std::vector<float> inv_freq;
    float attention_factor = 1.0f;
};
// For a context stretched by `factor` beyond original_positions (nvk_rotary_inv_freq has the formulas).
RotaryFrequencies rotary_inv_freq(int rotary_dim, double base, RopeScaling scaling = RopeScaling::kPlain, double factor = 1.0,
                                  double original_positions = 0.0, double low_turns = 1.0, double high_turns = 32.0);

}  // namespace nano_vllm
