// Refusals of the 8-bit cache with block scales, of the rotary positions and of the step metadata in the C++ layer: what is wrong is thrown before any CUDA call, so that no
// GPU is needed (device tensors here are borrowed addresses that nothing reads).
#include "check.h"

#include "engine/step_metadata.h"
#include "kernels/attention.h"
#include "kernels/kvcache.h"
#include "kernels/rotary.h"
#include "layers/attention.h"
#include "utils/context.h"
#include "utils/cuda_allocator.h"

#include <stdexcept>

using namespace nano_vllm;

namespace {

class NoAllocator : public DeviceAllocator {
public:
    Memory::Ptr allocate(size_t, Device) override { throw std::logic_error("nothing may be allocated here"); }
    void memset_async(void*, int, size_t, cudaStream_t) const override {}
    void copy_to_device_async(void*, const void*, size_t, cudaStream_t) const override {}
    void copy_to_host_async(void*, const void*, size_t, cudaStream_t) const override {}
    void synchronize_stream(cudaStream_t) const override {}
};

Tensor borrowed(const std::vector<int64_t>& sizes, ScalarType type, DeviceType where = DeviceType::kCUDA, int device = 0) {
    static uintptr_t next = 0x100000;   // (no two alike)
    next += 0x100000;
    const size_t bytes = compute_numel(sizes) * scalar_type_size(type);
    return Tensor::from_memory(Memory::make_borrowed(reinterpret_cast<void*>(next), bytes, Device{where, device}), sizes, type);
}

struct Case {
    Tensor key = borrowed({3, 2, 128}, ScalarType::kBFloat16), k_cache = borrowed({4, 16, 2, 128}, ScalarType::kInt8), v_cache = borrowed({4, 16, 2, 128}, ScalarType::kInt8),
           scale = borrowed({4, 2}, ScalarType::kFloat32), cu = borrowed({3}, ScalarType::kInt32), lens = borrowed({2}, ScalarType::kInt32),
           tables = borrowed({2, 2}, ScalarType::kInt32), query = borrowed({2, 4, 128}, ScalarType::kBFloat16), output = borrowed({2, 4, 128}, ScalarType::kBFloat16), none;
    NoAllocator alloc;
};

}  // namespace

TEST_CASE(store_and_gather_refuse) {
    Case c;
    Tensor host = borrowed({3, 2, 128}, ScalarType::kBFloat16, DeviceType::kCPU), floats = borrowed({3, 2, 128}, ScalarType::kFloat32), few = borrowed({3, 2}, ScalarType::kFloat32),
           half = borrowed({4, 2}, ScalarType::kFloat16), three = borrowed({3}, ScalarType::kInt32), heads = borrowed({3, 4, 128}, ScalarType::kBFloat16),
           other = borrowed({2}, ScalarType::kInt32, DeviceType::kCUDA, 1), wide = borrowed({3, 1024}, ScalarType::kBFloat16), flat = borrowed({64, 2, 128}, ScalarType::kInt8);
    auto store = [&](const Tensor& k, Tensor& cache, Tensor& scale, const Tensor& cu, const Tensor& lens, const Tensor& tables) {
        store_kvcache_blocks8(k, k, cache, cache, scale, scale, cu, lens, tables);
    };
    CHECK_THROWS(store(host, c.k_cache, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(floats, c.k_cache, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(heads, c.k_cache, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.key, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, flat, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, few, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, half, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, c.scale, c.lens, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, c.scale, c.none, c.lens, c.tables), std::invalid_argument);   // three rows, two sequences
    CHECK_THROWS(store(c.key, c.k_cache, c.scale, c.cu, c.none, c.tables), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, c.scale, c.cu, c.lens, c.lens), std::invalid_argument);
    CHECK_THROWS(store(c.key, c.k_cache, c.scale, c.cu, other, c.tables), std::invalid_argument);
    CHECK_THROWS(store(wide, c.k_cache, c.scale, c.cu, c.lens, c.tables), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_blocks8(c.k_cache, c.v_cache, c.scale, c.scale, c.lens, c.tables, c.key, c.key), std::invalid_argument);   // one sequence, two rows
    CHECK_THROWS(gather_kvcache_blocks8(c.k_cache, c.v_cache, c.scale, c.scale, c.cu, c.tables, floats, floats), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_blocks8(c.k_cache, c.v_cache, c.scale, c.scale, c.cu, c.tables, heads, heads), std::invalid_argument);
}

TEST_CASE(decode_refuses) {
    Case c;
    Tensor one = borrowed({1}, ScalarType::kInt32), nine = borrowed({2, 18, 128}, ScalarType::kBFloat16), nine_out = borrowed({2, 18, 128}, ScalarType::kBFloat16),
           half = borrowed({2, 4, 64}, ScalarType::kBFloat16), half_out = borrowed({2, 4, 64}, ScalarType::kBFloat16);
    CHECK_THROWS(launch_decode_attention_paged_blocks8(c.query, c.k_cache, c.v_cache, c.scale, c.scale, one, c.tables, 1.0f, c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_blocks8(half, c.k_cache, c.v_cache, c.scale, c.scale, c.lens, c.tables, 1.0f, half_out, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_blocks8(nine, c.k_cache, c.v_cache, c.scale, c.scale, c.lens, c.tables, 1.0f, nine_out, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_blocks8(c.query, c.k_cache, c.v_cache, c.scale, c.scale, c.lens, c.tables, INFINITY, c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_blocks8(c.query, c.k_cache, c.v_cache, c.none, c.scale, c.lens, c.tables, 1.0f, c.output, c.alloc), std::invalid_argument);
}

TEST_CASE(the_layer_refuses) {
    Case c;
    Attention attention(4, 2, 128, 16), wide(4, 2, 64, 16);
    Tensor few = borrowed({3, 2}, ScalarType::kFloat32), half = borrowed({4, 2}, ScalarType::kFloat16), blocks = borrowed({4, 32, 2, 128}, ScalarType::kInt8);
    CHECK_THROWS(attention.set_kv_cache_blocks8(c.key, c.key, c.scale, c.scale), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_blocks8(c.k_cache, c.v_cache, few, few), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_blocks8(c.k_cache, c.v_cache, half, half), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_blocks8(blocks, blocks, c.scale, c.scale), std::invalid_argument);
    CHECK_THROWS(wide.set_kv_cache_blocks8(c.k_cache, c.v_cache, c.scale, c.scale), std::invalid_argument);
    attention.set_kv_cache_blocks8(c.k_cache, c.v_cache, c.scale, c.scale);
    CHECK(attention.is_blocks8() && attention.is_quantised() && !attention.is_int8() && !attention.is_int4());
    // a prefill whose context has no lengths of contexts
    const Tensor q = borrowed({3, 4, 128}, ScalarType::kBFloat16);
    set_context(true, c.cu, c.cu, 2, 2, borrowed({3}, ScalarType::kInt32), Tensor(), c.tables);
    CHECK_THROWS(attention.forward(q, c.key, c.key, c.alloc), std::invalid_argument);
    attention.set_key_weights(borrowed({2, 2, 32}, ScalarType::kFloat32));
    set_context(false, Tensor(), Tensor(), 0, 0, Tensor(), c.lens, c.tables);
    CHECK_THROWS(attention.forward_decode_flash_only(c.query, c.alloc), std::logic_error);   // (nothing may be allocated: the output comes first)
    reset_context();
    const Tensor full = borrowed({4, 16, 2, 128}, ScalarType::kBFloat16);
    attention.set_kv_cache(full, full);
    CHECK(!attention.is_quantised());
}

TEST_CASE(rotary_refuses) {
    Tensor q = borrowed({3, 4, 128}, ScalarType::kBFloat16), k = borrowed({3, 2, 128}, ScalarType::kBFloat16), pos = borrowed({3}, ScalarType::kInt32),
           f = borrowed({64}, ScalarType::kFloat32), half = borrowed({64}, ScalarType::kFloat16), few = borrowed({2}, ScalarType::kInt32), none, many = borrowed({65}, ScalarType::kFloat32),
           other = borrowed({3, 4, 128}, ScalarType::kFloat16), rows = borrowed({2, 4, 128}, ScalarType::kBFloat16);
    auto rotate = [&](Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& f, Tensor& q_out, Tensor& k_out, int heads = 4) {
        rotary_embedding(q, k, pos, f, heads, 2, 128, false, 1.0f, q_out, k_out);
    };
    CHECK_THROWS(rotate(q, k, pos, half, q, k), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, few, f, q, k), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, pos, many, q, k), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, pos, f, q, none), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, pos, f, other, k), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, pos, f, rows, k), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, pos, f, q, k, 8), std::invalid_argument);
    CHECK_THROWS(rotate(q, k, f, f, q, k), std::invalid_argument);
    CHECK_THROWS(rotary_inv_freq(7, 1e4), std::invalid_argument);
    CHECK_THROWS(rotary_inv_freq(0, 1e4), std::invalid_argument);
    CHECK_THROWS(rotary_inv_freq(8, 1e4, RopeScaling::kYarn, 4.0), std::invalid_argument);
    const RotaryFrequencies plain = rotary_inv_freq(4, 1e4), yarn = rotary_inv_freq(4, 1e4, RopeScaling::kYarn, 4.0, 100.0, 1.0, 2.0);
    CHECK(plain.inv_freq.size() == 2 && plain.inv_freq[0] == 1.0f);
    CHECK_NEAR(plain.inv_freq[1], 0.01, 1e-9);
    CHECK(yarn.inv_freq[0] == 1.0f);   // 100 / 2 pi turns
    CHECK_NEAR(yarn.inv_freq[1], 0.0025, 1e-9);
    CHECK_NEAR(yarn.attention_factor, 0.1 * std::log(4.0) + 1.0, 1e-6);
}

TEST_CASE(step_refuses) {
    auto i32 = [](const std::vector<int64_t>& s) { return borrowed(s, ScalarType::kInt32); };
    RequestTables t{i32({4}), i32({4, 8}), i32({30}), i32({1}), 16, 32};
    DeviceStep s{i32({2, 8}), i32({2}), i32({3}), i32({3}), i32({10}), i32({10})};
    const Tensor n = i32({2}), none, wide = borrowed({2}, ScalarType::kInt64);
    auto with_tables = [&](auto change) { RequestTables x = t; change(x); build_step(n, none, x, s); };
    auto with_step = [&](auto change) { DeviceStep x = s; change(x); build_step(n, none, t, x); };
    CHECK_THROWS(build_step(none, none, t, s), std::invalid_argument);
    CHECK_THROWS(build_step(wide, none, t, s), std::invalid_argument);
    CHECK_THROWS(build_step(n, i32({3}), t, s), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.lens = i32({5}); }), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.free_count = i32({2}); }), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.free_blocks = borrowed({30}, ScalarType::kInt64); }), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.blocks = borrowed({4, 8}, ScalarType::kInt32, DeviceType::kCUDA, 1); }), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.block_size = 0; }), std::invalid_argument);
    CHECK_THROWS(with_tables([&](RequestTables& x) { x.num_cache_blocks = 0; }), std::invalid_argument);
    CHECK_THROWS(with_step([&](DeviceStep& x) { x.block_tables = i32({3, 8}); }), std::invalid_argument);
    CHECK_THROWS(with_step([&](DeviceStep& x) { x.context_lens = none; }), std::invalid_argument);
    CHECK_THROWS(with_step([&](DeviceStep& x) { x.cu_seqlens_q = i32({2}); }), std::invalid_argument);
    CHECK_THROWS(with_step([&](DeviceStep& x) { x.slot_mapping = none; }), std::invalid_argument);
    CHECK_THROWS(with_step([&](DeviceStep& x) { x.slot_mapping = i32({9}); }), std::invalid_argument);
    CHECK_THROWS(release_blocks(none, i32({3}), t), std::invalid_argument);
    CHECK_THROWS(release_blocks(wide, none, t), std::invalid_argument);
}

TEST_CASE(prefill_arrays_by_sequences) {
    // Blocks of 4: a prompt of 6, one of 8 of which 4 are cached, one that is cached whole, the chunk [5, 7) of one of 9.
    std::vector<int32_t> tokens(9, 1);
    auto view = [&](int n, const std::vector<int32_t>& table, int cached, int computed = 0, int chunk = 0) {
        SequenceView s;
        s.token_ids = tokens.data();
        s.num_tokens = n;
        s.num_cached_tokens = cached;
        s.num_computed_tokens = computed;
        s.num_tokens_to_process = chunk;
        s.block_table = table.data();
        s.block_table_len = static_cast<int32_t>(table.size());
        return s;
    };
    const std::vector<int32_t> a = {3, 1}, b = {5, 6}, c = {5, 7}, d = {0, 2, 4};
    const StepArrays x = build_prefill_arrays({view(6, a, 0), view(8, b, 4), view(8, c, 8), view(9, d, 4, 5, 2)}, 4, true);
    CHECK_EQ(x.cu_seqlens_q, (std::vector<int32_t>{0, 6, 10, 11, 13}));
    CHECK_EQ(x.cu_seqlens_k, (std::vector<int32_t>{0, 6, 14, 22, 29}));
    CHECK_EQ(x.context_lens, (std::vector<int32_t>{6, 8, 0, 7}));
    CHECK_EQ(x.max_blocks, int64_t(3));
    CHECK_EQ(x.block_tables, (std::vector<int32_t>{3, 1, 0, 5, 6, 0, 5, 7, 0, 0, 2, 4}));
    // without a cached key too; and nothing of it unless asked for
    const StepArrays fresh = build_prefill_arrays({view(6, a, 0)}, 4, true), slots = build_prefill_arrays({view(6, a, 0)}, 4);
    CHECK_EQ(fresh.context_lens, (std::vector<int32_t>{6}));
    CHECK_EQ(fresh.block_tables, a);
    CHECK(slots.context_lens.empty() && slots.block_tables.empty());
    CHECK_THROWS(build_prefill_arrays({view(9, d, 4, 2, 5)}, 4, true), std::invalid_argument);
    CHECK_EQ(build_prefill_arrays({view(9, d, 4, 2, 5)}, 4).positions.front(), 2);
}

int main() { return check::run_all(); }
