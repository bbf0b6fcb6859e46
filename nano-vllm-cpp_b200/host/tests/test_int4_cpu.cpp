// Refusals of the 4-bit cache's operators, of the key weights and of eviction in the C++ layer: what is wrong is thrown before any CUDA call, so that no GPU is
// needed (device tensors here are borrowed addresses that nothing reads).
#include "check.h"

#include "kernels/attention.h"
#include "kernels/flash_attn.h"
#include "kernels/kvcache.h"
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

Tensor borrowed(const std::vector<int64_t>& sizes, ScalarType type, DeviceType where = DeviceType::kCUDA) {
    static uintptr_t next = 0x100000;   // (no two alike)
    next += 0x100000;
    const size_t bytes = compute_numel(sizes) * scalar_type_size(type);
    return Tensor::from_memory(Memory::make_borrowed(reinterpret_cast<void*>(next), bytes, Device{where, 0}), sizes, type);
}

struct Case {
    Tensor key = borrowed({3, 2, 128}, ScalarType::kBFloat16), k_cache = borrowed({2, 16, 2, 64}, ScalarType::kInt8), v_cache = borrowed({2, 16, 2, 64}, ScalarType::kInt8),
           params = borrowed({2, 16, 2, 2}, ScalarType::kBFloat16), slots = borrowed({3}, ScalarType::kInt64), query = borrowed({1, 4, 128}, ScalarType::kBFloat16),
           output = borrowed({1, 4, 128}, ScalarType::kBFloat16), lens = borrowed({1}, ScalarType::kInt32), tables = borrowed({1, 2}, ScalarType::kInt32),
           weights = borrowed({1, 2, 32}, ScalarType::kFloat32), none;
    NoAllocator alloc;
};

}  // namespace

TEST_CASE(store_and_gather_refuse) {
    Case c;
    Tensor host = borrowed({3, 2, 128}, ScalarType::kBFloat16, DeviceType::kCPU), floats = borrowed({3, 2, 128}, ScalarType::kFloat32),
           half_params = borrowed({2, 16, 2, 2}, ScalarType::kFloat16), few = borrowed({16, 2, 2}, ScalarType::kBFloat16), two = borrowed({2}, ScalarType::kInt32),
           wide = borrowed({2, 16, 2, 128}, ScalarType::kInt8), narrow = borrowed({3, 4, 64}, ScalarType::kBFloat16);
    CHECK_THROWS(store_kvcache_int4(host, host, c.k_cache, c.v_cache, c.params, c.params, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(floats, floats, c.k_cache, c.v_cache, c.params, c.params, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(narrow, narrow, c.k_cache, c.v_cache, c.params, c.params, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.k_cache, c.v_cache, half_params, half_params, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.k_cache, c.v_cache, few, few, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.k_cache, wide, c.params, c.params, c.slots), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.k_cache, c.v_cache, c.params, c.params, two), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.k_cache, c.v_cache, c.params, c.params, c.none), std::invalid_argument);
    CHECK_THROWS(store_kvcache_int4(c.key, c.key, c.key, c.key, c.params, c.params, c.slots), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, c.slots, c.tables, 2, 128, 16, c.key, c.key), std::invalid_argument);   // two sequences, one row
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, two, c.tables, 4, 128, 16, c.key, c.key), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, two, c.tables, 2, 128, 0, c.key, c.key), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, two, c.tables, 2, 128, 16, floats, floats), std::invalid_argument);
}

TEST_CASE(decode_refuses) {
    Case c;
    Tensor half = borrowed({1, 4, 128}, ScalarType::kFloat16), lens2 = borrowed({2}, ScalarType::kInt32), small = borrowed({1, 2, 31}, ScalarType::kFloat32),
           heads3 = borrowed({1, 3, 32}, ScalarType::kFloat32), odd = borrowed({1, 4, 64}, ScalarType::kBFloat16);
    CHECK_THROWS(launch_decode_attention_paged_int4(half, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, half, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_int4(c.query, c.k_cache, c.v_cache, c.params, c.params, lens2, c.tables, 2, 128, 16, 1.0f, c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_int4(odd, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, odd, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_int4(c.query, c.k_cache, c.v_cache, c.params, c.none, c.lens, c.tables, 2, 128, 16, 1.0f, c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.none, c.none, c.lens, c.tables, 2, 128, 16, 1.0f, c.none, c.none, c.weights, c.output,
                                                       c.alloc), std::invalid_argument);   // bytes are no 16-bit cache
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, small, c.none, c.weights,
                                                       c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, c.none, c.none, heads3,
                                                       c.output, c.alloc), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, c.none, lens2, c.weights,
                                                       c.output, c.alloc), std::invalid_argument);
}

TEST_CASE(evict_refuses) {
    Case c;
    Tensor new_lens = borrowed({1}, ScalarType::kInt64), lens2 = borrowed({2}, ScalarType::kInt32), new_lens32 = borrowed({1}, ScalarType::kInt32),
           host = borrowed({1, 2, 32}, ScalarType::kFloat32, DeviceType::kCPU);
    auto evict = [&](const Tensor& weights, const Tensor& lens, Tensor& to, int64_t budget, int64_t recent) {
        evict_kvcache(c.k_cache, c.v_cache, c.params, c.params, weights, c.none, lens, c.tables, c.weights, c.tables, to, 2, 128, 16, budget, 1, recent);
    };
    CHECK_THROWS(evict(c.weights, c.lens, new_lens, 8, 2), std::invalid_argument);          // another width
    CHECK_THROWS(evict(c.weights, lens2, lens2, 8, 2), std::invalid_argument);              // another batch
    CHECK_THROWS(evict(host, c.lens, new_lens32, 8, 2), std::invalid_argument);
    CHECK_THROWS(evict(c.weights, c.lens, c.lens, 8, 2), std::invalid_argument);            // the lengths over themselves
    CHECK_THROWS(evict(c.weights, c.lens, new_lens32, 0, 0), std::invalid_argument);
    CHECK_THROWS(evict(c.weights, c.lens, new_lens32, 8, 8), std::invalid_argument);        // more kept than the budget
}

TEST_CASE(evict_refuses_tensors_of_another_device) {
    Case c;
    Tensor new_lens = borrowed({1}, ScalarType::kInt32), rows = borrowed({1}, ScalarType::kInt32);
    auto elsewhere = [](uintptr_t at) {
        return Tensor::from_memory(Memory::make_borrowed(reinterpret_cast<void*>(at), 4, Device{DeviceType::kCUDA, 1}), {1}, ScalarType::kInt32);
    };
    Tensor far_lens = elsewhere(0x90000000), far_rows = elsewhere(0x91000000);
    auto evict = [&](const Tensor& row_of, Tensor& to) {
        evict_kvcache(c.k_cache, c.v_cache, c.params, c.params, c.weights, row_of, c.lens, c.tables, c.weights, c.tables, to, 2, 128, 16, 8, 1, 2);
    };
    CHECK_THROWS(evict(c.none, far_lens), std::invalid_argument);
    CHECK_THROWS(evict(far_rows, new_lens), std::invalid_argument);
}

TEST_CASE(decode_and_gather_refuse_tensors_of_another_device) {
    Case c;
    NoAllocator none;
    auto far = [](const std::vector<int64_t>& sizes, ScalarType type, uintptr_t at) {
        return Tensor::from_memory(Memory::make_borrowed(reinterpret_cast<void*>(at), compute_numel(sizes) * scalar_type_size(type), Device{DeviceType::kCUDA, 1}),
                                   sizes, type);
    };
    Tensor rows = far({1}, ScalarType::kInt32, 0x92000000), starts = far({2}, ScalarType::kInt32, 0x93000000), tables = far({1, 2}, ScalarType::kInt32, 0x94000000),
           near_starts = borrowed({2}, ScalarType::kInt32), value = borrowed({3, 2, 128}, ScalarType::kBFloat16), new_lens = borrowed({1}, ScalarType::kInt32),
           k16 = borrowed({2, 16, 2, 128}, ScalarType::kBFloat16), v16 = far({2, 16, 2, 128}, ScalarType::kBFloat16, 0x95000000);
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, c.tables, 2, 128, 16, 1.0f, c.none, rows, c.weights,
                                                       c.output, none, nullptr), std::invalid_argument);
    CHECK_THROWS(launch_decode_attention_paged_weights(c.query, k16, v16, c.none, c.none, c.lens, c.tables, 2, 128, 16, 1.0f, c.none, c.none, c.weights, c.output, none,
                                                       nullptr), std::invalid_argument);
    CHECK_THROWS(evict_kvcache(k16, v16, c.none, c.none, c.weights, c.none, c.lens, c.tables, c.weights, c.tables, new_lens, 2, 128, 16, 8, 1, 2), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, starts, c.tables, 2, 128, 16, c.key, value), std::invalid_argument);
    CHECK_THROWS(gather_kvcache_int4(c.k_cache, c.v_cache, c.params, c.params, near_starts, tables, 2, 128, 16, c.key, value), std::invalid_argument);
}

TEST_CASE(layer_refuses) {
    Case c;
    Attention attention(4, 2, 128, 16), narrow(4, 2, 64, 16);
    Tensor half_params = borrowed({2, 16, 2, 2}, ScalarType::kFloat16), few = borrowed({16, 2, 2}, ScalarType::kBFloat16), floats = borrowed({2, 16, 2, 2}, ScalarType::kFloat32);
    CHECK_THROWS(attention.set_kv_cache_int4(c.key, c.key, c.params, c.params), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_int4(c.k_cache, c.v_cache, c.params, half_params), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_int4(c.k_cache, c.v_cache, few, few), std::invalid_argument);
    CHECK_THROWS(attention.set_kv_cache_int4(c.k_cache, c.v_cache, floats, floats), std::invalid_argument);
    CHECK_THROWS(narrow.set_kv_cache_int4(c.k_cache, c.v_cache, c.params, c.params), std::invalid_argument);
    CHECK_THROWS(attention.set_key_weights(c.key), std::invalid_argument);
    CHECK_THROWS(attention.set_key_weights(c.weights, c.key), std::invalid_argument);
    attention.set_kv_cache_int4(c.k_cache, c.v_cache, c.params, c.params);
    CHECK(attention.is_int4() && attention.is_quantised() && !attention.is_int8());
    attention.set_kv_cache(c.key, c.key);
    CHECK(!attention.is_quantised());
}

namespace {

// Scratch is asked for by stream; the first request ends the call.
struct Asked {};
class StreamAllocator final : public NoAllocator {
public:
    Memory::Ptr allocate(size_t bytes, Device device) override { return Memory::make_borrowed(reinterpret_cast<void*>(uintptr_t(1) << 40), bytes, device); }
    Memory::Ptr allocate_on(size_t bytes, Device, cudaStream_t stream) override {
        last = stream;
        size = bytes;
        throw Asked();
    }
    cudaStream_t last = nullptr;
    size_t size = 0;
};

}  // namespace

TEST_CASE(scratch_belongs_to_the_stream_of_the_call) {
    Case c;
    StreamAllocator alloc;
    const cudaStream_t stream = reinterpret_cast<cudaStream_t>(uintptr_t(0x77));
    Tensor tables = borrowed({1, 512}, ScalarType::kInt32), weights = borrowed({1, 2, 8192}, ScalarType::kFloat32), full = borrowed({2, 16, 2, 128}, ScalarType::kBFloat16);
    auto asks = [&](auto call) {
        alloc.last = nullptr;
        CHECK_THROWS(call(), Asked);
        CHECK(alloc.last == stream && alloc.size > 0);
    };
    asks([&] { launch_decode_attention_paged_int4(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, tables, 2, 128, 16, 1.0f, c.output, alloc, stream); });
    asks([&] { launch_decode_attention_paged_weights(c.query, c.k_cache, c.v_cache, c.params, c.params, c.lens, tables, 2, 128, 16, 1.0f, c.none, c.none, weights, c.output, alloc, stream); });
    asks([&] { launch_decode_attention_paged_weights(c.query, full, full, c.none, c.none, c.lens, tables, 2, 128, 16, 1.0f, c.none, c.none, weights, c.output, alloc, stream); });
    asks([&] { flash_attn_decode_kvcache(c.query, full, full, c.lens, tables, 2, 128, 16, 1.0f, c.output, alloc, stream); });
    Attention layer(4, 2, 128, 16);
    layer.set_kv_cache_int4(c.k_cache, c.v_cache, c.params, c.params);
    const Tensor cu = borrowed({2}, ScalarType::kInt32), q = borrowed({3, 4, 128}, ScalarType::kBFloat16);
    set_context(true, cu, cu, 3, 20, Tensor(), Tensor(), borrowed({1, 2}, ScalarType::kInt32));
    asks([&] { layer.forward(q, c.key, c.key, alloc, stream); });
    reset_context();
}

TEST_CASE(a_prefill_takes_rows_for_the_keys_that_there_are) {
    Case c;
    StreamAllocator alloc;
    Attention layer(4, 2, 128, 16);
    layer.set_kv_cache_int4(c.k_cache, c.v_cache, c.params, c.params);
    const Tensor cu = borrowed({33}, ScalarType::kInt32), tables = borrowed({32, 2048}, ScalarType::kInt32), q = borrowed({3, 4, 128}, ScalarType::kBFloat16);
    const size_t row = 2 * 128 * sizeof(uint16_t);
    auto rows = [&](int longest, int64_t total) {   // one sequence of 32768 keys among 31 of 100
        set_context(true, cu, cu, 3, longest, Tensor(), Tensor(), tables, total);
        CHECK_THROWS(layer.forward(q, c.key, c.key, alloc), Asked);
        reset_context();
        return static_cast<int64_t>(alloc.size / row);
    };
    CHECK_EQ(rows(32768, 32768 + 31 * 100), 32768 + 31 * 100);
    CHECK_EQ(rows(0, 32768 + 31 * 100), 32768 + 31 * 100);
    CHECK_EQ(rows(1000, 0), 32 * 1000);     // not known: as many for each as the longest has
    CHECK_EQ(rows(0, 0), 32 * 2048 * 16);   // or as the table could hold
}

int main() { return check::run_all(); }
