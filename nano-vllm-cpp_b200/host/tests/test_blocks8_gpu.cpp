// The 8-bit cache with block scales, the rotary positions and the step metadata through the C++ layer on a GPU.  Keys and values are whole numbers from -127 to 127, with one of 127 in
// every row, which an int8 cache of scale 1 holds exactly; the layer over it and the layer over a 16-bit cache then attend over the same numbers.
#include "check.h"

#include "engine/step_metadata.h"
#include "kernels/attention.h"
#include "kernels/kvcache.h"
#include "kernels/rotary.h"
#include "layers/attention.h"
#include "utils/context.h"
#include "utils/cuda_allocator.h"
#include "utils/cuda_common.h"

#include <cuda_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstring>

using namespace nano_vllm;

namespace {

const Device kDev{DeviceType::kCUDA, 0};
constexpr int kHeads = 4, kKvHeads = 2, kDim = 128, kBlock = 16;

template <typename T> Tensor upload(const std::vector<int64_t>& sizes, ScalarType type, const std::vector<T>& values) {
    CudaAllocator& alloc = CudaAllocator::instance();
    Tensor t = Tensor::empty(sizes, type, kDev, alloc);
    alloc.copy_to_device_async(t.data(), values.data(), t.nbytes(), nullptr);
    alloc.synchronize_stream(nullptr);
    return t;
}
template <typename T> std::vector<T> download(const Tensor& t) {
    std::vector<T> out(t.nbytes() / sizeof(T));
    CudaAllocator& alloc = CudaAllocator::instance();
    alloc.copy_to_host_async(out.data(), t.data(), t.nbytes(), nullptr);
    alloc.synchronize_stream(nullptr);
    return out;
}
Tensor ints(const std::vector<int64_t>& sizes, const std::vector<int32_t>& v) { return upload(sizes, ScalarType::kInt32, v); }
uint16_t bf16(float x) {   // (exact for the values used here)
    uint32_t u;
    std::memcpy(&u, &x, 4);
    return static_cast<uint16_t>(u >> 16);
}
std::vector<float> floats(const Tensor& t) {
    std::vector<float> out;
    for (uint16_t b : download<uint16_t>(t)) {
        const uint32_t u = static_cast<uint32_t>(b) << 16;
        float f;
        std::memcpy(&f, &u, 4);
        out.push_back(f);
    }
    return out;
}

uint32_t state = 4321;
uint32_t next_random() { return (state = state * 1664525u + 1013904223u) >> 8; }
Tensor numbers(int tokens) {   // whole numbers from -127 to 127; every row of a head has 127
    std::vector<uint16_t> v;
    for (int i = 0; i < tokens * kKvHeads * kDim; ++i) v.push_back(bf16(i % kDim == 5 ? 127.0f : static_cast<float>(next_random() % 255) - 127.0f));
    return upload({tokens, kKvHeads, kDim}, ScalarType::kBFloat16, v);
}
Tensor queries(int tokens) {   // multiples of 1/256
    std::vector<uint16_t> v;
    for (int i = 0; i < tokens * kHeads * kDim; ++i) v.push_back(bf16((static_cast<float>(next_random() % 17) - 8.0f) / 256.0f));
    return upload({tokens, kHeads, kDim}, ScalarType::kBFloat16, v);
}
void check_close(const Tensor& a, const Tensor& b) {
    // Two roundings of results up to 127 (half a step, 2^-8 of it, each), and of the probabilities, 2^-8 and 2^-11 of values up to 127.
    const std::vector<float> x = floats(a), y = floats(b);
    CHECK_EQ(x.size(), y.size());
    double most = 0.0;
    for (size_t i = 0; i < x.size(); ++i) most = std::max(most, std::fabs(static_cast<double>(x[i]) - y[i]));
    CHECK(most <= 127.0 * (3.0 / 256 + 1.0 / 2048));
}

}  // namespace

TEST_CASE(steps_without_the_host_equal_the_16_bit_layer_on_whole_numbers) {
    CudaAllocator& alloc = CudaAllocator::instance();
    Attention eight(kHeads, kKvHeads, kDim, kBlock), full(kHeads, kKvHeads, kDim, kBlock);
    const int blocks = 7;
    eight.set_kv_cache_blocks8(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc),
                               Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc),
                               Tensor::zeros({blocks, kKvHeads}, ScalarType::kFloat32, kDev, alloc), Tensor::zeros({blocks, kKvHeads}, ScalarType::kFloat32, kDev, alloc));
    full.set_kv_cache(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc),
                      Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc));
    RequestTables tables{ints({3}, {0, 0, 0}), ints({3, 3}, std::vector<int32_t>(9, -1)), ints({7}, {6, 2, 4, 0, 1, 5, 3}), ints({1}, {7}), kBlock, blocks};
    // a prompt of 20 tokens in row 2, a second chunk of 17 behind it, three decode steps
    for (int begin = 0, end = 20; begin < 40; begin = end, end = end < 37 ? 37 : end + 1) {
        const int n = end - begin;
        DeviceStep step{ints({1, 3}, {0, 0, 0}), ints({1}, {0}), ints({2}, {0, 0}), ints({2}, {0, 0}), ints({n}, std::vector<int32_t>(n, 0)), ints({n}, std::vector<int32_t>(n, 0))};
        build_step(ints({1}, {n}), ints({1}, {2}), tables, step);
        CHECK(download<int32_t>(step.context_lens)[0] == end && download<int32_t>(step.cu_seqlens_k)[1] == end && download<int32_t>(step.positions)[0] == begin);
        const Tensor q = queries(n), k = numbers(n), v = numbers(n);
        if (n > 1) set_context(true, step.cu_seqlens_q, step.cu_seqlens_k, n, end, step.slot_mapping, step.context_lens, step.block_tables, end);
        else set_context(false, Tensor(), Tensor(), 0, 0, step.slot_mapping, step.context_lens, step.block_tables);
        check_close(eight.forward(q, k, v, alloc), full.forward(q, k, v, alloc));
    }
    throw_if_prefill_error();
    reset_context();
    for (float s : download<float>(eight.k_scale())) CHECK(s == 0.0f || s == 1.0f);
    CHECK_EQ(download<int32_t>(tables.free_count)[0], 4);
    release_blocks(ints({1}, {2}), Tensor(), tables);
    CHECK_EQ(download<int32_t>(tables.free_count)[0], 7);
    CHECK_EQ(download<int32_t>(tables.lens)[2], 0);
    CHECK(download<int32_t>(tables.free_blocks) == std::vector<int32_t>({6, 2, 4, 0, 3, 5, 1}));
}

TEST_CASE(rotary_of_packed_rows) {
    // Frequency 0 turns nothing, half a turn changes signs: angles pi at position 1 (rounded to fp32: cos -1, sin -8.7e-8).
    std::vector<uint16_t> v;
    for (int i = 0; i < 2 * 4 * 8; ++i) v.push_back(bf16(static_cast<float>(i % 23) + 1.0f));
    const Tensor packed = upload({2, 32}, ScalarType::kBFloat16, v);   // two query heads, a key head and a value head of 8
    CudaAllocator& alloc = CudaAllocator::instance();
    Tensor q = Tensor::empty({2, 2, 8}, ScalarType::kBFloat16, kDev, alloc), k = Tensor::empty({2, 1, 8}, ScalarType::kBFloat16, kDev, alloc);
    const Tensor freq = upload({2}, ScalarType::kFloat32, std::vector<float>({3.14159265f, 0.0f}));
    for (bool pairs : {false, true}) {
        rotary_embedding(packed.slice(1, 0, 16), packed.slice(1, 16, 24), ints({2}, {0, 1}), freq, 2, 1, 8, pairs, 1.0f, q, k);
        const std::vector<float> in = floats(packed), got_q = floats(q), got_k = floats(k);
        for (int r = 0; r < 2; ++r) {
            for (int i = 0; i < 24; ++i) {
                const int d = i % 8;
                const bool turned = r == 1 && (pairs ? d < 2 : d == 0 || d == 2);
                CHECK_EQ(i < 16 ? got_q[r * 16 + i] : got_k[r * 8 + i - 16], (turned ? -1.0f : 1.0f) * in[r * 32 + i]);
            }
        }
    }
}

TEST_CASE(prompts_and_chunks_of_the_host_path) {
    // What StepUploader publishes, into the layer: prompts, chunks of them, one behind a cached prefix, one that is cached whole; then decode.
    CudaAllocator& alloc = CudaAllocator::instance();
    Attention eight(kHeads, kKvHeads, kDim, kBlock), full(kHeads, kKvHeads, kDim, kBlock);
    const int blocks = 40;
    eight.set_kv_cache_blocks8(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc),
                               Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc),
                               Tensor::zeros({blocks, kKvHeads}, ScalarType::kFloat32, kDev, alloc), Tensor::zeros({blocks, kKvHeads}, ScalarType::kFloat32, kDev, alloc));
    full.set_kv_cache(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc),
                      Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc));
    std::vector<int32_t> tokens(200, 1);
    const std::vector<std::vector<int32_t>> tables = {{9, 30, 2}, {17, 4}, {9, 30, 21, 8}, {17, 4}, {11}};   // the third has two blocks of the first, the fourth all of the second
    const std::vector<int> lens = {48, 32, 61, 32, 1}, cached = {0, 0, 32, 32, 0};
    auto view = [&](int i, int computed, int chunk) {
        SequenceView s;
        s.token_ids = tokens.data();
        s.num_tokens = lens[i];
        s.num_cached_tokens = cached[i];
        s.num_computed_tokens = computed;
        s.num_tokens_to_process = chunk;
        s.block_table = tables[i].data();
        s.block_table_len = static_cast<int32_t>(tables[i].size());
        return s;
    };
    StepUploader uploader(alloc, kDev);
    const std::vector<std::vector<SequenceView>> steps = {{view(0, 0, 33), view(1, 0, 0), view(4, 0, 0)}, {view(0, 33, 15)}, {view(2, 0, 0), view(3, 0, 0)}};
    for (const auto& seqs : steps) {
        const StepArrays step = build_prefill_arrays(seqs, kBlock, true);
        uploader.upload(step);
        CHECK(get_context().context_lens.defined() && get_context().block_tables.defined());
        const int rows = static_cast<int>(step.input_ids.size());
        const Tensor q = queries(rows), k = numbers(rows), v = numbers(rows);
        if (&seqs == &steps[2]) {   // the last row of a prompt that is cached whole is the one that is there: nothing of it is stored in the 8-bit cache, so that the 16-bit one must not either
            const std::vector<uint16_t> k_rows = download<uint16_t>(full.k_cache()), v_rows = download<uint16_t>(full.v_cache());
            const size_t row = kKvHeads * kDim, from = (4 * kBlock + 15) * row;
            CHECK_EQ(step.slot_mapping.back(), 4 * kBlock + 15);
            alloc.copy_to_device_async(static_cast<uint16_t*>(k.data()) + (rows - 1) * row, k_rows.data() + from, row * 2, nullptr);
            alloc.copy_to_device_async(static_cast<uint16_t*>(v.data()) + (rows - 1) * row, v_rows.data() + from, row * 2, nullptr);
            alloc.synchronize_stream(nullptr);
        }
        const std::vector<int8_t> before = download<int8_t>(eight.k_cache());
        check_close(eight.forward(q, k, v, alloc), full.forward(q, k, v, alloc));
        const std::vector<int8_t> after = download<int8_t>(eight.k_cache());
        if (&seqs == &steps[2]) {
            for (int block : {9, 30, 17, 4}) {
                const size_t at = static_cast<size_t>(block) * kBlock * kKvHeads * kDim;
                CHECK(std::equal(before.begin() + at, before.begin() + at + kBlock * kKvHeads * kDim, after.begin() + at));
            }
        }
    }
    std::vector<SequenceView> all;
    for (int i : {0, 2, 4}) all.push_back(view(i, 0, 0));
    uploader.upload(build_decode_arrays(all, kBlock));
    const Tensor q = queries(3), k = numbers(3), v = numbers(3);
    check_close(eight.forward(q, k, v, alloc), full.forward(q, k, v, alloc));
    throw_if_prefill_error();
    reset_context();
}

TEST_CASE(prompts_without_cached_keys_attend_over_exact_rows) {
    // Keys and values that no 8-bit element stands for: bit for bit what a layer without a cache gives, where over the cache's rows there would be a difference.
    CudaAllocator& alloc = CudaAllocator::instance();
    auto halves = [](int rows) {
        std::vector<uint16_t> v;
        for (int i = 0; i < rows * kKvHeads * kDim; ++i) v.push_back(bf16((static_cast<float>(next_random() % 255) - 127.0f) * (i % 3 ? 1.0f : 1.0f / 128)));
        return upload({rows, kKvHeads, kDim}, ScalarType::kBFloat16, v);
    };
    Attention eight(kHeads, kKvHeads, kDim, kBlock), none(kHeads, kKvHeads, kDim, kBlock);
    eight.set_kv_cache_blocks8(Tensor::zeros({6, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc), Tensor::zeros({6, kBlock, kKvHeads, kDim}, ScalarType::kInt8, kDev, alloc),
                               Tensor::zeros({6, kKvHeads}, ScalarType::kFloat32, kDev, alloc), Tensor::zeros({6, kKvHeads}, ScalarType::kFloat32, kDev, alloc));
    const std::vector<int32_t> tokens(40, 1), a = {4, 1, 0}, b = {2};
    std::vector<SequenceView> seqs(2);
    seqs[0].token_ids = seqs[1].token_ids = tokens.data();
    seqs[0].num_tokens = 40; seqs[0].block_table = a.data(); seqs[0].block_table_len = 3;
    seqs[1].num_tokens = 7; seqs[1].block_table = b.data(); seqs[1].block_table_len = 1;
    StepUploader uploader(alloc, kDev);
    uploader.upload(build_prefill_arrays(seqs, kBlock, true));
    CHECK(get_context().only_new_keys);
    const Tensor q = queries(47), k = halves(47), v = halves(47);
    const std::vector<uint16_t> exact = download<uint16_t>(eight.forward(q, k, v, alloc));
    Context context = get_context();
    context.only_new_keys = false;
    set_context(context);
    const std::vector<uint16_t> rounded = download<uint16_t>(eight.forward(q, k, v, alloc));
    context.block_tables = Tensor();
    set_context(context);
    const std::vector<uint16_t> want = download<uint16_t>(none.forward(q, k, v, alloc));
    CHECK(exact == want);
    CHECK(rounded != want);
    // behind cached keys there is more than the new ones
    seqs[0].num_computed_tokens = 30;
    seqs[0].num_tokens_to_process = 10;
    uploader.upload(build_prefill_arrays({seqs[0]}, kBlock, true));
    CHECK(!get_context().only_new_keys);
    reset_context();
    CHECK(!get_context().only_new_keys);
}

int main() { return check::run_all(); }
