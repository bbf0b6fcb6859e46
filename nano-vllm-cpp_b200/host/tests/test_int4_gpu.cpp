// The 4-bit cache, the key weights and the eviction through the C++ layer on a GPU.  Keys and values are whole numbers from 0 to 15 (0 and 15 in every head vector),
// which a 4-bit cache holds exactly: step 1, low 0; the layer over it and the layer over a 16-bit cache then attend over the same numbers.
#include "check.h"

#include "engine/step_metadata.h"
#include "kernels/attention.h"
#include "kernels/kvcache.h"
#include "layers/attention.h"
#include "utils/context.h"
#include "utils/cuda_allocator.h"
#include "utils/cuda_common.h"

#include <cuda_runtime_api.h>

#include <cmath>
#include <cstring>
#include <numeric>

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

uint32_t state = 12345;
uint32_t next_random() { return (state = state * 1664525u + 1013904223u) >> 8; }
Tensor numbers(int tokens) {   // whole numbers from 0 to 15, both ends among them
    std::vector<uint16_t> v;
    for (int i = 0; i < tokens * kKvHeads * kDim; ++i) v.push_back(bf16(i % kDim == 0 ? 0.0f : i % kDim == 1 ? 15.0f : static_cast<float>(next_random() % 16)));
    return upload({tokens, kKvHeads, kDim}, ScalarType::kBFloat16, v);
}
Tensor queries(int tokens) {   // multiples of 1/32
    std::vector<uint16_t> v;
    for (int i = 0; i < tokens * kHeads * kDim; ++i) v.push_back(bf16((static_cast<float>(next_random() % 17) - 8.0f) / 32.0f));
    return upload({tokens, kHeads, kDim}, ScalarType::kBFloat16, v);
}
void check_close(const Tensor& a, const Tensor& b) {
    // Two roundings of results up to 15 (half a step, 2^-8 of it, each), and of the probabilities, 2^-8 and 2^-11 of values up to 15.
    const std::vector<float> x = floats(a), y = floats(b);
    CHECK_EQ(x.size(), y.size());
    double most = 0.0;
    for (size_t i = 0; i < x.size(); ++i) most = std::max(most, std::fabs(static_cast<double>(x[i]) - y[i]));
    CHECK(most <= 15.0 * (3.0 / 256 + 1.0 / 2048));
}

}  // namespace

TEST_CASE(layer_over_a_4_bit_cache_equals_the_16_bit_one_on_whole_numbers) {
    CudaAllocator& alloc = CudaAllocator::instance();
    Attention four(kHeads, kKvHeads, kDim, kBlock), full(kHeads, kKvHeads, kDim, kBlock);
    const int blocks = 6;
    four.set_kv_cache_int4(Tensor::zeros({blocks, kBlock, kKvHeads, kDim / 2}, ScalarType::kInt8, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, kDim / 2}, ScalarType::kInt8, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, 2}, ScalarType::kBFloat16, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, 2}, ScalarType::kBFloat16, kDev, alloc));
    full.set_kv_cache(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc),
                      Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc));
    const std::vector<int32_t> table = {4, 1, 3};
    auto slot = [&](int pos) { return table[pos / kBlock] * kBlock + pos % kBlock; };
    auto slots = [&](int from, int to) {
        std::vector<int32_t> s;
        for (int i = from; i < to; ++i) s.push_back(slot(i));
        return ints({to - from}, s);
    };
    const Tensor tables = ints({1, 3}, table);
    // a prompt of 20 tokens, a second chunk of 17 behind it, two decode steps
    for (int begin = 0, end = 20; begin < 37; begin = end, end = 37) {
        const Tensor q = queries(end - begin), k = numbers(end - begin), v = numbers(end - begin);
        set_context(true, ints({2}, {0, end - begin}), ints({2}, {0, end}), end - begin, begin == 0 ? 0 : end, slots(begin, end), Tensor(), tables);
        check_close(four.forward(q, k, v, alloc), full.forward(q, k, v, alloc));
    }
    throw_if_prefill_error();
    Tensor weights = Tensor::zeros({1, kKvHeads, 3 * kBlock}, ScalarType::kFloat32, kDev, alloc);
    for (int n = 38; n < 40; ++n) {
        const Tensor q = queries(1), k = numbers(1), v = numbers(1);
        set_context(false, Tensor(), Tensor(), 0, 0, slots(n - 1, n), ints({1}, {n}), tables);
        const Tensor plain = four.forward(q, k, v, alloc);
        check_close(plain, full.forward(q, k, v, alloc));
        four.set_key_weights(weights);
        CHECK(floats(four.forward_decode_flash_only(q, alloc)) == floats(plain));
        four.set_key_weights(Tensor());
    }
    reset_context();
    // every step's weights of a KV head add up to its number of query heads
    const std::vector<float> w = download<float>(weights);
    for (int j = 0; j < kKvHeads; ++j)
        CHECK_NEAR(std::accumulate(w.begin() + j * 3 * kBlock, w.begin() + (j + 1) * 3 * kBlock, 0.0), 2.0 * kHeads / kKvHeads, 1e-4);
}

TEST_CASE(evict_keeps_the_first_the_last_and_the_heaviest) {
    CudaAllocator& alloc = CudaAllocator::instance();
    const int blocks = 3, n = 30, budget = 10;
    std::vector<uint16_t> rows;   // the number of a row in all its elements (up to 95: exact)
    for (int r = 0; r < blocks * kBlock; ++r) rows.insert(rows.end(), kKvHeads * kDim, bf16(static_cast<float>(r)));
    Tensor k = upload({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, rows), v = upload({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, rows);
    std::vector<float> w(kKvHeads * 2 * kBlock, 0.0f);
    for (int i = 0; i < n; ++i) {
        w[i] = static_cast<float>(i % 7);                                // head 0: 6, 13, 20, 27, then of the fives 5, 12, 19
        w[2 * kBlock + i] = static_cast<float>(n - i);                   // head 1: the first ones
    }
    Tensor weights = upload({1, kKvHeads, 2 * kBlock}, ScalarType::kFloat32, w), none, new_lens = ints({1}, {0});
    const Tensor tables = ints({1, 2}, {2, 0}), lens = ints({1}, {n});
    evict_kvcache(k, v, none, none, weights, none, lens, tables, weights, tables, new_lens, kKvHeads, kDim, kBlock, budget, 1, 2);
    CHECK_EQ(download<int32_t>(new_lens)[0], budget);
    const int stay[2][10] = {{0, 5, 6, 12, 13, 19, 20, 27, 28, 29}, {0, 1, 2, 3, 4, 5, 6, 7, 28, 29}};
    const std::vector<float> got_k = floats(k), got_v = floats(v), got_w = download<float>(weights);
    for (int j = 0; j < kKvHeads; ++j) {
        for (int i = 0; i < budget; ++i) {
            const int at = ((2 * kBlock + i) * kKvHeads + j) * kDim, old = stay[j][i], from = (old < kBlock ? 2 * kBlock : 0) + old % kBlock;
            CHECK_EQ(got_k[at], static_cast<float>(from));
            CHECK_EQ(got_v[at + kDim - 1], static_cast<float>(from));
            CHECK_EQ(got_w[j * 2 * kBlock + i], w[j * 2 * kBlock + old]);
        }
        for (int i = budget; i < 2 * kBlock; ++i) CHECK_EQ(got_w[j * 2 * kBlock + i], 0.0f);
    }
}

TEST_CASE(scratch_of_one_stream_does_not_go_to_another) {
    CudaAllocator& alloc = CudaAllocator::instance();
    cudaStream_t a = nullptr, b = nullptr;
    throw_if_cuda_error(cudaStreamCreateWithFlags(&a, cudaStreamNonBlocking), "cudaStreamCreate");
    throw_if_cuda_error(cudaStreamCreateWithFlags(&b, cudaStreamNonBlocking), "cudaStreamCreate");
    const size_t bytes = 5 << 20;
    void* first = alloc.allocate_on(bytes, kDev, a)->data();
    CHECK(alloc.allocate_on(bytes, kDev, b)->data() != first);
    CHECK(alloc.allocate_on(bytes, kDev, nullptr)->data() != first);
    CHECK(alloc.allocate(bytes, kDev)->data() != first);
    CHECK(alloc.allocate_on(bytes - 1000, kDev, a)->data() == first);
    // a stream that is being captured, with nothing in its list
    cudaStream_t c = nullptr;
    throw_if_cuda_error(cudaStreamCreateWithFlags(&c, cudaStreamNonBlocking), "cudaStreamCreate");
    throw_if_cuda_error(cudaStreamBeginCapture(c, cudaStreamCaptureModeGlobal), "cudaStreamBeginCapture");
    void* captured = nullptr;
    {
        const Memory::Ptr m = alloc.allocate_on(bytes, kDev, c);
        alloc.memset_async(m->data(), 0, bytes, c);
        captured = m->data();
    }
    CHECK(alloc.allocate_on(bytes, kDev, c)->data() == captured);
    CHECK(alloc.allocate_on(bytes, kDev, a)->data() == first);   // (the others go on)
    CHECK(alloc.allocate_on(3 * bytes, kDev, b)->data() != nullptr);
    cudaGraph_t graph = nullptr;
    throw_if_cuda_error(cudaStreamEndCapture(c, &graph), "cudaStreamEndCapture");
    CHECK(alloc.allocate_on(bytes, kDev, c)->data() != captured);   // (the graph's)
    throw_if_cuda_error(cudaGraphDestroy(graph), "cudaGraphDestroy");
    for (cudaStream_t s : {a, b, c}) throw_if_cuda_error(cudaStreamDestroy(s), "cudaStreamDestroy");
}

TEST_CASE(two_streams_that_share_the_allocator_give_what_one_gives) {
    CudaAllocator& alloc = CudaAllocator::instance();
    const int batch = 24, width = 128, blocks = 256, keys = width * kBlock;   // chunks and a merge
    cudaStream_t streams[2];
    struct Side { Tensor query, k, v, lens, tables; } side[2];
    for (int i = 0; i < 2; ++i) {
        throw_if_cuda_error(cudaStreamCreateWithFlags(&streams[i], cudaStreamNonBlocking), "cudaStreamCreate");
        std::vector<int32_t> lens, tables;
        for (int b = 0; b < batch; ++b) lens.push_back(1 + static_cast<int32_t>(next_random() % keys));
        for (int b = 0; b < batch * width; ++b) tables.push_back(static_cast<int32_t>(next_random() % blocks));
        side[i] = {queries(batch), numbers(blocks * kBlock), numbers(blocks * kBlock), ints({batch}, lens), ints({batch, width}, tables)};
    }
    const Tensor none;
    const int rounds = 20;
    std::vector<float> out[2][2], sum[2][2];   // [in turn | at once][side]
    for (int way = 0; way < 2; ++way) {
        Tensor outs[2], weights[2];
        for (int i = 0; i < 2; ++i) {
            outs[i] = Tensor::zeros({batch, kHeads, kDim}, ScalarType::kBFloat16, kDev, alloc);
            weights[i] = Tensor::zeros({batch, kKvHeads, keys}, ScalarType::kFloat32, kDev, alloc);
        }
        throw_if_cuda_error(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
        auto step = [&](int i) {
            launch_decode_attention_paged_weights(side[i].query, side[i].k, side[i].v, none, none, side[i].lens, side[i].tables, kKvHeads, kDim, kBlock, 0.1f, weights[i], none,
                                                  weights[i], outs[i], alloc, streams[i]);
        };
        if (way == 0) {
            for (int i = 0; i < 2; ++i) {
                for (int r = 0; r < rounds; ++r) step(i);
                alloc.synchronize_stream(streams[i]);
            }
        } else {
            for (int r = 0; r < rounds; ++r) { step(0); step(1); }
        }
        throw_if_cuda_error(cudaDeviceSynchronize(), "cudaDeviceSynchronize");
        for (int i = 0; i < 2; ++i) {
            out[way][i] = floats(outs[i]);
            sum[way][i] = download<float>(weights[i]);
        }
    }
    for (int i = 0; i < 2; ++i) {
        CHECK(out[0][i] == out[1][i]);
        CHECK(sum[0][i] == sum[1][i]);
        throw_if_cuda_error(cudaStreamDestroy(streams[i]), "cudaStreamDestroy");
    }
}

namespace {

// CudaAllocator that counts the scratch asked for.
class CountingAllocator final : public DeviceAllocator {
public:
    Memory::Ptr allocate(size_t bytes, Device device) override { return inner.allocate(bytes, device); }
    Memory::Ptr allocate_on(size_t bytes, Device device, cudaStream_t stream) override {
        scratch += bytes;
        return inner.allocate_on(bytes, device, stream);
    }
    void memset_async(void* p, int value, size_t bytes, cudaStream_t stream) const override { inner.memset_async(p, value, bytes, stream); }
    void copy_to_device_async(void* dst, const void* src, size_t bytes, cudaStream_t stream) const override { inner.copy_to_device_async(dst, src, bytes, stream); }
    void copy_to_host_async(void* dst, const void* src, size_t bytes, cudaStream_t stream) const override { inner.copy_to_host_async(dst, src, bytes, stream); }
    void synchronize_stream(cudaStream_t stream) const override { inner.synchronize_stream(stream); }
    CudaAllocator& inner = CudaAllocator::instance();
    size_t scratch = 0;
};

}  // namespace

TEST_CASE(chunks_of_prompts_of_unequal_lengths_over_a_4_bit_cache) {
    // prompts of 500 and of a few tokens, the first ones cached; the second step has a longer chunk of each
    CountingAllocator alloc;
    const std::vector<int> lens = {500, 3, 40, 17, 16, 100};
    Attention four(kHeads, kKvHeads, kDim, kBlock), full(kHeads, kKvHeads, kDim, kBlock);
    const int blocks = 64;
    four.set_kv_cache_int4(Tensor::zeros({blocks, kBlock, kKvHeads, kDim / 2}, ScalarType::kInt8, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, kDim / 2}, ScalarType::kInt8, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, 2}, ScalarType::kBFloat16, kDev, alloc),
                           Tensor::zeros({blocks, kBlock, kKvHeads, 2}, ScalarType::kBFloat16, kDev, alloc));
    full.set_kv_cache(Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc),
                      Tensor::zeros({blocks, kBlock, kKvHeads, kDim}, ScalarType::kBFloat16, kDev, alloc));
    std::vector<int32_t> tokens(500, 1);
    std::vector<std::vector<int32_t>> tables;
    std::vector<SequenceView> seqs;
    int next = 0;
    for (int n : lens) {
        std::vector<int32_t> table;
        for (int i = 0; i < (n + kBlock - 1) / kBlock; ++i) table.push_back(next++ * 37 % blocks);
        tables.push_back(table);
    }
    CHECK(next <= blocks);
    for (size_t i = 0; i < lens.size(); ++i) {
        SequenceView s;
        s.token_ids = tokens.data();
        s.num_tokens = lens[i];
        s.block_table = tables[i].data();
        s.block_table_len = static_cast<int32_t>(tables[i].size());
        seqs.push_back(s);
    }
    StepUploader uploader(alloc, kDev);
    for (int part = 0; part < 2; ++part) {
        for (size_t i = 0; i < lens.size(); ++i) {
            seqs[i].num_computed_tokens = part == 0 ? 0 : (lens[i] + 1) / 3;
            seqs[i].num_tokens_to_process = part == 0 ? (lens[i] + 1) / 3 : lens[i] - (lens[i] + 1) / 3;
        }
        const StepArrays step = build_prefill_arrays(seqs, kBlock);
        uploader.upload(step);
        CHECK_EQ(get_context().total_seqlen_k, static_cast<int64_t>(step.cu_seqlens_k.back()));
        const int rows = static_cast<int>(step.input_ids.size());
        const Tensor q = queries(rows), k = numbers(rows), v = numbers(rows);
        alloc.scratch = 0;
        const Tensor out = four.forward(q, k, v, alloc);
        if (part == 1) CHECK_EQ(alloc.scratch, static_cast<size_t>(2 * 676 * kKvHeads * kDim * 2));
        check_close(out, full.forward(q, k, v, alloc));
    }
    throw_if_prefill_error();
    reset_context();
}

int main() {
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
        std::printf("no CUDA device\n");
        return 77;
    }
    throw_if_cuda_error(cudaSetDevice(0), "cudaSetDevice");
    return check::run_all();
}
