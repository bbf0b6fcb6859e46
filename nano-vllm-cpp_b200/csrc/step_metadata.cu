// The metadata of a step on the GPU: block tables, context lengths, cumulative lengths, positions and slots from the lengths of the step's requests, with
// new cache blocks taken from a list of free ones; and the blocks of requests that ended back onto that list.  What the reference's ModelRunner builds on
// the host for every step (src/engine/model_runner.cpp:482-632, :748-769) and its BlockManager hands out.
//
// With old length l_b, n_b new tokens and blocks of s tokens, request b needs ceil((l_b + n_b) / s) - ceil(l_b / s) new blocks; the prefix sums of these
// say which of the free blocks are its own, and whether there are enough.  Two sums over the batch, then every table entry and every token by itself.
//
// A call is bound by the trips to memory one after the other (row, its length, its blocks) and by the launch: all blocks of one cluster do the sums over the
// whole batch for themselves, so that nothing is handed over, and share out the table entries and the tokens.  A cluster because lengths and the count of free
// blocks may be updated in place: each block has read them when the cluster's barrier is passed.
#include "nvk_internal.cuh"

#include <algorithm>
#include <atomic>

namespace nvk {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 16;            // of a cluster (not portable, but there on every B200)
constexpr int kMaxBatch = 8192;           // 16 bytes of shared memory for each
constexpr uint32_t kMost = 0x7fffffffu;

// Sums of numbers below 2^31, held at 2^31 - 1: lengths come from the device, and no sum of them may wrap round.
__device__ __forceinline__ uint32_t add_held(uint32_t a, uint32_t b) { return min(a + b, kMost); }

__device__ __forceinline__ void put(void* p, int wide, int64_t i, int64_t v) {
    if (wide) static_cast<int64_t*>(p)[i] = v;
    else static_cast<int32_t*>(p)[i] = static_cast<int32_t>(v);
}

// Sums over the threads before this one and, in `total`, over all.  Two numbers at a time.
struct Two { uint32_t a, b; };
__device__ __forceinline__ Two scan_block(Two v, Two& total, Two* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Two x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, x.a, d), b = __shfl_up_sync(0xffffffffu, x.b, d);
        if (lane >= d) { x.a = add_held(x.a, a); x.b = add_held(x.b, b); }
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    Two w = lane < kWarps ? s_warp[lane] : Two{0u, 0u};
#pragma unroll
    for (int d = 1; d < kWarps; d *= 2) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, w.a, d), b = __shfl_up_sync(0xffffffffu, w.b, d);
        if (lane >= d) { w.a = add_held(w.a, a); w.b = add_held(w.b, b); }
    }
    total = Two{__shfl_sync(0xffffffffu, w.a, kWarps - 1), __shfl_sync(0xffffffffu, w.b, kWarps - 1)};
    const uint32_t a = __shfl_sync(0xffffffffu, w.a, max(warp - 1, 0)), b = __shfl_sync(0xffffffffu, w.b, max(warp - 1, 0));
    Two before{__shfl_up_sync(0xffffffffu, x.a, 1), __shfl_up_sync(0xffffffffu, x.b, 1)};
    if (lane == 0) before = Two{0u, 0u};
    if (warp > 0) before = Two{add_held(before.a, a), add_held(before.b, b)};
    __syncthreads();                      // (s_warp is used again)
    return before;
}

// Every block of the cluster has come here, and has read what comes before it in its program.
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }

// What is known of a request of the step, in shared memory.
struct Request {
    int row;      // of the table of requests; -1: padding
    int old_len;  // -1: there is no place for it
    int cu;       // first token
    int first;    // the first of its new blocks among those of the step
};

struct StepParams {
    IndexArray new_lens, rows, lens, free_blocks, free_count;
    void *request_blocks, *block_tables, *context_lens, *cu_q, *cu_k, *positions, *slots, *new_lens_out, *new_count;
    int64_t num_rows, row_blocks, num_free, num_cache_blocks, num_tokens;
    int batch, max_blocks, wide;
    uint32_t capacity;                    // tokens of a request, at most
    FastDiv by_block, by_width;
};

__device__ __forceinline__ uint32_t blocks_of(const FastDiv& by_block, uint32_t tokens) { return by_block.div(tokens + by_block.d - 1); }

__global__ void __launch_bounds__(kThreads) step_metadata_kernel(const __grid_constant__ StepParams p) {
    extern __shared__ Request s_request[];
    __shared__ Two s_warp[kWarps];
    pdl_wait_then_release();
    const int tid = threadIdx.x;
    const bool first_block = blockIdx.x == 0;
    const int64_t count_in = p.free_count[0];
    const uint32_t count = static_cast<uint32_t>(min(max(count_in, static_cast<int64_t>(0)), p.num_free));
    Two base{0u, 0u};                     // tokens, new blocks
    uint32_t keys = 0, taken = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int b = b0 + tid;
        const bool there = b < p.batch;
        int64_t row = -1, n64 = 0;
        if (there) {
            row = p.rows != nullptr ? p.rows[b] : b;
            n64 = p.new_lens[b];
        }
        const bool known = there && row >= 0 && row < p.num_rows;
        const int64_t len64 = known ? p.lens[row] : 0;
        const uint32_t n = static_cast<uint32_t>(min(max(n64, static_cast<int64_t>(0)), static_cast<int64_t>(kMost)));
        const uint32_t len = static_cast<uint32_t>(min(max(len64, static_cast<int64_t>(0)), static_cast<int64_t>(kMost)));
        const bool fits = known && len <= p.capacity && n <= p.capacity - len;
        const uint32_t need = fits ? blocks_of(p.by_block, len + n) - blocks_of(p.by_block, len) : 0;
        Two total;
        Two at = scan_block(Two{n, need}, total, s_warp);
        at = Two{add_held(at.a, base.a), add_held(at.b, base.b)};
        const bool placed = fits && (need == 0 || add_held(at.b, need) <= count);
        if (placed && need > 0) taken = max(taken, add_held(at.b, need));
        base = Two{add_held(base.a, total.a), add_held(base.b, total.b)};
        if (there) s_request[b] = Request{known ? static_cast<int>(row) : -1, placed ? static_cast<int>(len) : -1, static_cast<int>(at.a), static_cast<int>(at.b)};
        const uint32_t ctx = placed ? len + n : 0;
        const Two before = scan_block(Two{ctx, 0u}, total, s_warp);
        if (first_block && there) {       // (outputs of their own: nobody reads them here)
            put(p.context_lens, p.wide, b, ctx);
            if (p.cu_q != nullptr) put(p.cu_q, p.wide, b + 1, add_held(at.a, n));
            if (p.cu_k != nullptr) put(p.cu_k, p.wide, b + 1, add_held(add_held(keys, before.a), ctx));
        }
        keys = add_held(keys, total.a);
    }
    if (first_block && tid == 0) {
        if (p.cu_q != nullptr) put(p.cu_q, p.wide, 0, 0);
        if (p.cu_k != nullptr) put(p.cu_k, p.wide, 0, 0);
    }
    const uint32_t tokens = base.a;
    taken = __reduce_max_sync(0xffffffffu, taken);
    if ((tid & 31) == 0) s_warp[tid >> 5].a = taken;
    const bool copy = p.new_lens_out != p.lens.ptr;
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads, me = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
    if (copy) {
        for (int64_t i = me; i < p.num_rows; i += threads) put(p.new_lens_out, p.wide, i, p.lens[i]);
    }
    if (gridDim.x > 1) cluster_sync();
    else __syncthreads();
    // From here on lengths and count are no longer read.
    const IndexArray held(p.request_blocks, p.wide);
    auto new_block = [&](const Request& r, uint32_t nth) { return p.free_blocks[static_cast<int64_t>(count) - 1 - r.first - nth]; };
    auto end_of = [&](int b) { return b + 1 < p.batch ? static_cast<uint32_t>(s_request[b + 1].cu) : tokens; };
    if (first_block) {
        for (int b = tid; b < p.batch; b += kThreads) {
            const Request r = s_request[b];
            if (r.old_len >= 0) put(p.new_lens_out, p.wide, r.row, r.old_len + (end_of(b) - r.cu));
        }
        if (tid < 32) {
            const uint32_t all = __reduce_max_sync(0xffffffffu, tid < kWarps ? s_warp[tid].a : 0u);
            if (tid == 0) put(p.new_count, p.wide, 0, count - all);
        }
    }
    // Table entries.
    const int64_t entries = static_cast<int64_t>(p.batch) * p.max_blocks;
    for (int64_t i = me; i < entries; i += threads) {
        const int b = static_cast<int>(p.by_width.div(static_cast<uint32_t>(i))), j = static_cast<int>(i - static_cast<int64_t>(b) * p.max_blocks);
        const Request r = s_request[b];
        int64_t id = 0;
        if (r.old_len >= 0) {
            const uint32_t had = blocks_of(p.by_block, r.old_len), used = blocks_of(p.by_block, r.old_len + (end_of(b) - r.cu));
            const int64_t at = r.row * p.row_blocks + j;
            if (j < had) {
                id = held[at];
            } else if (j < used) {
                id = new_block(r, j - had);
                put(p.request_blocks, p.wide, at, id);
            }
        }
        put(p.block_tables, p.wide, i, id);
    }
    // Tokens.
    for (int64_t t = me; t < p.num_tokens; t += threads) {
        int64_t pos = 0, slot = -1;
        if (t < tokens) {
            // The last request that begins at or before t (those of no tokens begin where the next one does); of single tokens it is request t.
            int lo = 0, hi = p.batch;
            if (t < p.batch && s_request[t].cu == t && end_of(static_cast<int>(t)) == t + 1) {
                lo = static_cast<int>(t);
            } else {
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s_request[mid].cu <= t) lo = mid;
                    else hi = mid;
                }
            }
            const Request r = s_request[lo];
            if (r.old_len >= 0) {
                const uint32_t at = r.old_len + static_cast<uint32_t>(t - r.cu), j = p.by_block.div(at), had = blocks_of(p.by_block, r.old_len);
                const int64_t id = j < had ? held[r.row * p.row_blocks + j] : new_block(r, j - had);
                pos = at;
                if (id >= 0 && id < p.num_cache_blocks) slot = id * p.by_block.d + (at - j * p.by_block.d);
            }
        }
        put(p.positions, p.wide, t, pos);
        put(p.slots, p.wide, t, slot);
    }
}

struct ReleaseParams {
    IndexArray rows, first_blocks, lens, request_blocks, free_count;
    void *free_blocks, *new_lens_out, *new_count;
    int64_t num_rows, row_blocks, num_free;
    int batch, wide;
    uint32_t capacity;
    FastDiv by_block;
};

// Blocks first_blocks[b] .. ceil(l_b / s) - 1 of each request behind those that are free already, in the requests' order.
__global__ void __launch_bounds__(kThreads) release_blocks_kernel(const __grid_constant__ ReleaseParams p) {
    extern __shared__ Request s_request[];   // row, first of its blocks, how many, where they go
    __shared__ Two s_warp[kWarps];
    pdl_wait_then_release();
    const int tid = threadIdx.x;
    const int64_t count = min(max(p.free_count[0], static_cast<int64_t>(0)), p.num_free);
    uint32_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int b = b0 + tid;
        const bool there = b < p.batch;
        const int64_t row = !there ? -1 : p.rows != nullptr ? p.rows[b] : b;
        const bool known = there && row >= 0 && row < p.num_rows;
        const int64_t len = known ? min(max(p.lens[row], static_cast<int64_t>(0)), static_cast<int64_t>(p.capacity)) : 0;
        const int64_t first = known && p.first_blocks != nullptr ? max(p.first_blocks[b], static_cast<int64_t>(0)) : 0;
        const int64_t held = blocks_of(p.by_block, static_cast<uint32_t>(len));
        const uint32_t n = first < held ? static_cast<uint32_t>(held - first) : 0;
        Two total;
        const Two at = scan_block(Two{n, 0u}, total, s_warp);
        if (there) s_request[b] = Request{known ? static_cast<int>(row) : -1, n > 0 ? static_cast<int>(first) : 0, static_cast<int>(n), static_cast<int>(add_held(at.a, base))};
        base = add_held(base, total.a);
    }
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads, me = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
    if (p.new_lens_out != p.lens.ptr) {
        for (int64_t i = me; i < p.num_rows; i += threads) put(p.new_lens_out, p.wide, i, p.lens[i]);
    }
    if (gridDim.x > 1) cluster_sync();
    else __syncthreads();
    // A warp to a request.
    for (int b = static_cast<int>(me >> 5); b < p.batch; b += static_cast<int>(threads >> 5)) {
        const Request r = s_request[b];
        if (r.row < 0) continue;
        if ((tid & 31) == 0) put(p.new_lens_out, p.wide, r.row, 0);
        for (int j = tid & 31; j < r.cu; j += 32) {
            const int64_t to = count + r.first + j;
            if (to < p.num_free) put(p.free_blocks, p.wide, to, p.request_blocks[r.row * p.row_blocks + r.old_len + j]);
        }
    }
    if (me == 0) put(p.new_count, p.wide, 0, min(count + base, p.num_free));
}

// One cluster of as many blocks as the work is worth: a block for each 4 entries of a thread.
template <typename P>
int launch(const char* what, void (*kernel)(P), const P& p, int64_t work, std::atomic<bool> (&attr_done)[64], cudaStream_t stream) {
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64 && !attr_done[device]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBatch * static_cast<int>(sizeof(Request)));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
        attr_done[device] = true;
    }
    int blocks = 1;
    while (blocks < kMaxBlocks && work > static_cast<int64_t>(blocks) * 4 * kThreads) blocks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.batch * sizeof(Request);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "%s kernel launch: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

}  // namespace

int launch_step_metadata(const StepArgs& a) {
    if (a.batch > kMaxBatch) return fail(NVK_ERR_UNSUPPORTED, "step_metadata: at most %d requests (got %lld)", kMaxBatch, static_cast<long long>(a.batch));
    const int64_t blocks = std::min(a.row_blocks, a.max_blocks), most = (1LL << 31) - 1 - a.block_size;
    if (a.batch * a.max_blocks > most || a.num_rows > most) return fail(NVK_ERR_UNSUPPORTED, "step_metadata: too many requests or table entries");
    static std::atomic<bool> attr_done[64] = {};
    StepParams p{};
    p.new_lens = a.new_lens; p.rows = a.rows; p.lens = a.lens; p.free_blocks = IndexArray(a.free_blocks, a.wide); p.free_count = a.free_count;
    p.request_blocks = a.request_blocks; p.block_tables = a.block_tables; p.context_lens = a.context_lens; p.cu_q = a.cu_q; p.cu_k = a.cu_k;
    p.positions = a.positions; p.slots = a.slots; p.new_lens_out = a.new_request_lens; p.new_count = a.new_free_count;
    p.num_rows = a.num_rows; p.row_blocks = a.row_blocks; p.num_free = a.num_free; p.num_cache_blocks = a.num_cache_blocks; p.num_tokens = a.num_tokens;
    p.batch = static_cast<int>(a.batch); p.max_blocks = static_cast<int>(a.max_blocks); p.wide = a.wide;
    p.capacity = static_cast<uint32_t>(blocks <= most / a.block_size ? blocks * a.block_size : most);
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    p.by_width = FastDiv(static_cast<uint32_t>(a.max_blocks));
    return launch("step_metadata", step_metadata_kernel, p, std::max(a.batch * a.max_blocks, a.num_tokens), attr_done, a.stream);
}

int launch_release_blocks(const StepArgs& a) {
    if (a.batch > kMaxBatch) return fail(NVK_ERR_UNSUPPORTED, "release_blocks: at most %d requests (got %lld)", kMaxBatch, static_cast<long long>(a.batch));
    const int64_t most = (1LL << 31) - 1 - a.block_size;
    if (a.row_blocks > most || a.num_rows > most) return fail(NVK_ERR_UNSUPPORTED, "release_blocks: too many requests or blocks");
    static std::atomic<bool> attr_done[64] = {};
    ReleaseParams p{};
    p.rows = a.rows; p.first_blocks = a.first_blocks; p.lens = a.lens; p.request_blocks = IndexArray(a.request_blocks, a.wide); p.free_count = a.free_count;
    p.free_blocks = a.free_blocks; p.new_lens_out = a.new_request_lens; p.new_count = a.new_free_count;
    p.num_rows = a.num_rows; p.row_blocks = a.row_blocks; p.num_free = a.num_free;
    p.batch = static_cast<int>(a.batch); p.wide = a.wide;
    p.capacity = static_cast<uint32_t>(a.row_blocks <= most / a.block_size ? a.row_blocks * a.block_size : most);
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    return launch("release_blocks", release_blocks_kernel, p, a.batch * 32, attr_done, a.stream);
}

}  // namespace nvk
