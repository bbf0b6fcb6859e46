// Eviction from a paged KV cache by accumulated attention weight, for sm_100a.  No counterpart in the reference.
//
// Of every (sequence, KV head) the first `sinks` keys stay, the last `recent`, and of those between the ones of the largest weights, `budget` in all
// (of equal weights the key that comes first; NaN counts as the least).  What stays closes up, in its order, its weights with it.
//
// One block has a (sequence, KV head).  The weight that just stays is found by its bits, eight at a time from the top: a histogram of the keys that
// agree so far, and a scan from the largest class down.  Then the keys are taken in order, a tile at a time: who stays goes to the place that the number of
// those before it gives.  A key never moves up, and a tile's rows are all read before any is written, so that the same blocks can be source and
// destination.
#include "nvk_internal.cuh"

#include <atomic>

namespace nvk {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = kThreads;           // keys looked at together
constexpr int kDim = 128;

struct EvictParams {
    void* k_cache; void* v_cache; uint32_t* k_params; uint32_t* v_params;
    const float* weights; float* new_weights; IndexArray rows;
    IndexArray context_lens; IndexArray block_tables; IndexArray new_tables;
    void* new_lens;
    int64_t num_rows, row_keys, max_blocks, new_max_blocks, num_cache_blocks, budget, sinks, recent;
    int num_kv_heads, block_size;
    FastDiv by_block;
};

// Weights as whole numbers of the same order; NaN below all.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);   // (-0 is 0)
    return w != w ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct Select { int hist[256]; int warp_sum[kWarps]; uint32_t prefix; int left; };

// The `take`-th largest of weights[0 .. n) (1 <= take <= n): its order, and how many of that order are among the `take`.
__device__ __forceinline__ void nth_largest(const float* weights, int n, int take, Select& sm, uint32_t& order, int& ties) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    int left = take;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) sm.hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t o = order_of(weights[i]);
            if (shift == 24 || (o >> (shift + 8)) == prefix) atomicAdd(&sm.hist[(o >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid < 32) {   // eight classes a lane, the largest first
            int count[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += count[i] = sm.hist[255 - (8 * tid + i)];
            int upto = sum;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, upto, d);
                if (tid >= d) upto += up;
            }
            int before = upto - sum;
            if (before < left && left <= upto) {   // (one lane)
                int i = 0;
                while (i < 7 && before + count[i] < left) before += count[i++];
                sm.prefix = (prefix << 8) | static_cast<uint32_t>(255 - (8 * tid + i));
                sm.left = left - before;
            }
        }
        __syncthreads();
        prefix = sm.prefix;
        left = sm.left;
        __syncthreads();
    }
    order = prefix;
    ties = left;
}

// Places of the flags before a thread's own, and how many there are in all.
__device__ __forceinline__ int count_before(bool flag, int* warp_sum, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned int mask = __ballot_sync(0xffffffffu, flag);
    __syncthreads();
    if (lane == 0) warp_sum[warp] = __popc(mask);
    __syncthreads();
    const int mine = warp_sum[lane];
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int up = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += up;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
    return __shfl_sync(0xffffffffu, upto - mine, warp) + __popc(mask & ((1u << lane) - 1u));
}

// Cache row of position `pos`, or -1.
__device__ __forceinline__ int64_t row_of(const EvictParams& p, const IndexArray& tables, int64_t max_blocks, int b, int pos) {
    const int blk = static_cast<int>(p.by_block.div(pos));
    if (blk >= max_blocks) return -1;
    const int64_t id = tables[b * max_blocks + blk];
    return id >= 0 && id < p.num_cache_blocks ? id * p.block_size + (pos - blk * p.block_size) : -1;
}

// PIECES: 16-byte pieces of a key's (value's) row of one head.
template <int PIECES, bool PARAMS>
__global__ void __launch_bounds__(kThreads) evict_kernel(const __grid_constant__ EvictParams p) {
    __shared__ Select sel;
    __shared__ int64_t s_from[kTile], s_to[kTile];
    pdl_wait_then_release();
    const int tid = threadIdx.x;
    const int b = blockIdx.x / p.num_kv_heads, kvh = blockIdx.x - b * p.num_kv_heads;
    const int64_t ctx = p.context_lens[b], cap = p.max_blocks * p.block_size;
    const int n = static_cast<int>(ctx < 0 ? 0 : ctx < cap ? ctx : cap);
    const int64_t wrow = p.rows != nullptr ? p.rows[b] : b;
    const bool live = wrow >= 0 && wrow < p.num_rows;
    const int new_n = live && n > p.budget ? static_cast<int>(p.budget) : n;
    if (kvh == 0 && tid == 0) {
        if (p.context_lens.wide) static_cast<int64_t*>(p.new_lens)[b] = new_n;
        else static_cast<int32_t*>(p.new_lens)[b] = new_n;
    }
    if (!live) return;
    const float* weights = p.weights + (wrow * p.num_kv_heads + kvh) * p.row_keys;
    float* new_weights = p.new_weights + (wrow * p.num_kv_heads + kvh) * p.row_keys;
    // Keys [lo, hi) go by their weight: those above `order` stay, and the first `ties` of that order.
    const bool all = n <= p.budget;
    const int lo = all ? n : static_cast<int>(p.sinks), hi = all ? n : n - static_cast<int>(p.recent), take = all ? 0 : static_cast<int>(p.budget - p.sinks - p.recent);
    uint32_t order = 0xffffffffu;
    int ties = 0;
    if (take > 0) nth_largest(weights + lo, hi - lo, take, sel, order, ties);
    int kept = 0, equal = 0;
    for (int base = 0; base < n; base += kTile) {
        const int pos = base + tid;
        const float w = pos < n ? weights[pos] : 0.0f;
        const bool mid = pos >= lo && pos < hi;
        const uint32_t o = order_of(w);
        const bool tie = mid && take > 0 && o == order;
        int in_tile, ties_in_tile;
        const int ties_before = equal + count_before(tie, sel.warp_sum, ties_in_tile);
        equal += ties_in_tile;
        const bool stays = pos < n && (!mid || (take > 0 && (o > order || (tie && ties_before < ties))));
        const int to = kept + count_before(stays, sel.warp_sum, in_tile);
        if (stays) {
            s_from[to - kept] = row_of(p, p.block_tables, p.max_blocks, b, pos);
            s_to[to - kept] = row_of(p, p.new_tables, p.new_max_blocks, b, to);
            new_weights[to] = w;          // (all weights of this tile and of those before have been read)
        }
        __syncthreads();
        // The rows, a set of pieces of every thread at a time: all read before any is written.
        constexpr int kSet = 8, kPerRow = 2 * PIECES + (PARAMS ? 1 : 0);
        const size_t stride = static_cast<size_t>(p.num_kv_heads) * PIECES;   // pieces of a cache row
        for (int first = 0; first < in_tile * kPerRow; first += kSet * kThreads) {
            uint4 v[kSet];
#pragma unroll
            for (int i = 0; i < kSet; ++i) {
                const int at = first + i * kThreads + tid;
                v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (at < in_tile * kPerRow) {
                    const int r = at / kPerRow, c = at - r * kPerRow;
                    const int64_t from = s_from[r];
                    if (from >= 0 && from != s_to[r]) {
                        if (c < PIECES) v[i] = static_cast<const uint4*>(p.k_cache)[from * stride + kvh * PIECES + c];
                        else if (c < 2 * PIECES) v[i] = static_cast<const uint4*>(p.v_cache)[from * stride + kvh * PIECES + c - PIECES];
                        else { v[i].x = p.k_params[from * p.num_kv_heads + kvh]; v[i].y = p.v_params[from * p.num_kv_heads + kvh]; }
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kSet; ++i) {
                const int at = first + i * kThreads + tid;
                if (at < in_tile * kPerRow) {
                    const int r = at / kPerRow, c = at - r * kPerRow;
                    const int64_t to_row = s_to[r];
                    if (to_row >= 0 && to_row != s_from[r]) {
                        if (c < PIECES) static_cast<uint4*>(p.k_cache)[to_row * stride + kvh * PIECES + c] = v[i];
                        else if (c < 2 * PIECES) static_cast<uint4*>(p.v_cache)[to_row * stride + kvh * PIECES + c - PIECES] = v[i];
                        else { p.k_params[to_row * p.num_kv_heads + kvh] = v[i].x; p.v_params[to_row * p.num_kv_heads + kvh] = v[i].y; }
                    }
                }
            }
        }
        kept += in_tile;
        __syncthreads();
    }
    for (int64_t i = new_n + tid; i < p.row_keys; i += kThreads) new_weights[i] = 0.0f;
}

}  // namespace

int launch_evict(const EvictArgs& a) {
    if (a.batch * a.num_kv_heads > 0x7fffffffLL || a.max_blocks * a.block_size >= 0x7fffffffLL - kTile || a.new_max_blocks * a.block_size >= 0x7fffffffLL)
        return fail(NVK_ERR_UNSUPPORTED, "evict_kvcache: batch or block table too large");
    const EvictParams p{a.k_cache, a.v_cache, static_cast<uint32_t*>(a.k_params), static_cast<uint32_t*>(a.v_params), a.weights, a.new_weights, a.rows,
                        a.context_lens, a.block_tables, a.new_tables, a.new_lens, a.num_rows, a.row_keys, a.max_blocks, a.new_max_blocks,
                        a.num_cache_blocks, a.budget, a.sinks, a.recent, a.num_kv_heads, a.block_size, FastDiv(static_cast<uint32_t>(a.block_size))};
    const dim3 grid(static_cast<unsigned>(a.batch * a.num_kv_heads)), block(kThreads);
    const cudaError_t e = a.k_params != nullptr ? launch_pdl(evict_kernel<kDim / 2 / 16, true>, grid, block, 0, a.stream, p)
                                                : launch_pdl(evict_kernel<kDim * 2 / 16, false>, grid, block, 0, a.stream, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "evict_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("evict_kernel launch");
}

}  // namespace nvk
