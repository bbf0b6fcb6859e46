// Eviction from a paged KV cache by accumulated attention weight, for sm_100a.  No counterpart in the reference.
//
// Of every (sequence, KV head) the first `sinks` keys stay, the last `recent`, and of those between the ones of the largest weights, `budget` in all
// (of equal weights the key that comes first; NaN counts as the least).  What stays closes up, in its order, its weights with it.
//
// HBM-bound: the weights are read, the rows of what stays are read and written (32 sequences of 1000 to 8192 keys, 8 KV heads, 2048 of them kept, 524 MB: 107 us,
// 4.9 TB/s; SMs are busy for 77 % of that, since 256 pairs are two blocks for some SMs and one for others).  Where there are few (sequence, KV head) pairs several blocks share one: each
// finds for itself who stays (weights are a small part of what is read, and come from L2; histograms added up through distributed shared memory took 10 us
// more a pass), and moves the rows of its share of the tiles.  A block
//   1  reads the weights as whole numbers of the same order into shared memory (contexts of up to 16384 keys, 45056 where it is alone on an SM; longer ones are
//      read again for every step);
//   2  finds the order that just stays by its bits, 11, 11 and 10 of them from the top: a histogram of the keys that agree so far, and a scan from the largest
//      class down (weights share exponents: with 8 bits at first the counters of a few classes are the bottleneck; sorting out a class of up to 256 keys by
//      counting, for each, those above it took as long as the two last histograms);
//   3  counts what stays in every tile of 128 keys, which gives the place where each tile's keys go;
//   4  lists the rows of its tiles, old place and new, and moves them, eight 16-byte pieces under way in every thread (a warp alone with the rows of
//      its tile: 4 sequences of 2000 to 4096 keys, 8 KV heads, 79 us; the last keys all stay, and who has them ends last).
// Where the new blocks are the old ones (in place) a row may be written where another one has still to be read.  Then a pair's first block does all of it in order:
// a key never moves up, and a set of rows is read before any of it is written (4 sequences of 2000 to 4096 keys, 8 KV heads, 1024 kept: 33.6 us instead of 16.9).
#include "nvk_internal.cuh"

#include <algorithm>
#include <atomic>

namespace nvk {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = kThreads;           // keys that a block looks at together
constexpr int kWarpTile = 128;            // keys that a warp looks at together
constexpr int kMaxTiles = 1024;           // warp tiles counted one by one; of longer contexts several together
constexpr int kCached = 16384;            // keys whose orders are kept, two blocks to an SM
constexpr int kCachedAlone = 45056;       // one block
constexpr int kList = kWarps * kWarpTile; // rows listed before they are moved
constexpr int kBins = 2048;
constexpr int kMaxSplit = 64;             // blocks of a pair
constexpr int kDim = 128;

struct EvictParams {
    void* k_cache; void* v_cache; uint32_t* k_params; uint32_t* v_params;
    const float* weights; float* new_weights; IndexArray rows;
    IndexArray context_lens; IndexArray block_tables; IndexArray new_tables;
    void* new_lens;
    int64_t num_rows, row_keys, max_blocks, new_max_blocks, num_cache_blocks, budget, sinks, recent;
    int num_kv_heads, block_size, split, cached;
    FastDiv by_block;
};

struct Shared {
    int bins[kBins];
    int2 tiles[kMaxTiles];                // of every tile, then before it: keys that stay without regard to ties, ties
    int2 warp[kWarps];
    int2 list[kList];                     // old row and new one, -1: none
    uint32_t prefix;
    int left, listed;
    uint32_t orders[1];                   // as many as there is room for
};
constexpr size_t shared_bytes(int cached) { return (offsetof(Shared, orders) + cached * sizeof(uint32_t) + 15) / 16 * 16; }
static_assert(shared_bytes(kCached) <= 113 * 1024 && shared_bytes(kCachedAlone) <= 227 * 1024, "two blocks to an SM, or one");

// Weights as whole numbers of the same order; NaN below all.
__device__ __forceinline__ uint32_t order_of(float w) {
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);   // (-0 is 0)
    return w != w ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sums over the threads before a thread's own, and over all.
__device__ __forceinline__ int2 scan(int2 v, Shared& sm, int2& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 upto = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, upto.x, d), y = __shfl_up_sync(0xffffffffu, upto.y, d);
        if (lane >= d) { upto.x += x; upto.y += y; }
    }
    __syncthreads();                      // (what was in sm.warp has been read)
    if (lane == 31) sm.warp[warp] = upto;
    __syncthreads();
    int2 before = make_int2(0, 0);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int2 t = sm.warp[w];
        if (w < warp) { before.x += t.x; before.y += t.y; }
        total.x += t.x; total.y += t.y;
    }
    return make_int2(before.x + upto.x - v.x, before.y + upto.y - v.y);
}

// Of one (sequence, KV head): who stays.  Keys [lo, hi) go by their weight: those above `order` stay, and the first `ties` of that order.
struct Choice {
    int n, lo, hi, take, ties;
    uint32_t order;
    bool cached;
    __device__ __forceinline__ uint32_t order_at(const Shared& sm, const float* weights, int pos) const {
        return cached ? sm.orders[pos] : order_of(weights[pos]);
    }
    // (stays without regard to ties, is a tie)
    __device__ __forceinline__ int2 of(const Shared& sm, const float* weights, int pos) const {
        if (pos >= n) return make_int2(0, 0);
        if (pos < lo || pos >= hi) return make_int2(1, 0);
        if (take == 0) return make_int2(0, 0);
        const uint32_t o = order_at(sm, weights, pos);
        return make_int2(o > order, o == order);
    }
};

// The `take`-th largest of weights[lo .. hi) (1 <= take <= hi - lo): its order, and how many of that order are among the `take`.
__device__ __forceinline__ void choose(const float* weights, Choice& c, Shared& sm, int cached) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    int left = c.take, known = 0;         // bits of the order that are known
    c.cached = c.hi <= cached;
#pragma unroll 1
    for (int bits = 11; known < 32; bits = known < 22 ? 11 : 10) {
        const int shift = 32 - known - bits, bins = 1 << bits;
        for (int i = tid; i < kBins; i += kThreads) sm.bins[i] = 0;
        __syncthreads();
        auto count = [&](uint32_t o) {
            if (known == 0 || (o >> (shift + bits)) == prefix) atomicAdd(&sm.bins[(o >> shift) & (bins - 1)], 1);
        };
        if (c.cached && known > 0) {
            for (int pos = c.lo + tid; pos < c.hi; pos += kThreads) count(sm.orders[pos]);
        } else {
            constexpr int kAhead = 8;
            for (int pos0 = c.lo + tid; pos0 < c.hi; pos0 += kAhead * kThreads) {
                float w[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) w[i] = pos0 + i * kThreads < c.hi ? weights[pos0 + i * kThreads] : 0.0f;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int pos = pos0 + i * kThreads;
                    if (pos < c.hi) {
                        const uint32_t o = order_of(w[i]);
                        if (c.cached) sm.orders[pos] = o;
                        count(o);
                    }
                }
            }
        }
        __syncthreads();
        constexpr int kEach = kBins / kThreads;   // neighbouring classes of a thread, the largest first
        static_assert(kEach == 4, "one int4 a thread");
        const int4 v = reinterpret_cast<const int4*>(sm.bins)[kThreads - 1 - tid];
        const int number[kEach] = {v.w, v.z, v.y, v.x}, sum = v.x + v.y + v.z + v.w;
        int2 total;
        int before = scan(make_int2(sum, 0), sm, total).x;
        if (before < left && left <= before + sum) {   // (one thread)
            int i = 0;
            while (i < kEach - 1 && before + number[i] < left) before += number[i++];
            sm.prefix = (prefix << bits) | static_cast<uint32_t>(kBins - 1 - (tid * kEach + i));
            sm.left = left - before;
        }
        __syncthreads();
        prefix = sm.prefix;
        left = sm.left;
        known += bits;
    }
    c.order = prefix;
    c.ties = left;
}

// Cache row of position `pos`, or -1.
__device__ __forceinline__ int row_of(const EvictParams& p, const IndexArray& tables, int64_t max_blocks, int b, int pos) {
    const int blk = static_cast<int>(p.by_block.div(pos));
    if (blk >= max_blocks) return -1;
    const int64_t id = tables[b * max_blocks + blk];
    return id >= 0 && id < p.num_cache_blocks ? static_cast<int>(id) * p.block_size + (pos - blk * p.block_size) : -1;
}

// Moves rows of one KV head: PIECES of 16 bytes of a key, as many of its value, and their params.  A thread has the same piece of every row that it moves: what is
// left to do for one is a place in the list, two multiplications and the copy (with pieces dealt out one by one 111 instructions, and 32 sequences of 1000
// to 8192 keys, 8 KV heads, took 119 us).
template <int PIECES, bool PARAMS>
struct Mover {
    static constexpr int kPerRow = 2 * PIECES, kRows = kThreads / kPerRow;   // pieces of a row, rows moved together
    const EvictParams& p;
    const int kvh;
    unsigned char* base;                   // this thread's piece of cache row 0
    uint32_t stride;                       // bytes of a cache row
    __device__ __forceinline__ Mover(const EvictParams& params, int head) : p(params), kvh(head), stride(static_cast<uint32_t>(params.num_kv_heads) * PIECES * 16) {
        const int c = static_cast<int>(threadIdx.x) % kPerRow;
        base = static_cast<unsigned char*>(c < PIECES ? p.k_cache : p.v_cache) + (static_cast<int64_t>(kvh) * PIECES + c % PIECES) * 16;
    }
    __device__ __forceinline__ uint4* at(int row) const { return reinterpret_cast<uint4*>(base + static_cast<uint64_t>(static_cast<uint32_t>(row)) * stride); }
    template <int N> struct Set { uint4 v[N]; int to[N]; };
    template <int N> __device__ __forceinline__ void load(Set<N>& set, const int2* list, int count, int r0) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = r0 + i * kRows;
            const int2 row = r < count ? list[r] : make_int2(-1, -1);
            set.to[i] = row.y;
            set.v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row.x >= 0) set.v[i] = *at(row.x);
        }
    }
    template <int N> __device__ __forceinline__ void store(const Set<N>& set) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (set.to[i] >= 0) *at(set.to[i]) = set.v[i];
    }
    // `count` rows of the list, by the whole block.  ORDERED: a set is read before any of it is written; otherwise the next set is on its way meanwhile.
    template <bool ORDERED> __device__ __forceinline__ void move(const int2* list, int count) const {
        const int first = static_cast<int>(threadIdx.x) / kPerRow;
        if constexpr (ORDERED) {
            Set<8> set;
            for (int r0 = first; r0 - first < count; r0 += 8 * kRows) {   // (all threads take the same number of trips)
                load(set, list, count, r0);
                __syncthreads();
                store(set);
            }
        } else {
            Set<4> a, b;
            load(a, list, count, first);
            for (int r0 = first; r0 < count; r0 += 8 * kRows) {
                load(b, list, count, r0 + 4 * kRows);
                store(a);
                load(a, list, count, r0 + 8 * kRows);
                store(b);
            }
        }
        if (PARAMS) {
            for (int r0 = 0; r0 < count; r0 += kThreads) {
                const int r = r0 + static_cast<int>(threadIdx.x);
                const int2 row = r < count ? list[r] : make_int2(-1, -1);
                const int64_t from = static_cast<int64_t>(row.x) * p.num_kv_heads + kvh, to = static_cast<int64_t>(row.y) * p.num_kv_heads + kvh;
                const uint32_t k = row.x >= 0 ? p.k_params[from] : 0u, v = row.x >= 0 ? p.v_params[from] : 0u;
                if (ORDERED) __syncthreads();
                if (row.y >= 0) { p.k_params[to] = k; p.v_params[to] = v; }
            }
        }
    }
};

// PIECES: 16-byte pieces of a key's (value's) row of one head.
template <int PIECES, bool PARAMS>
__global__ void __launch_bounds__(kThreads, 2) evict_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sm = *reinterpret_cast<Shared*>(smem);
    pdl_wait_then_release();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pair = blockIdx.x / p.split, rank = blockIdx.x - pair * p.split;
    const int b = pair / p.num_kv_heads, kvh = pair - b * p.num_kv_heads;
    // (the first blocks' ids come with the context length)
    const bool there = tid < p.new_max_blocks && tid < p.max_blocks;
    const int64_t new_id = there ? p.new_tables[b * p.new_max_blocks + tid] : 0, old_id = there ? p.block_tables[b * p.max_blocks + tid] : 0;
    const int64_t ctx = p.context_lens[b], cap = p.max_blocks * p.block_size;
    Choice c{};
    c.n = static_cast<int>(ctx < 0 ? 0 : ctx < cap ? ctx : cap);
    const int64_t wrow = p.rows != nullptr ? p.rows[b] : b;
    const bool live = wrow >= 0 && wrow < p.num_rows, all = !live || c.n <= p.budget;
    const int new_n = all ? c.n : static_cast<int>(p.budget);
    if (kvh == 0 && rank == 0 && tid == 0) {
        if (p.context_lens.wide) static_cast<int64_t*>(p.new_lens)[b] = new_n;
        else static_cast<int32_t*>(p.new_lens)[b] = new_n;
    }
    if (!live) return;
    const float* weights = p.weights + (wrow * p.num_kv_heads + kvh) * p.row_keys;
    float* new_weights = p.new_weights + (wrow * p.num_kv_heads + kvh) * p.row_keys;
    // In place, if a block is its own successor, or if the weights are: whoever reads a place has to have done so before it is written.
    bool same = weights == new_weights || (there && static_cast<int64_t>(tid) * p.block_size < new_n && new_id == old_id);
    for (int i = tid + kThreads; i < p.new_max_blocks && i < p.max_blocks && static_cast<int64_t>(i) * p.block_size < new_n; i += kThreads)
        same |= p.new_tables[b * p.new_max_blocks + i] == p.block_tables[b * p.max_blocks + i];
    const bool ordered = __syncthreads_or(same);
    if (ordered && rank > 0) return;
    c.lo = all ? c.n : static_cast<int>(p.sinks);
    c.hi = all ? c.n : c.n - static_cast<int>(p.recent);
    c.take = all ? 0 : static_cast<int>(p.budget - p.sinks - p.recent);
    if (c.take > 0) choose(weights, c, sm, p.cached);
    const Mover<PIECES, PARAMS> mover(p, kvh);
    if (ordered) {
        int2 at = make_int2(0, 0);         // keys that stay without regard to ties, and ties, so far
        for (int pos = tid; pos - tid < c.n; pos += kTile) {
            const float w = pos < c.n ? weights[pos] : 0.0f;
            const int2 s = c.of(sm, weights, pos);
            int2 total;
            const int2 place = scan(s, sm, total);
            const int ties = at.y + place.y, to = at.x + place.x + min(ties, c.ties), base = at.x + min(at.y, c.ties);
            if (s.x != 0 || (s.y != 0 && ties < c.ties)) {
                const int from_row = row_of(p, p.block_tables, p.max_blocks, b, pos), to_row = row_of(p, p.new_tables, p.new_max_blocks, b, to);
                sm.list[to - base] = make_int2(from_row, from_row != to_row ? to_row : -1);
                new_weights[to] = w;       // (all weights of this tile and of those before have been read)
            }
            at.x += total.x; at.y += total.y;
            __syncthreads();
            mover.template move<true>(sm.list, at.x + min(at.y, c.ties) - base);
            __syncthreads();
        }
        for (int64_t i = new_n + tid; i < p.row_keys; i += kThreads) new_weights[i] = 0.0f;
        return;
    }
    // What stays of every tile; of longer contexts of `per` tiles together.
    const int per = (c.n + kMaxTiles * kWarpTile - 1) / (kMaxTiles * kWarpTile), keys = per * kWarpTile, tiles = c.n > 0 ? (c.n + keys - 1) / keys : 0;
    constexpr int kEach = kWarpTile / 32;
    for (int t = warp; t < tiles; t += kWarps) {
        int2 sum = make_int2(0, 0);
        for (int pos0 = t * keys; pos0 < min(c.n, (t + 1) * keys); pos0 += kWarpTile) {
            int2 s[kEach];
#pragma unroll
            for (int j = 0; j < kEach; ++j) s[j] = c.of(sm, weights, pos0 + 32 * j + lane);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                sum.x += __popc(__ballot_sync(0xffffffffu, s[j].x != 0));
                sum.y += __popc(__ballot_sync(0xffffffffu, s[j].y != 0));
            }
        }
        if (lane == 0) sm.tiles[t] = sum;
    }
    __syncthreads();
    {   // before every tile
        constexpr int kOwn = kMaxTiles / kThreads;
        int2 own[kOwn], sum = make_int2(0, 0), total;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int t = tid * kOwn + i;
            own[i] = t < tiles ? sm.tiles[t] : make_int2(0, 0);
            sum.x += own[i].x; sum.y += own[i].y;
        }
        int2 before = scan(sum, sm, total);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (tid * kOwn + i < tiles) sm.tiles[tid * kOwn + i] = before;
            before.x += own[i].x; before.y += own[i].y;
        }
        if (tid == 0) sm.listed = 0;
        __syncthreads();
    }
    const uint32_t below = (1u << lane) - 1u;
    for (int t0 = rank; t0 < tiles; t0 += kWarps * p.split) {   // a tile of every warp
        const int t = t0 + warp * p.split;
        int2 at = t < tiles ? sm.tiles[t] : make_int2(0, 0);
        for (int i = 0; i < per; ++i) {
            const int pos0 = t < tiles ? t * keys + i * kWarpTile : c.n;
            int2 s[kEach];
            uint32_t stay[kEach], tie[kEach];
            const int2 was = at;
#pragma unroll
            for (int j = 0; j < kEach; ++j) s[j] = c.of(sm, weights, pos0 + 32 * j + lane);
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                stay[j] = __ballot_sync(0xffffffffu, s[j].x != 0);
                tie[j] = __ballot_sync(0xffffffffu, s[j].y != 0);
                at.x += __popc(stay[j]); at.y += __popc(tie[j]);
            }
            const int base = was.x + min(was.y, c.ties), count = at.x + min(at.y, c.ties) - base;
            int slot = 0;
            if (lane == 0 && count > 0) slot = atomicAdd(&sm.listed, count);   // (in whatever order)
            slot = __shfl_sync(0xffffffffu, slot, 0) - base;
            int2 here = was;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int pos = pos0 + 32 * j + lane, ties = here.y + __popc(tie[j] & below), to = here.x + __popc(stay[j] & below) + min(ties, c.ties);
                if (s[j].x != 0 || (s[j].y != 0 && ties < c.ties)) {
                    sm.list[slot + to] = make_int2(row_of(p, p.block_tables, p.max_blocks, b, pos), row_of(p, p.new_tables, p.new_max_blocks, b, to));
                    new_weights[to] = weights[pos];
                }
                here.x += __popc(stay[j]); here.y += __popc(tie[j]);
            }
            __syncthreads();
            mover.template move<false>(sm.list, sm.listed);
            __syncthreads();
            if (tid == 0) sm.listed = 0;
            __syncthreads();
        }
    }
    for (int64_t i = new_n + tid + rank * kThreads; i < p.row_keys; i += p.split * kThreads) new_weights[i] = 0.0f;
}

template <int PIECES, bool PARAMS>
cudaError_t launch_typed(const EvictParams& p, unsigned grid, cudaStream_t stream) {
    static std::atomic<bool> attr_done[64] = {};  // per device; the attribute call is idempotent
    int device = 0;
    cudaGetDevice(&device);
    if (device < 0 || device >= 64 || !attr_done[device]) {
        const cudaError_t e = cudaFuncSetAttribute(evict_kernel<PIECES, PARAMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes(kCachedAlone));
        if (e != cudaSuccess) return e;
        if (device >= 0 && device < 64) attr_done[device] = true;
    }
    return launch_pdl(evict_kernel<PIECES, PARAMS>, dim3(grid), dim3(kThreads), shared_bytes(p.cached), stream, p);
}

}  // namespace

int launch_evict(const EvictArgs& a) {
    if (a.batch * a.num_kv_heads > 0x7fffffffLL || a.max_blocks * a.block_size > (1LL << 30) || a.new_max_blocks * a.block_size > (1LL << 30) ||
        a.num_cache_blocks > 0x7fffffffLL / a.block_size)
        return fail(NVK_ERR_UNSUPPORTED, "evict_kvcache: batch, block table or cache too large");
    // As many blocks to a pair as there are places for, and no more than there are pairs of tiles; more than that do not even out contexts of different lengths
    // (256 pairs of 1000 to 8192 keys: one block each 107.2 us, two 108.9, four 110.6, eight 137.9).
    // Two to an SM where there is enough to do, since the second costs some 3 us whatever there is.  One to an SM (us, one / two, a third of the keys kept)
    //   * up to 300000 keys of all pairs' tables: 16 pairs of 4096 12.7 / 15.7, 64 of 1024 11.1 / 13.6, 72 of 4096 29.2 / 30.0; but 40 of 8192 36.7 / 34.2;
    //   * up to 150000 with more than half as many pairs as SMs, which then have one block each: 144 of 1024 16.2 / 17.6; but 88 of 3000 31.7 / 27.5;
    //   * up to 100000 over 4-bit rows: 48 of 2048 17.4 / 20.3, 24 of 4096 17.7 / 20.9; but 40 of 4096 26.4 / 25.1, 144 of 2048 35.3 / 31.8;
    //   * where that lets few pairs of long contexts keep their orders.
    const int64_t pairs = a.batch * a.num_kv_heads, tokens = a.max_blocks * a.block_size, most = (tokens + 2 * kWarpTile - 1) / (2 * kWarpTile);
    const bool alone = tokens > kCached && 2 * pairs <= kSmCount;
    const bool single = alone || pairs * tokens <= (a.k_params != nullptr ? 100000 : 2 * pairs <= kSmCount ? 300000 : 150000);
    const int cached = alone ? kCachedAlone : kCached;
    const int split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((single ? 1 : 2) * kSmCount / pairs, most), kMaxSplit)));
    const EvictParams p{a.k_cache, a.v_cache, static_cast<uint32_t*>(a.k_params), static_cast<uint32_t*>(a.v_params), a.weights, a.new_weights, a.rows,
                        a.context_lens, a.block_tables, a.new_tables, a.new_lens, a.num_rows, a.row_keys, a.max_blocks, a.new_max_blocks,
                        a.num_cache_blocks, a.budget, a.sinks, a.recent, a.num_kv_heads, a.block_size, split, cached, FastDiv(static_cast<uint32_t>(a.block_size))};
    const unsigned grid = static_cast<unsigned>(pairs * split);
    const cudaError_t e = a.k_params != nullptr ? launch_typed<kDim / 2 / 16, true>(p, grid, a.stream) : launch_typed<kDim * 2 / 16, false>(p, grid, a.stream);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "evict_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("evict_kernel launch");
}

}  // namespace nvk
