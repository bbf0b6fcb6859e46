// The metadata of a step on the GPU: block tables, context lengths, cumulative lengths, positions and slots from the lengths of the step's requests, with
// new cache blocks taken from a list of free ones; and the blocks of requests that ended back onto that list.  What the reference's ModelRunner builds on
// the host for every step (src/engine/model_runner.cpp:482-632, :748-769) and its BlockManager hands out.
//
// With old length l_b, n_b new tokens and blocks of s tokens, request b needs ceil((l_b + n_b) / s) - ceil(l_b / s) new blocks; the prefix sums of these
// say which of the free blocks are its own, and whether there are enough.  Sums over the batch, then every table entry and every token by itself.
//
// A call is bound by the trips to memory one after the other (row, its length and its blocks) and by the launch.  So every block does the sums over the whole batch for itself, so that
// nothing is handed over, and the blocks share out the table entries and the tokens.  Lengths and the count of free blocks may be updated in place, when every block has read them.  Where
// they are, the blocks are one cluster, whose first one writes them behind a barrier, up to four pieces of 16 bytes to a thread; beyond, and wherever the new ones are of their own, there
// are as many blocks as the work is worth, and what is updated in place follows in a kernel of one block.  us, in a cluster / by many blocks (and that kernel), behind a small copy: 256 requests, table
// rows of 33 int32 (8448 pieces) 4.1 / 5.2, 16 of 2304 new tokens, int64 (36864 pieces) 5.2 / 5.4, 1024 with rows of 33 6.2 / 7.1, of 129 (132096) 8.1 / 7.2.  Of their own: 3.8, 3.9, 5.9,
// 6.0; steps one after the other, a decode step of one request 2.8, of 256 (rows of 32) 3.4, 1024 requests of rows of 512 6.5 (2.1 MB written), 8192 of 33 26 us (every block goes through
// the batch 1024 requests at a time, with two barriers each).  Up to 256 requests by blocks of 256 threads (a scan over
// 1024 takes 1 us more: 256 requests, rows of 33, 4.7), beyond by 1024.
#include "nvk_internal.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace nvk {
namespace {

constexpr int kFewThreads = 256, kManyThreads = 1024;
constexpr int kMaxBlocks = 16;            // of a cluster (not portable, but there on every B200)
constexpr int kMaxBatch = 8192;           // 24 bytes of shared memory for each
constexpr int kAhead = 2;                 // pieces of table rows that a thread has under way
constexpr int64_t kClusterPieces = 4;     // of 16 bytes to a thread, up to which one cluster takes a step that updates in place
constexpr uint32_t kMost = 0x7fffffffu, kNone = 0xffffffffu;

// Sums of numbers below 2^31, held at 2^31 - 1: lengths come from the device, and no sum of them may wrap round.
__device__ __forceinline__ uint32_t add_held(uint32_t a, uint32_t b) { return min(a + b, kMost); }
template <typename E> __device__ __forceinline__ uint32_t held(E v, uint32_t most = kMost) {   // within 0 .. most
    return v < 0 ? 0u : v > static_cast<E>(most) ? most : static_cast<uint32_t>(v);
}

// Sums of three numbers over the threads before this one and, in `total`, over all.
struct Three { uint32_t a, b, c; };
__device__ __forceinline__ Three add_held(Three x, Three y) { return Three{add_held(x.a, y.a), add_held(x.b, y.b), add_held(x.c, y.c)}; }
__device__ __forceinline__ Three shfl(Three x, int lane) {
    return Three{__shfl_sync(0xffffffffu, x.a, lane), __shfl_sync(0xffffffffu, x.b, lane), __shfl_sync(0xffffffffu, x.c, lane)};
}
__device__ __forceinline__ Three scan_warp(Three x, int lane) {   // with its own
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const Three y{__shfl_up_sync(0xffffffffu, x.a, d), __shfl_up_sync(0xffffffffu, x.b, d), __shfl_up_sync(0xffffffffu, x.c, d)};
        if (lane >= d) x = add_held(x, y);
    }
    return x;
}
__device__ __forceinline__ Three before_in_warp(Three x, int lane) {
    const Three y = shfl(x, max(lane - 1, 0));
    return lane > 0 ? y : Three{0u, 0u, 0u};
}
template <int WARPS> __device__ __forceinline__ Three scan_block(Three v, Three& total, Three* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Three x = scan_warp(v, lane);
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    const Three w = scan_warp(lane < WARPS ? s_warp[lane] : Three{0u, 0u, 0u}, lane);
    total = shfl(w, 31);
    const Three others = shfl(w, max(warp - 1, 0)), before = before_in_warp(x, lane);
    __syncthreads();                      // (s_warp is used again)
    return warp > 0 ? add_held(before, others) : before;
}

// All blocks of the cluster arrive when they have read what is updated in place; the first one, which writes it, waits at its end.  The others' reads have to come before its
// writes, so that they arrive with .release (the wait acquires); they have nothing written by then that this would wait for.  The first block's own arrival orders nothing: what it
// has written by then nobody of the cluster reads, and to wait for it took 1 us of the 5 of 256 requests; its own reads come before the block's barrier that follows.  Not the .aligned
// forms, which a warp has to execute together: its threads come here from loops and branches of their own.
__device__ __forceinline__ void cluster_arrive(bool first_block) {
    if (first_block) asm volatile("barrier.cluster.arrive.relaxed;\n" ::: "memory");
    else asm volatile("barrier.cluster.arrive.release;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory"); }

// What is known of the requests of a step, in shared memory.
struct Request {
    int row;      // of the table of requests; -1: padding
    int had;      // blocks in use before
    int used;     // and after; 0: there is no place for it
    int first;    // the first of its new blocks among those of the step
};
struct Tokens {
    int cu;       // the first one
    int old_len;  // -1: there is no place for it
};

template <typename E> struct StepParams {
    const E *new_lens, *rows, *lens, *free_blocks, *free_count;
    E *request_blocks, *block_tables, *context_lens, *cu_q, *cu_k, *positions, *slots, *new_lens_out, *new_count;
    int64_t num_rows, row_blocks, num_free, num_cache_blocks, num_tokens;
    int batch, max_blocks;
    int token_pieces;                     // positions and slots are written 16 bytes at a time
    int wide;                             // many blocks instead of one cluster; what is updated in place is left to commit_step_kernel
    uint32_t capacity;                    // tokens of a request, at most
    FastDiv by_block, by_pieces;          // by_pieces: of a table row
};

__device__ __forceinline__ uint32_t blocks_of(const FastDiv& by_block, uint32_t tokens) { return by_block.div(tokens + by_block.d - 1); }

// V numbers next to each other.
template <typename E, int V> struct alignas(V * sizeof(E)) Entries { E e[V]; };

template <typename E, int V, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) step_metadata_kernel(const __grid_constant__ StepParams<E> p) {
    constexpr int kWarps = THREADS / 32, kTokens = 4;
    constexpr bool kRounds = THREADS > kFewThreads;   // (few threads: where there are no more requests than those)
    extern __shared__ __align__(16) Request s_request[];
    Tokens* s_token = reinterpret_cast<Tokens*>(s_request + p.batch);
    __shared__ Three s_warp[kWarps];
    __shared__ uint32_t s_tokens, s_taken;
    __shared__ E s_free[THREADS];         // the blocks that are taken first
    using Piece = Entries<E, V>;
    pdl_wait_then_release();
    const int tid = threadIdx.x, lane = tid & 31;
    const bool first_block = blockIdx.x == 0;
    const int threads = static_cast<int>(gridDim.x) * THREADS, me = static_cast<int>(blockIdx.x) * THREADS + tid;
    const int pieces = p.batch * static_cast<int>(p.by_pieces.d);
    // What needs no other number first, then what needs those: two trips to memory before the sums.
    auto known = [&](E row) { return row >= 0 && row < p.num_rows; };
    auto row_of = [&](int b) { return p.rows != nullptr ? p.rows[b] : static_cast<E>(b); };
    const E count_in = p.free_count[0];
    E row0 = -1, new0 = 0, len0 = 0, free0 = 0, piece_row[kAhead];
    if (tid < p.batch) {
        row0 = row_of(tid);
        new0 = p.new_lens[tid];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) piece_row[u] = me + u * threads < pieces ? row_of(static_cast<int>(p.by_pieces.div(me + u * threads))) : static_cast<E>(-1);
    if (known(row0)) len0 = p.lens[row0];
    // And of the requests that follow, THREADS at a time: two rounds ahead the row and the new tokens, one round ahead the length.
    E row1 = -1, new1 = 0;
    auto load_row = [&](int b) {
        row1 = b < p.batch ? row_of(b) : static_cast<E>(-1);
        new1 = b < p.batch ? p.new_lens[b] : static_cast<E>(0);
    };
    if constexpr (kRounds) load_row(tid + THREADS);
    // The first pieces of the table rows: which of their entries count is seen later.
    auto load = [&](int i, E row, Piece& to) {
        const int64_t j = static_cast<int64_t>(i - static_cast<int>(p.by_pieces.div(i)) * static_cast<int>(p.by_pieces.d)) * V;
        if (j < p.row_blocks) to = *reinterpret_cast<const Piece*>(p.request_blocks + static_cast<int64_t>(row) * p.row_blocks + j);
    };
    Piece piece[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
        if (known(piece_row[u])) load(me + u * threads, piece_row[u], piece[u]);
    const uint32_t count = held(count_in, static_cast<uint32_t>(min(p.num_free, static_cast<int64_t>(kMost))));
    if (static_cast<uint32_t>(tid) < count) free0 = p.free_blocks[static_cast<int64_t>(count) - 1 - tid];
    // Where there is a thread for every token: token t is most often request t's only one, in a decode step.  The block that it would then be in, while the sums are taken.
    const bool single = p.num_tokens <= threads;
    E guess = -1;
    if (single && me < p.batch && me < p.num_tokens) {
        const E row = first_block ? row0 : row_of(me);
        if (known(row)) {
            const uint32_t j = p.by_block.div(held(first_block ? len0 : p.lens[row]));
            if (j < p.row_blocks) guess = p.request_blocks[static_cast<int64_t>(row) * p.row_blocks + j];
        }
    }
    if (tid == 0) s_taken = 0;
    // The requests, THREADS at a time (up to 32 by one warp, without barriers).
    Three base{0u, 0u, 0u};               // tokens, new blocks, keys
    uint32_t taken = 0;
    auto requests = [&](int b0, auto scan) {
        const int b = b0 + tid;
        const bool there = b < p.batch;
        const E row = row0, n_in = new0, len_in = len0;
        if (kRounds && b0 + THREADS < p.batch) {
            row0 = row1;
            new0 = new1;
            len0 = known(row0) ? p.lens[row0] : static_cast<E>(0);
            load_row(b + 2 * THREADS);
        }
        const bool ours = known(row);
        const uint32_t len = held(len_in), n = held(n_in);
        const bool fits = ours && len <= p.capacity && n <= p.capacity - len;
        const uint32_t had = fits ? blocks_of(p.by_block, len) : 0u, used = fits ? blocks_of(p.by_block, len + n) : 0u, need = used - had;
        Three total;
        Three at = add_held(scan(Three{n, need, fits ? len + n : 0u}, total), base);
        const bool placed = fits && (need == 0 || add_held(at.b, need) <= count);
        const uint32_t ctx = placed ? len + n : 0;
        if (placed && need > 0) taken = max(taken, add_held(at.b, need));
        Three upto = add_held(base, total);
        if (upto.b > count) {             // not all have a place: the sum of the contexts again
            Three keys;
            at.c = add_held(base.c, scan(Three{ctx, 0u, 0u}, keys).a);
            upto.c = add_held(base.c, keys.a);
        }
        base = upto;
        if (there) {
            s_request[b] = Request{ours ? static_cast<int>(row) : -1, placed ? static_cast<int>(had) : 0, placed ? static_cast<int>(used) : 0, static_cast<int>(at.b)};
            s_token[b] = Tokens{static_cast<int>(at.a), placed ? static_cast<int>(len) : -1};
        }
        if (first_block && there) {       // (outputs of their own: nobody reads them here)
            p.context_lens[b] = ctx;
            if (p.cu_q != nullptr) p.cu_q[b + 1] = add_held(at.a, n);
            if (p.cu_k != nullptr) p.cu_k[b + 1] = add_held(at.c, ctx);
        }
    };
    if (p.batch <= 32) {
        if (tid < 32) {
            requests(0, [&](Three v, Three& total) {
                const Three x = scan_warp(v, lane);
                total = shfl(x, 31);
                return before_in_warp(x, lane);
            });
        }
    } else {
        for (int b0 = 0; b0 < p.batch; b0 += THREADS) requests(b0, [&](Three v, Three& total) { return scan_block<kWarps>(v, total, s_warp); });
    }
    s_free[tid] = free0;
    if (tid == 0) {
        s_tokens = base.a;
        if (first_block && p.cu_q != nullptr) p.cu_q[0] = 0;
        if (first_block && p.cu_k != nullptr) p.cu_k[0] = 0;
    }
    if (first_block) {
        if (p.batch > 32) __syncthreads();   // (s_taken is zero)
        else __syncwarp();
        if (taken > 0) atomicMax(&s_taken, taken);
    }
    if (first_block && p.new_lens_out != p.lens) {   // (whole; the new ones follow)
        for (int64_t i = tid; i < p.num_rows; i += THREADS) p.new_lens_out[i] = p.lens[i];
    }
    if (!p.wide && gridDim.x > 1) cluster_arrive(first_block);
    __syncthreads();
    // From here on lengths and count are no longer read.
    const uint32_t tokens = s_tokens;
    auto new_block = [&](uint32_t i) { return i < THREADS ? s_free[i] : p.free_blocks[static_cast<int64_t>(count) - 1 - i]; };
    auto end_of = [&](int b) { return b + 1 < p.batch ? static_cast<uint32_t>(s_token[b + 1].cu) : tokens; };
    // Table entries.
    for (int i0 = me; i0 < pieces; i0 += kAhead * threads) {
        if (i0 != me) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + u * threads;
                if (i < pieces) {
                    const int row = s_request[p.by_pieces.div(i)].row;
                    if (row >= 0) load(i, row, piece[u]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * threads;
            if (i >= pieces) break;
            const int b = static_cast<int>(p.by_pieces.div(i)), j0 = (i - b * static_cast<int>(p.by_pieces.d)) * V;
            const Request r = s_request[b];
            if (j0 >= r.used) {
#pragma unroll
                for (int k = 0; k < V; ++k) piece[u].e[k] = 0;
            } else if (j0 + V > r.had) {                  // (not all of it was in use)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int j = j0 + k;
                    if (j >= r.had) piece[u].e[k] = 0;
                    if (j >= r.had && j < r.used) {
                        piece[u].e[k] = new_block(r.first + (j - r.had));
                        p.request_blocks[r.row * p.row_blocks + j] = piece[u].e[k];
                    }
                }
            }
            *reinterpret_cast<Piece*>(p.block_tables + static_cast<int64_t>(i) * V) = piece[u];   // (rows are whole pieces)
        }
    }
    // The last request that begins at or before token t (those of no tokens begin where the next one does); of single tokens it is request t.
    auto request_of = [&](int64_t t) {
        int lo = 0, hi = p.batch;
        if (t < p.batch && s_token[t].cu == t && end_of(static_cast<int>(t)) == t + 1) return static_cast<int>(t);
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_token[mid].cu <= t) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    auto block_of = [&](const Request& r, uint32_t j) {
        return static_cast<int64_t>(j < static_cast<uint32_t>(r.had) ? p.request_blocks[r.row * p.row_blocks + j] : new_block(r.first + (j - r.had)));
    };
    auto slot_of = [&](int64_t id, uint32_t off) { return id >= 0 && id < p.num_cache_blocks ? static_cast<E>(id * p.by_block.d + off) : static_cast<E>(-1); };
    if (single) {
        if (me < p.num_tokens) {
            E pos = 0, slot = -1;
            if (static_cast<uint32_t>(me) < tokens) {
                const int b = request_of(me);
                const Tokens x = s_token[b];
                if (x.old_len >= 0) {
                    const Request r = s_request[b];
                    const uint32_t at = x.old_len + (me - x.cu), j = p.by_block.div(at);
                    const bool guessed = b == me && x.cu == me && j < static_cast<uint32_t>(r.had);
                    pos = static_cast<E>(at);
                    slot = slot_of(guessed ? static_cast<int64_t>(guess) : block_of(r, j), at - j * p.by_block.d);
                }
            }
            p.positions[me] = pos;
            p.slots[me] = slot;
        }
    } else {
        // Four next to each other a thread.
        for (int64_t t0 = static_cast<int64_t>(me) * kTokens; t0 < p.num_tokens; t0 += static_cast<int64_t>(threads) * kTokens) {
            int lo = t0 < tokens ? request_of(t0) : 0;
            uint32_t at[kTokens], off[kTokens];
            int64_t id[kTokens];
            const Tokens x = s_token[lo];
            const uint32_t at0 = x.old_len + static_cast<uint32_t>(t0 - x.cu), j0 = p.by_block.div(at0 & kMost), off0 = at0 - j0 * p.by_block.d;
            if (t0 + kTokens <= tokens && x.old_len >= 0 && end_of(lo) >= t0 + kTokens && off0 + kTokens <= p.by_block.d) {   // all in one block
                const int64_t one = block_of(s_request[lo], j0);
#pragma unroll
                for (int k = 0; k < kTokens; ++k) { at[k] = at0 + k; off[k] = off0 + k; id[k] = one; }
            } else {
#pragma unroll
                for (int k = 0; k < kTokens; ++k) {
                    const int64_t t = t0 + k;
                    at[k] = off[k] = 0;
                    id[k] = -1;
                    if (t < tokens && t < p.num_tokens) {
                        while (end_of(lo) <= t) ++lo;     // (t < tokens, where the last one ends)
                        const Tokens y = s_token[lo];
                        if (y.old_len >= 0) {
                            at[k] = y.old_len + static_cast<uint32_t>(t - y.cu);
                            const uint32_t j = p.by_block.div(at[k]);
                            off[k] = at[k] - j * p.by_block.d;
                            id[k] = block_of(s_request[lo], j);
                        }
                    }
                }
            }
            constexpr int kPiece = 16 / sizeof(E);
            if (p.token_pieces && t0 + kTokens <= p.num_tokens) {
#pragma unroll
                for (int k0 = 0; k0 < kTokens; k0 += kPiece) {
                    Entries<E, kPiece> pos, slot;
#pragma unroll
                    for (int k = 0; k < kPiece; ++k) {
                        pos.e[k] = static_cast<E>(at[k0 + k]);
                        slot.e[k] = slot_of(id[k0 + k], off[k0 + k]);
                    }
                    *reinterpret_cast<Entries<E, kPiece>*>(p.positions + t0 + k0) = pos;
                    *reinterpret_cast<Entries<E, kPiece>*>(p.slots + t0 + k0) = slot;
                }
            } else {
#pragma unroll
                for (int k = 0; k < kTokens; ++k) {
                    if (t0 + k < p.num_tokens) {
                        p.positions[t0 + k] = static_cast<E>(at[k]);
                        p.slots[t0 + k] = slot_of(id[k], off[k]);
                    }
                }
            }
        }
    }
    if (first_block) {
        if (!p.wide && gridDim.x > 1) cluster_wait();
        if (!p.wide || p.new_lens_out != p.lens) {
            for (int b = tid; b < p.batch; b += THREADS) {
                const Tokens x = s_token[b];
                if (x.old_len >= 0) p.new_lens_out[s_request[b].row] = x.old_len + (end_of(b) - x.cu);
            }
        }
        if (tid == 0 && (!p.wide || p.new_count != p.free_count)) p.new_count[0] = count - s_taken;
    }
}

// After the many blocks of a large step: the lengths and the count that are updated in place.  A request with a place has a context length of its new length; what it
// took is what that needs beyond its old one.  One block, one pass.
template <typename E> __global__ void __launch_bounds__(kManyThreads) commit_step_kernel(const __grid_constant__ StepParams<E> p) {
    __shared__ uint32_t s_taken;
    pdl_wait_then_release();
    if (threadIdx.x == 0) s_taken = 0;
    __syncthreads();
    uint32_t taken = 0;
    // `each` requests of a thread (where new lengths are of their own, the first kernel has set them: lens are still the old ones)
    auto commit = [&](auto each) {
        constexpr int kEach = decltype(each)::value;
        uint32_t ctx[kEach], old[kEach];
        int row[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int b = threadIdx.x + i * kManyThreads;
            const E id = b >= p.batch ? static_cast<E>(-1) : p.rows != nullptr ? p.rows[b] : static_cast<E>(b);
            ctx[i] = b < p.batch ? static_cast<uint32_t>(p.context_lens[b]) : 0u;
            row[i] = id >= 0 && id < p.num_rows ? static_cast<int>(id) : -1;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) old[i] = ctx[i] > 0 && row[i] >= 0 ? held(p.lens[row[i]]) : kNone;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (old[i] == kNone) continue;
            taken += blocks_of(p.by_block, ctx[i]) - blocks_of(p.by_block, old[i]);
            if (p.new_lens_out == p.lens) p.new_lens_out[row[i]] = ctx[i];
        }
    };
    if (p.batch <= kManyThreads) commit(std::integral_constant<int, 1>());
    else commit(std::integral_constant<int, kMaxBatch / kManyThreads>());
    taken = __reduce_add_sync(0xffffffffu, taken);
    if ((threadIdx.x & 31) == 0) atomicAdd(&s_taken, taken);
    __syncthreads();
    if (threadIdx.x == 0 && p.new_count == p.free_count)
        p.new_count[0] = held(p.free_count[0], static_cast<uint32_t>(min(p.num_free, static_cast<int64_t>(kMost)))) - s_taken;
}

template <typename E> struct ReleaseParams {
    const E *rows, *first_blocks, *lens, *request_blocks, *free_count;
    E *free_blocks, *new_lens_out, *new_count;
    int64_t num_rows, row_blocks, num_free;
    int batch;
    uint32_t capacity;
    FastDiv by_block, by_chunks;          // by_chunks: of a request's blocks
};

// Blocks first_blocks[b] .. ceil(l_b / s) - 1 of each request behind those that are free already, in the requests' order.  A warp takes a chunk of a request's.
constexpr int kChunk = 256;
template <typename E>
__global__ void __launch_bounds__(kFewThreads) release_blocks_kernel(const __grid_constant__ ReleaseParams<E> p) {
    extern __shared__ __align__(16) Request s_request[];   // row, first of its blocks, how many, where they go
    __shared__ Three s_warp[kFewThreads / 32];
    pdl_wait_then_release();
    const int tid = threadIdx.x;
    const int threads = static_cast<int>(gridDim.x) * kFewThreads, me = static_cast<int>(blockIdx.x) * kFewThreads + tid;
    const E count_in = p.free_count[0];
    uint32_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kFewThreads) {
        const int b = b0 + tid;
        const bool there = b < p.batch;
        const E row = !there ? -1 : p.rows != nullptr ? p.rows[b] : static_cast<E>(b);
        const bool ours = there && row >= 0 && row < p.num_rows;
        const uint32_t first = ours && p.first_blocks != nullptr ? held(p.first_blocks[b]) : 0;
        const uint32_t used = blocks_of(p.by_block, ours ? held(p.lens[row], p.capacity) : 0);
        const uint32_t n = first < used ? used - first : 0;
        Three total;
        const Three at = scan_block<kFewThreads / 32>(Three{n, 0u, 0u}, total, s_warp);
        if (there) s_request[b] = Request{ours ? static_cast<int>(row) : -1, n > 0 ? static_cast<int>(first) : 0, static_cast<int>(n), static_cast<int>(add_held(at.a, base))};
        base = add_held(base, total.a);
    }
    const int64_t count = held(count_in, static_cast<uint32_t>(min(p.num_free, static_cast<int64_t>(kMost))));
    if (blockIdx.x == 0 && p.new_lens_out != p.lens) {
        for (int64_t i = tid; i < p.num_rows; i += kFewThreads) p.new_lens_out[i] = p.lens[i];
    }
    if (gridDim.x > 1) cluster_arrive(blockIdx.x == 0);
    __syncthreads();
    const int lane = tid & 31, chunks = static_cast<int>(p.by_chunks.d), units = p.batch * chunks;
    for (int i = me >> 5; i < units; i += threads >> 5) {
        const int b = static_cast<int>(p.by_chunks.div(i)), j0 = (i - b * chunks) * kChunk + lane;
        const Request r = s_request[b];
        if (r.row < 0) continue;
        const E* from = p.request_blocks + r.row * p.row_blocks + r.had;
        E id[kChunk / 32];
#pragma unroll
        for (int u = 0; u < kChunk / 32; ++u)
            if (j0 + u * 32 < r.used) id[u] = from[j0 + u * 32];
#pragma unroll
        for (int u = 0; u < kChunk / 32; ++u) {
            const int64_t to = count + r.first + j0 + u * 32;
            if (j0 + u * 32 < r.used && to < p.num_free) p.free_blocks[to] = id[u];
        }
    }
    if (blockIdx.x == 0) {
        if (gridDim.x > 1) cluster_wait();
        for (int b = tid; b < p.batch; b += kFewThreads) {
            const int row = s_request[b].row;
            if (row >= 0) p.new_lens_out[row] = 0;
        }
        if (tid == 0) p.new_count[0] = static_cast<E>(min(count + base, p.num_free));
    }
}

// One cluster of as many blocks as the work is worth, or, `wide`, so many blocks by themselves.
template <typename P>
int launch(const char* what, void (*kernel)(P), const P& p, int threads, int64_t blocks_worth, bool wide, std::atomic<bool> (&attr_done)[64], cudaStream_t stream) {
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64 && !attr_done[device]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBatch * static_cast<int>(sizeof(Request) + sizeof(Tokens)));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
        attr_done[device] = true;
    }
    int blocks = 1;
    if (wide) blocks = static_cast<int>(std::min<int64_t>(blocks_worth, kSmCount));
    else while (blocks < kMaxBlocks && blocks_worth > blocks) blocks *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = p.batch * (sizeof(Request) + sizeof(Tokens));
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = blocks > 1 && !wide ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "%s kernel launch: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

template <typename E, int V> int launch_step(const StepArgs& a, uint32_t capacity) {
    static std::atomic<bool> few_done[64] = {}, many_done[64] = {};
    auto in = [](const IndexArray& x) { return static_cast<const E*>(x.ptr); };
    auto out = [](void* x) { return static_cast<E*>(x); };
    StepParams<E> p{};
    p.new_lens = in(a.new_lens); p.rows = in(a.rows); p.lens = in(a.lens); p.free_blocks = static_cast<const E*>(a.free_blocks); p.free_count = in(a.free_count);
    p.request_blocks = out(a.request_blocks); p.block_tables = out(a.block_tables); p.context_lens = out(a.context_lens); p.cu_q = out(a.cu_q); p.cu_k = out(a.cu_k);
    p.positions = out(a.positions); p.slots = out(a.slots); p.new_lens_out = out(a.new_request_lens); p.new_count = out(a.new_free_count);
    p.num_rows = a.num_rows; p.row_blocks = a.row_blocks; p.num_free = a.num_free; p.num_cache_blocks = a.num_cache_blocks; p.num_tokens = a.num_tokens;
    p.batch = static_cast<int>(a.batch); p.max_blocks = static_cast<int>(a.max_blocks);
    p.capacity = capacity;
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    p.by_pieces = FastDiv(static_cast<uint32_t>(a.max_blocks / V));
    p.token_pieces = aligned_to(a.positions, 16) && aligned_to(a.slots, 16);
    const int64_t work = std::max(a.batch * a.max_blocks / V, a.num_tokens / 4);
    const bool in_place = p.new_lens_out == p.lens || p.new_count == p.free_count;
    const int threads = a.batch <= kFewThreads ? kFewThreads : kManyThreads;
    p.wide = in_place ? std::max(work, a.num_tokens * 2 * static_cast<int64_t>(sizeof(E)) / 16) > kClusterPieces * kMaxBlocks * threads : work > threads;
    const int rc = threads == kFewThreads ? launch("step_metadata", step_metadata_kernel<E, V, kFewThreads>, p, threads, work / threads + 1, p.wide, few_done, a.stream)
                                          : launch("step_metadata", step_metadata_kernel<E, V, kManyThreads>, p, threads, work / threads + 1, p.wide, many_done, a.stream);
    if (rc != NVK_OK || !p.wide || !in_place) return rc;
    const cudaError_t e = launch_pdl(commit_step_kernel<E>, dim3(1), dim3(kManyThreads), 0, a.stream, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "commit_step_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("commit_step_kernel launch");
}

template <typename E> int launch_release(const StepArgs& a, uint32_t capacity) {
    static std::atomic<bool> attr_done[64] = {};
    auto in = [](const IndexArray& x) { return static_cast<const E*>(x.ptr); };
    ReleaseParams<E> p{};
    p.rows = in(a.rows); p.first_blocks = in(a.first_blocks); p.lens = in(a.lens); p.request_blocks = static_cast<const E*>(a.request_blocks); p.free_count = in(a.free_count);
    p.free_blocks = static_cast<E*>(a.free_blocks); p.new_lens_out = static_cast<E*>(a.new_request_lens); p.new_count = static_cast<E*>(a.new_free_count);
    p.num_rows = a.num_rows; p.row_blocks = a.row_blocks; p.num_free = a.num_free;
    p.batch = static_cast<int>(a.batch);
    p.capacity = capacity;
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    p.by_chunks = FastDiv(static_cast<uint32_t>((a.row_blocks + kChunk - 1) / kChunk));
    return launch("release_blocks", release_blocks_kernel<E>, p, kFewThreads, a.batch * p.by_chunks.d * 32 / kFewThreads + 1, false, attr_done, a.stream);
}

}  // namespace

int launch_step_metadata(const StepArgs& a) {
    if (a.batch > kMaxBatch) return fail(NVK_ERR_UNSUPPORTED, "step_metadata: at most %d requests (got %lld)", kMaxBatch, static_cast<long long>(a.batch));
    // (entries are counted in 32 bits, and beyond the last one by as many as all threads take at a time; lengths as well, and beyond the longest by a block)
    const int64_t blocks = std::min(a.row_blocks, a.max_blocks), most = (1LL << 31) - 1 - a.block_size, ahead = kAhead * kSmCount * kManyThreads;
    if (a.max_blocks > ((1LL << 31) - ahead) / std::max<int64_t>(a.batch, 1) || a.num_rows > most) return fail(NVK_ERR_UNSUPPORTED, "step_metadata: too many requests or table entries");
    const uint32_t capacity = static_cast<uint32_t>(blocks <= most / a.block_size ? blocks * a.block_size : most);
    // Table rows in pieces of 16 bytes where both tables' rows are whole ones.
    const int v = a.wide ? 2 : 4;
    const bool pieces = a.max_blocks % v == 0 && a.row_blocks % v == 0 && aligned_to(a.block_tables, 16) && aligned_to(a.request_blocks, 16);
    if (a.wide) return pieces ? launch_step<int64_t, 2>(a, capacity) : launch_step<int64_t, 1>(a, capacity);
    return pieces ? launch_step<int32_t, 4>(a, capacity) : launch_step<int32_t, 1>(a, capacity);
}

int launch_release_blocks(const StepArgs& a) {
    if (a.batch > kMaxBatch) return fail(NVK_ERR_UNSUPPORTED, "release_blocks: at most %d requests (got %lld)", kMaxBatch, static_cast<long long>(a.batch));
    const int64_t most = (1LL << 31) - 1 - a.block_size;
    if (a.row_blocks > ((1LL << 31) - 1) / kMaxBatch * kChunk || a.num_rows > most) return fail(NVK_ERR_UNSUPPORTED, "release_blocks: too many requests or blocks");
    const uint32_t capacity = static_cast<uint32_t>(a.row_blocks <= most / a.block_size ? a.row_blocks * a.block_size : most);
    return a.wide ? launch_release<int64_t>(a, capacity) : launch_release<int32_t>(a, capacity);
}

}  // namespace nvk
