// 8-bit paged KV cache with one scale for each (cache block, KV head): store by sequences, and the gather of whole contexts into dense 16-bit rows.  (Decode
// attention over this cache: CacheBlocks8 in decode_body.cuh.)  No counterpart in the reference, whose int8 cache has a scale for every token
// (src/kernels/kvcache.cu:222-296).
//
// Format: int8 or e4m3 elements [cache blocks, block_size, Hkv, 128] and fp32 scales [cache blocks, Hkv], powers of two: with A the largest |x| among a
// block's rows of a head,
//   scale = max(2^-126, the smallest 2^e with A <= top 2^e), top = 127 (int8) or 448 (e4m3);   element = x / scale, to nearest, ties to even.
// Rows join a block one after the other.  One that is larger than all before raises the scale from s to s', and the rows that are there become
// round(n s / s'): powers of two, because then n s / s' is a shift, a block that has grown by several factors is off by less than one step of the last scale
// (1/2 + 1/4 + ..), and no product with a scale rounds.  (By absmax / 127 a block would be rounded again with nearly every row that is larger by a little, off by half
// a step each time.)  The price is up to one bit of int8's seven; e4m3 loses nothing.  A block of which a row holds an infinity or a NaN gets a scale of NaN, and reads
// as NaN until it begins anew.
//
// The store goes by sequences, not by slots: rows that share a scale have to come together, and a block of threads finds those of one cache block from the lengths.
#include "nvk_internal.cuh"

#include <atomic>
#include <type_traits>

namespace nvk {
namespace {

constexpr int kDim = 128;
constexpr int kThreads = 256;
constexpr int kLanes = kDim / 8;          // 16-byte pieces (eight elements) of a 16-bit head vector
constexpr int kMaxSets = 16;              // (head, K or V) of a block of threads
constexpr int kPasses = 16;               // pieces of a thread of store_blocks_kernel, in registers or shared memory
constexpr int kTileRows = kThreads * kPasses / kLanes;   // rows of a head, or of several together, that a block of threads holds
constexpr int kTileBytes = kThreads * kPasses * 16;      // 64 KiB, three blocks to an SM

// Two elements of T as one register.
template <typename T> struct PairOf;
template <> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct PairOf<__half> { using type = __half2; };
template <typename T> __device__ __forceinline__ typename PairOf<T>::type as_pair(uint32_t w) { return *reinterpret_cast<const typename PairOf<T>::type*>(&w); }
template <typename P> __device__ __forceinline__ uint32_t as_word(P p) { return *reinterpret_cast<const uint32_t*>(&p); }

// The largest absolute values so far of the elements in both halves of a word, NaN if one is.
template <typename T> __device__ __forceinline__ uint32_t top_of(uint32_t top, uint32_t pair) { return as_word(__hmax2_nan(as_pair<T>(top), __habs2(as_pair<T>(pair)))); }
template <typename T> __device__ __forceinline__ uint32_t top_of(uint32_t top, const uint4& v) {
    return top_of<T>(top_of<T>(top_of<T>(top_of<T>(top, v.x), v.y), v.z), v.w);
}
// Of both halves, as a whole number: absolute values order like that, infinity and NaN above all.
__device__ __forceinline__ uint32_t halves_top(uint32_t top) { return max(top & 0x7fffu, (top >> 16) & 0x7fffu); }

template <typename T> __device__ __forceinline__ float2 floats_of(uint32_t w);
template <> __device__ __forceinline__ float2 floats_of<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 floats_of<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// The scale that a largest absolute value (16 bits of T) asks for.
template <typename T, bool FP8> __device__ __forceinline__ float scale_for(uint32_t top) {
    const uint32_t bits = __float_as_uint(floats_of<T>(top).x);
    if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // 127 = 1.984375 2^6, 448 = 1.75 2^8: a mantissa above that takes the next power of two.
    const int e = static_cast<int>(bits >> 23) - (FP8 ? 8 : 6) + ((bits & 0x7fffffu) > (FP8 ? 0x600000u : 0x7e0000u) ? 1 : 0);   // biased by 127
    return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}
// The larger of a block's scale and of what its new rows ask for; (no scale is negative, and NaN is above all others as a whole number).
__device__ __forceinline__ float larger(float a, float b) { return __int_as_float(max(__float_as_int(a), __float_as_int(b))); }

template <bool FP8> __device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    if constexpr (FP8) return pack_e4m3x4(a, b, c, d);
    else return pack_s8x4(__float2int_rn(a), __float2int_rn(b), __float2int_rn(c), __float2int_rn(d));
}
// Four elements as floats.
template <bool FP8> __device__ __forceinline__ float4 unpack4(uint32_t w) {
    if constexpr (FP8) {
        uint32_t lo, hi;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(lo) : "h"(static_cast<unsigned short>(w & 0xffffu)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(hi) : "h"(static_cast<unsigned short>(w >> 16)));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        // Bytes with their signs flipped, in the mantissa of 2^23, less 2^23 + 128.
        const uint32_t u = w ^ 0x80808080u;
        auto one = [&](uint32_t pick) { return __uint_as_float(__byte_perm(u, 0x4b000000u, pick)) - 8388736.0f; };
        return make_float4(one(0x7550), one(0x7551), one(0x7552), one(0x7553));
    }
}

// Bytes 0 of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); }
// Eight elements over the block's scale, `inv` = 1 / scale.  Products with a power of two are exact, and so
//   * F16 -> e4m3: in f16 (what gets lost below its smallest normal number is far below half of e4m3's smallest);
//   * F16 -> int8: one fma with 1536, whose spacing is 1, leaves the rounded number in the sum's low byte;
//   * BF16: the same in fp32 (12582912), two at a time.
// The f16 forms need `inv` to be a normal f16 number: scales from 2^-15 to 2^14.
template <typename T, bool FP8> __device__ __forceinline__ uint2 quantise8(const uint4& v, float inv, bool narrow) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (std::is_same<T, __half>::value) {
        if (narrow) {
            const __half2 by = __float2half2_rn(inv);
            uint32_t o[4];
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned short e;
                    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;\n" : "=h"(e) : "r"(as_word(__hmul2(as_pair<T>(w[i]), by))));
                    o[i] = e;
                }
                return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
            } else {
                const uint32_t magic = 0x66006600u;   // 1536
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = as_word(__hfma2(as_pair<T>(w[i]), by, as_pair<T>(magic)));
                return make_uint2(__byte_perm(o[0], o[1], 0x6420), __byte_perm(o[2], o[3], 0x6420));
            }
        }
    }
    if constexpr (FP8) {
        const float2 a = floats_of<T>(w[0]), b = floats_of<T>(w[1]), c = floats_of<T>(w[2]), d = floats_of<T>(w[3]);
        return make_uint2(pack4<FP8>(a.x * inv, a.y * inv, b.x * inv, b.y * inv), pack4<FP8>(c.x * inv, c.y * inv, d.x * inv, d.y * inv));
    } else {
        if (inv != inv) return make_uint2(0u, 0u);
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = floats_of<T>(w[i]);
            asm("{\n\t.reg .b64 x, y, m, d;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 m, {%5, %5};\n\tfma.rn.f32x2 d, x, y, m;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
                : "=r"(o[2 * i]), "=r"(o[2 * i + 1]) : "f"(f.x), "f"(f.y), "f"(inv), "f"(12582912.0f));
        }
        return make_uint2(low_bytes(o[0], o[1], o[2], o[3]), low_bytes(o[4], o[5], o[6], o[7]));
    }
}
__device__ __forceinline__ bool narrow_scale(float scale) { return scale >= 0x1p-15f && scale <= 0x1p14f; }

// Rows [0, rows) of a head in a cache block, elements times `ratio`, by thread t of n.
template <bool FP8> __device__ __forceinline__ void scale_rows(unsigned char* base, size_t stride, int rows, float ratio, int t, int n) {
    constexpr int kPieces = kDim / 16, kFlight = 8;
    for (int i0 = t; i0 < rows * kPieces; i0 += n * kFlight) {
        uint4 v[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int i = i0 + u * n;
            if (i < rows * kPieces) v[u] = *reinterpret_cast<const uint4*>(base + (i / kPieces) * stride + (i % kPieces) * 16);
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int i = i0 + u * n;
            if (i >= rows * kPieces) break;
            auto word = [&](uint32_t w) {
                const float4 f = unpack4<FP8>(w);
                return pack4<FP8>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
            };
            *reinterpret_cast<uint4*>(base + (i / kPieces) * stride + (i % kPieces) * 16) = make_uint4(word(v[u].x), word(v[u].y), word(v[u].z), word(v[u].w));
        }
    }
}

// cp_async16 of what is read once: it gives way first in L2, where the elements that are written stay for the gather or the attention that comes next.  (So do the gather's dense rows, which are
// too many to stay; together, a store of 36864 rows and a gather of 43008: 83.4 -> 77.8 us.)
__device__ __forceinline__ uint64_t read_once() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void cp_async16_once(uint32_t dst, const void* src, int src_bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;\n" ::"r"(dst), "l"(src), "r"(src_bytes), "l"(policy) : "memory");
}

struct StoreParams {
    const void* rows[2]; unsigned char* cache[2]; float* scale[2];   // of K and of V
    int64_t stride[2];                                               // elements from a token to the next
    IndexArray cu; IndexArray context_lens; IndexArray block_tables;
    int64_t total_q, max_blocks, num_cache_blocks;
    int num_seqs, num_kv_heads, block_size;
    int sets;                                                        // of a block of threads
    FastDiv by_block, by_sets;                                       // by_sets: 2 Hkv
};

// One new row for each sequence (1.4 us for one, 2.7 for 256 of 8 KV heads: latency): a warp takes one head of K or of V of one, and the whole block of threads the rows of those whose scale it raised.
template <typename T, bool FP8>
__global__ void __launch_bounds__(kThreads) store_row_kernel(const __grid_constant__ StoreParams p) {
    struct Raise { unsigned char* base; int rows; float ratio; };
    __shared__ Raise s_raise[kThreads / 32];
    pdl_wait_then_release();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t task = blockIdx.x * (kThreads / 32) + warp, all = static_cast<uint32_t>(p.num_seqs) * p.by_sets.d;
    const size_t row_bytes = static_cast<size_t>(p.num_kv_heads) * kDim;
    int raised = 0;
    if (task < all) {
        const int seq = static_cast<int>(p.by_sets.div(task)), set = static_cast<int>(task - seq * p.by_sets.d);
        const int which = set >= p.num_kv_heads ? 1 : 0, head = set - which * p.num_kv_heads;
        const IndexArray::Raw raw = p.context_lens.raw(seq);
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const T*>(p.rows[which]) + seq * p.stride[which] + head * kDim + lane * 4);
        const int64_t pos = p.context_lens.value(raw) - 1;
        if (pos >= 0 && pos < p.max_blocks * p.block_size) {
            const int blk = static_cast<int>(p.by_block.div(static_cast<uint32_t>(pos))), row = static_cast<int>(pos) - blk * p.block_size;
            const int64_t id = p.block_tables[seq * p.max_blocks + blk];
            if (id >= 0 && id < p.num_cache_blocks) {
                float* scale = p.scale[which] + id * p.num_kv_heads + head;
                const float old = row > 0 ? *scale : 0.0f;
                const uint32_t top = __reduce_max_sync(0xffffffffu, halves_top(top_of<T>(top_of<T>(0u, v.x), v.y)));
                const float now = larger(old, scale_for<T, FP8>(top)), inv = __fdiv_rn(1.0f, now);
                unsigned char* base = p.cache[which] + static_cast<size_t>(id) * p.block_size * row_bytes + head * kDim;
                const float2 a = floats_of<T>(v.x), b = floats_of<T>(v.y);
                *reinterpret_cast<uint32_t*>(base + row * row_bytes + lane * 4) = pack4<FP8>(a.x * inv, a.y * inv, b.x * inv, b.y * inv);
                raised = row > 0 && __float_as_int(old) != __float_as_int(now);
                if (lane == 0) {
                    if (row == 0 || raised) *scale = now;
                    if (raised) s_raise[warp] = Raise{base, row, old * inv};
                }
            }
        }
    }
    if (lane == 0 && !raised) s_raise[warp].rows = 0;
    if (__syncthreads_or(raised) == 0) return;
    for (int w = 0; w < kThreads / 32; ++w) {
        const Raise r = s_raise[w];
        if (r.rows > 0) scale_rows<FP8>(r.base, row_bytes, r.rows, r.ratio, threadIdx.x, kThreads);
    }
}

// Any number of new rows: a block of threads takes those that fall into one cache block, of one or several sets.  Which sequence its unit
// belongs to: sequence s has the units from floor(cu[s] / block_size) + 2 s on, which are at least as many as the cache blocks that its rows can touch.
// Between their maximum and their rounding the rows wait in shared memory, or in registers; of blocks too large for that they are read again.
// Bound by HBM: 36864 rows of 8 KV heads of F16, blocks of 256, 41.2 us, 5.5 TB/s of what is read and written (over and over; 39.1 where its input may stay in L2).  What a block of threads does is load, wait, round and store, one after the
// other, so that several of them have to be there to keep the memory busy: three with 64 KiB each on their way by asynchronous copies to shared memory, where registers hold two (43.4 us;
// blocks that go from task to task and load the next one meanwhile 46.8 and 50.5).  Where there are no more than two to an SM anyway registers take less time: 77 rows 3.3 us instead of 3.8.
enum StoreRows { kInRegisters, kInShared, kAgain };
template <typename T, bool FP8, StoreRows ROWS>
__global__ void __launch_bounds__(kThreads, ROWS == kInShared ? 3 : 2) store_blocks_kernel(const __grid_constant__ StoreParams p) {
    extern __shared__ __align__(16) uint4 s_rows[];
    __shared__ uint32_t s_top[kMaxSets];
    pdl_wait_then_release();
    const int tid = threadIdx.x, unit = blockIdx.x;
    if (tid < kMaxSets) s_top[tid] = 0;
    auto token_at = [&](int s) { return static_cast<uint32_t>(min(max(p.cu[s], static_cast<int64_t>(0)), p.total_q)); };
    auto unit_at = [&](int s, uint32_t token) { return static_cast<int64_t>(p.by_block.div(token)) + 2ll * s; };
    int seq = -1;
    for (int s0 = 0; s0 < p.num_seqs; s0 += kThreads) {
        const int s = s0 + tid, n = __syncthreads_count(s < p.num_seqs && unit_at(s, token_at(s)) <= unit);
        seq += n;
        if (n < kThreads) break;
    }
    if (seq < 0) return;
    const uint32_t q0 = token_at(seq), q1 = token_at(seq + 1);
    if (q1 <= q0) return;
    const int64_t ctx = p.context_lens[seq], start = ctx - (q1 - q0);   // positions [start, ctx)
    const int64_t from = max(start, static_cast<int64_t>(0)), to = min(ctx, p.max_blocks * p.block_size);
    if (from >= to) return;
    const int64_t blk = static_cast<int64_t>(p.by_block.div(static_cast<uint32_t>(from))) + (unit - unit_at(seq, q0));
    const int64_t first = max(from, blk * p.block_size), last = min(to, (blk + 1) * p.block_size);
    if (first >= last) return;
    const int64_t id = p.block_tables[seq * p.max_blocks + blk];
    if (id < 0 || id >= p.num_cache_blocks) return;
    const int row0 = static_cast<int>(first - blk * p.block_size), rows = static_cast<int>(last - first);

    const int set_threads = kThreads / p.sets, in_block = tid / set_threads, t = tid - in_block * set_threads;
    const int set = blockIdx.y * p.sets + in_block, sub = t & (kLanes - 1), rank = t / kLanes, ranks = set_threads / kLanes;
    const bool live = set < static_cast<int>(p.by_sets.d);
    const int which = live && set >= p.num_kv_heads ? 1 : 0, head = live ? set - which * p.num_kv_heads : 0;
    const int mine = live ? rows : 0;                                   // (threads without a set go along)
    const T* src = static_cast<const T*>(p.rows[which]) + (q0 + (first - start) + rank) * p.stride[which] + head * kDim + sub * 8;
    const int64_t step = ranks * p.stride[which];
    auto load = [](const T* at) { return __ldcs(reinterpret_cast<const uint4*>(at)); };
    float* scale = p.scale[which] + id * p.num_kv_heads + head;
    const float old = live && row0 > 0 ? *scale : 0.0f;
    uint4* held = s_rows + tid;              // this thread's own pieces, kThreads apart (zeros where there is no row)
    uint4 v[ROWS == kInRegisters ? kPasses : 1];
    uint32_t top = 0;
    if constexpr (ROWS == kInShared) {
        const uint64_t policy = read_once();
        const T* at = src;
#pragma unroll
        for (int i = 0; i < kPasses; ++i, at += step) {
            const bool there = rank + i * ranks < mine;
            cp_async16_once(smem_u32(held + i * kThreads), there ? at : static_cast<const T*>(p.rows[which]), there ? 16 : 0, policy);
        }
        cp_async_commit();
        cp_async_wait<0>();
#pragma unroll
        for (int i = 0; i < kPasses; ++i) top = top_of<T>(top, held[i * kThreads]);
    } else if constexpr (ROWS == kInRegisters) {
        const T* at = src;
#pragma unroll
        for (int i = 0; i < kPasses; ++i, at += step) v[i] = rank + i * ranks < mine ? load(at) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) top = top_of<T>(top, v[i]);
    } else {
        const T* at = src;
        for (int r = rank; r < mine; r += ranks, at += step) top = top_of<T>(top, *reinterpret_cast<const uint4*>(at));
    }
    top = halves_top(top);
#pragma unroll
    for (int x = kLanes / 2; x > 0; x >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (sub == 0) atomicMax(&s_top[in_block], top);
    __syncthreads();
    if (!live) return;
    const float now = larger(old, scale_for<T, FP8>(s_top[in_block])), inv = __fdiv_rn(1.0f, now);
    const bool narrow = narrow_scale(now);
    const size_t row_bytes = static_cast<size_t>(p.num_kv_heads) * kDim;
    unsigned char* base = p.cache[which] + static_cast<size_t>(id) * p.block_size * row_bytes + head * kDim;
    unsigned char* dst = base + (row0 + rank) * row_bytes + sub * 8;
    const size_t dst_step = ranks * row_bytes;
    if constexpr (ROWS != kAgain) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i, dst += dst_step)
            if (rank + i * ranks < rows) *reinterpret_cast<uint2*>(dst) = quantise8<T, FP8>(ROWS == kInShared ? held[i * kThreads] : v[i], inv, narrow);
    } else {
        const T* at = src;
        for (int r = rank; r < rows; r += ranks, at += step, dst += dst_step) *reinterpret_cast<uint2*>(dst) = quantise8<T, FP8>(load(at), inv, narrow);
    }
    const bool raised = __float_as_int(old) != __float_as_int(now);
    if (t == 0 && raised) *scale = now;   // (read by this set's threads before the barrier)
    if (row0 > 0 && raised) scale_rows<FP8>(base, row_bytes, row0, old * inv, t, set_threads);
}

template <typename T, bool FP8> int launch_store_typed(const StoreParams& in, cudaStream_t stream) {
    StoreParams p = in;
    cudaError_t e;
    if (p.cu == nullptr) {
        const int64_t blocks = (static_cast<int64_t>(p.num_seqs) * p.by_sets.d + kThreads / 32 - 1) / (kThreads / 32);
        e = launch_pdl(store_row_kernel<T, FP8>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, p);
    } else {
        static std::atomic<bool> attr_done[64] = {};
        int device = 0;
        cudaGetDevice(&device);
        if (device >= 0 && device < 64 && !attr_done[device]) {
            e = cudaFuncSetAttribute(store_blocks_kernel<T, FP8, kInShared>, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileBytes);
            if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "store_kvcache_blocks8: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
            attr_done[device] = true;
        }
        // As many sets to a block of threads as it has room for.
        p.sets = 1;
        while (p.sets < kMaxSets && 2 * p.sets * p.block_size <= kTileRows) p.sets *= 2;
        const int64_t units = p.total_q / p.block_size + 2ll * p.num_seqs;
        if (units > 0x7fffffffLL) return fail(NVK_ERR_UNSUPPORTED, "store_kvcache_blocks8: too many tokens");
        const dim3 grid(static_cast<unsigned>(units), (p.by_sets.d + p.sets - 1) / p.sets);
        if (grid.y > 65535) return fail(NVK_ERR_UNSUPPORTED, "store_kvcache_blocks8: too many heads");
        if (p.sets * p.block_size > kTileRows) e = launch_pdl(store_blocks_kernel<T, FP8, kAgain>, grid, dim3(kThreads), 0, stream, p);
        else if (units * grid.y <= 2 * kSmCount) e = launch_pdl(store_blocks_kernel<T, FP8, kInRegisters>, grid, dim3(kThreads), 0, stream, p);
        else e = launch_pdl(store_blocks_kernel<T, FP8, kInShared>, grid, dim3(kThreads), kTileBytes, stream, p);
    }
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "store_kvcache_blocks8 kernel launch: %s", cudaGetErrorString(e));
    return check_launch("store_kvcache_blocks8 kernel launch");
}

// ---- gather ----------------------------------------------------------------------------------------------------------------
constexpr int kGatherRows = 256;          // dense rows of a block of threads, at most
constexpr int kGatherVectors = 128;       // and of K and of V head vectors, where there are enough of them for two blocks to an SM
constexpr int kGatherAhead = 4;           // head vectors of K and of V that a lane has under way
constexpr int kGatherLanes = kDim / 16;   // lanes of a head vector

struct GatherParams {
    const unsigned char* cache[2]; const float* scale[2]; void* out[2];
    IndexArray cu; IndexArray block_tables;
    int64_t num_seqs, total, max_blocks, num_cache_blocks;
    int block_size, rows;                 // `rows` of a block of threads
    FastDiv by_heads, by_block;
};

// 32 bytes next to each other: one store where they lie on such a boundary.
template <bool WIDE> __device__ __forceinline__ void store32(uint4* out, const uint32_t (&o)[8]) {
    if constexpr (WIDE) {
        asm volatile("st.global.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                     ::"l"(out), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
    } else {
        __stcs(out, make_uint4(o[0], o[1], o[2], o[3]));
        __stcs(out + 1, make_uint4(o[4], o[5], o[6], o[7]));
    }
}
template <typename T, bool FP8, bool WIDE> __device__ __forceinline__ void dequantise16(const uint4& v, float scale, uint4* out) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 f = unpack4<FP8>(w[i]);
        o[2 * i] = ElemTraits<T>::pack2(f.x * scale, f.y * scale);
        o[2 * i + 1] = ElemTraits<T>::pack2(f.z * scale, f.w * scale);
    }
    store32<WIDE>(out, o);
}

// Bound by HBM: 43008 rows of 8 KV heads, 42.6 us, 6.2 TB/s, behind their store some 37.  A lane has four head vectors of K and of V under way by loads without branches, and writes 32 bytes at a time; a block of threads
// has 128 of each (256: 44.1 us and, at a sixth of the rows, 12.9 instead of 10.2, since the last blocks run alone for longer; 64: 42.9 to 46.7).
template <typename T, bool FP8, bool WIDE>
__global__ void __launch_bounds__(kThreads) gather_blocks8_kernel(const __grid_constant__ GatherParams p) {
    __shared__ int64_t s_row[kGatherRows];     // cache row of a dense row; -1: zeros
    __shared__ int64_t s_block[kGatherRows];   // its cache block
    __shared__ int64_t s_cu[kThreads];
    pdl_wait_then_release();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(p.rows), p.total - first));
    // The last sequence that begins at or before the first row: all threads look, one trip to memory where there are up to kThreads sequences.
    int64_t seq = -1, base = 0;
    for (;; base += kThreads) {
        const int64_t s = base + threadIdx.x, begin = s <= p.num_seqs ? p.cu[s] : 0;
        s_cu[threadIdx.x] = begin;
        const int n = __syncthreads_count(s < p.num_seqs && begin <= first);
        seq += n;
        if (n < kThreads || base + kThreads >= p.num_seqs) break;
        __syncthreads();
    }
    auto begin_of = [&](int64_t s) { return s >= base && s < base + kThreads ? s_cu[s - base] : p.cu[s]; };
    if (threadIdx.x < static_cast<unsigned>(rows)) {
        const int64_t r = first + threadIdx.x;
        int64_t row = -1, at = 0;
        if (seq >= 0) {
            while (seq + 1 < p.num_seqs && begin_of(seq + 1) <= r) ++seq;
            const int64_t pos = r - begin_of(seq);
            if (pos >= 0 && r < begin_of(seq + 1) && pos < p.max_blocks * p.block_size) {
                const int64_t blk = p.by_block.div(static_cast<uint32_t>(pos)), block = p.block_tables[seq * p.max_blocks + blk];
                if (block >= 0 && block < p.num_cache_blocks) {
                    row = block * p.block_size + (pos - blk * p.block_size);
                    at = block;
                }
            }
        }
        s_row[threadIdx.x] = row;
        s_block[threadIdx.x] = at;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, sub = lane % kGatherLanes, heads = static_cast<int>(p.by_heads.d), vectors = rows * heads;
    constexpr int kStride = kThreads / kGatherLanes;
    uint4* out[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) out[w] = static_cast<uint4*>(p.out[w]) + first * heads * kLanes + sub * 2;
    for (int i0 = threadIdx.x / kGatherLanes; i0 < vectors; i0 += kStride * kGatherAhead) {
        uint4 v[kGatherAhead][2];
        float scale[kGatherAhead][2];
#pragma unroll
        for (int u = 0; u < kGatherAhead; ++u) {
            // (loads without branches, so that all are under way at once)
            const int i = min(i0 + u * kStride, vectors - 1), r = static_cast<int>(p.by_heads.div(i)), head = i - r * heads;
            const int64_t row = s_row[r], at = row >= 0 ? row * heads + head : 0, scale_at = s_block[r] * heads + head;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                v[u][w] = __ldcs(reinterpret_cast<const uint4*>(p.cache[w] + at * kDim) + sub);
                scale[u][w] = p.scale[w][scale_at];
                if (row < 0) { v[u][w] = make_uint4(0u, 0u, 0u, 0u); scale[u][w] = 0.0f; }
            }
        }
#pragma unroll
        for (int u = 0; u < kGatherAhead; ++u) {
            const int i = i0 + u * kStride;
            if (i < vectors) {
#pragma unroll
                for (int w = 0; w < 2; ++w) dequantise16<T, FP8, WIDE>(v[u][w], scale[u][w], out[w] + static_cast<int64_t>(i) * kLanes);
            }
        }
    }
}

template <typename T, bool FP8> cudaError_t launch_gather_typed(const GatherParams& p, int64_t blocks, cudaStream_t stream) {
    const auto kernel = aligned_to(p.out[0], 32) && aligned_to(p.out[1], 32) ? gather_blocks8_kernel<T, FP8, true> : gather_blocks8_kernel<T, FP8, false>;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, p);
}

}  // namespace

int launch_store_blocks8(const Blocks8StoreArgs& a) {
    StoreParams p{};
    p.rows[0] = a.key; p.rows[1] = a.value;
    p.stride[0] = a.key_stride; p.stride[1] = a.value_stride;
    p.cache[0] = static_cast<unsigned char*>(a.k_cache); p.cache[1] = static_cast<unsigned char*>(a.v_cache);
    p.scale[0] = a.k_scale; p.scale[1] = a.v_scale;
    p.cu = a.cu; p.context_lens = a.context_lens; p.block_tables = a.block_tables;
    p.total_q = a.total_q; p.max_blocks = a.max_blocks; p.num_cache_blocks = a.num_cache_blocks;
    p.num_seqs = static_cast<int>(a.num_seqs); p.num_kv_heads = a.num_kv_heads; p.block_size = a.block_size;
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    p.by_sets = FastDiv(static_cast<uint32_t>(2 * a.num_kv_heads));
    using bf = __nv_bfloat16;
    if (a.dtype == NVK_BF16) return a.fp8 ? launch_store_typed<bf, true>(p, a.stream) : launch_store_typed<bf, false>(p, a.stream);
    return a.fp8 ? launch_store_typed<__half, true>(p, a.stream) : launch_store_typed<__half, false>(p, a.stream);
}

int launch_gather_blocks8(const Blocks8GatherArgs& a) {
    // Few rows are spread over the SMs.
    int rows = kGatherVectors / a.num_kv_heads;
    while (rows > 1 && (a.total + rows - 1) / rows < 2 * kSmCount) rows >>= 1;
    if (rows < 1) rows = 1;
    const int64_t blocks = (a.total + rows - 1) / rows;
    if (blocks > 0x7fffffffLL || a.num_kv_heads > 0x7fffffff / kGatherRows) return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_blocks8: too many rows");
    GatherParams p{};
    p.cache[0] = static_cast<const unsigned char*>(a.k_cache); p.cache[1] = static_cast<const unsigned char*>(a.v_cache);
    p.scale[0] = a.k_scale; p.scale[1] = a.v_scale; p.out[0] = a.key; p.out[1] = a.value;
    p.cu = a.cu; p.block_tables = a.block_tables;
    p.num_seqs = a.num_seqs; p.total = a.total; p.max_blocks = a.max_blocks; p.num_cache_blocks = a.num_cache_blocks;
    p.block_size = a.block_size; p.rows = rows;
    p.by_heads = FastDiv(static_cast<uint32_t>(a.num_kv_heads));
    p.by_block = FastDiv(static_cast<uint32_t>(a.block_size));
    using bf = __nv_bfloat16;
    const cudaError_t e = a.dtype == NVK_BF16 ? (a.fp8 ? launch_gather_typed<bf, true>(p, blocks, a.stream) : launch_gather_typed<bf, false>(p, blocks, a.stream))
                                              : (a.fp8 ? launch_gather_typed<__half, true>(p, blocks, a.stream) : launch_gather_typed<__half, false>(p, blocks, a.stream));
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "gather_blocks8_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("gather_blocks8_kernel launch");
}

}  // namespace nvk
