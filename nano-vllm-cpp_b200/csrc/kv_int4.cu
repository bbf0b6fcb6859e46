// 4-bit paged KV cache for sm_100a: quantising store, and the gather of whole contexts into dense 16-bit rows.  (Decode attention over
// this cache: Cache4 in decode_body.cuh.)  No counterpart in the reference, whose smallest cache is the int8 one
// (src/kernels/kvcache.cu:222-296).
//
// Format: of a head vector x of 128 elements in F16 / BF16, with low = min x and step = (max x - min x) / 15 rounded to the type, the numbers
//   n = min(15, floor((x - low) / step + 1/2)), 0 where step is 0,
// two to a byte (element 2i in the low half of byte i), and the pair (step, low) in the type itself: x stands for low + step n, off by half a step
// at most (and by 15 / 2 of what the rounding of step took off it at the top).  low is an element of x, so that it needs no rounding.  A vector whose
// range is not finite gets a pair of NaN, and reads as NaN.
#include "nvk_internal.cuh"

namespace nvk {
namespace {

constexpr int kDim = 128;
constexpr int kLanes = kDim / 8;          // lanes to a head vector: eight elements, 16 bytes, each
constexpr int kStoreWarps = 8;

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    using type = __nv_bfloat162;
    static __device__ __forceinline__ float2 floats(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
};
template <> struct Pair<__half> {
    using type = __half2;
    static __device__ __forceinline__ float2 floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <typename T> __device__ __forceinline__ typename Pair<T>::type as_pair(uint32_t w) { return *reinterpret_cast<const typename Pair<T>::type*>(&w); }
template <typename P> __device__ __forceinline__ uint32_t as_word(P p) { return *reinterpret_cast<const uint32_t*>(&p); }

// The extremes of the eight elements of a piece, NaN if one is: (min | max) of both halves' lanes still apart.
template <typename T> __device__ __forceinline__ uint32_t lowest2(const uint4& v) {
    return as_word(__hmin2_nan(__hmin2_nan(as_pair<T>(v.x), as_pair<T>(v.y)), __hmin2_nan(as_pair<T>(v.z), as_pair<T>(v.w))));
}
template <typename T> __device__ __forceinline__ uint32_t highest2(const uint4& v) {
    return as_word(__hmax2_nan(__hmax2_nan(as_pair<T>(v.x), as_pair<T>(v.y)), __hmax2_nan(as_pair<T>(v.z), as_pair<T>(v.w))));
}
// Of K's and V's pairs: one pair (K, V) of the extremes over both halves.
template <typename T> __device__ __forceinline__ uint32_t join_lowest(uint32_t k, uint32_t v) {
    return as_word(__hmin2_nan(as_pair<T>(__byte_perm(k, v, 0x5410)), as_pair<T>(__byte_perm(k, v, 0x7632))));
}
template <typename T> __device__ __forceinline__ uint32_t join_highest(uint32_t k, uint32_t v) {
    return as_word(__hmax2_nan(as_pair<T>(__byte_perm(k, v, 0x5410)), as_pair<T>(__byte_perm(k, v, 0x7632))));
}

// The numbers of eight elements, as a word.  floor(q + 1/2) of the true quotient q = (x - low) / step, without a division: the product with 1 / step,
// made smaller by more than its error (2^-16; the error is below 15 x 2^-21), rounds to that number or to the one before it, and it is the one after exactly if
// x >= low + (n + 1/2) step, which fma rounded upwards decides exactly, x being representable.
__device__ __forceinline__ uint32_t numbers(float (&x)[8], float low, float step) {
    if (step < 0x1p-100f) {   // (1 / step may not be finite; the elements are small as well, since low's own spacing is no larger than the range)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= 0x1p100f;
        low *= 0x1p100f;
        step *= 0x1p100f;
    }
    const float inv = __fdiv_rn(1.0f, step);
    constexpr float kMagic = 12582912.0f;   // 1.5 x 2^23: adding it rounds to a whole number, in the low bits of the sum
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float m = __fadd_rn(__fmaf_rn(__fsub_rn(x[i], low), inv, -0x1p-16f), kMagic);
        const float border = __fmaf_ru(__fadd_rn(__fsub_rn(m, kMagic), 0.5f), step, low);
        const uint32_t n = (__float_as_uint(m) & 0x3fu) + (x[i] >= border ? 1u : 0u);
        word |= min(n, 15u) << (4 * i);     // (above 15 only where step is a subnormal number, rounded down)
    }
    return word;
}

// A head vector's share of one lane -> numbers; step and low as stored.
template <typename T> __device__ __forceinline__ uint32_t quantise(const uint4& v, float low, float high, T& step_out, T& low_out) {
    const float span = __fsub_rn(high, low);
    const bool fine = fabsf(span) < INFINITY;
    step_out = ElemTraits<T>::from_float(fine ? __fdiv_rn(span, 15.0f) : NAN);
    low_out = ElemTraits<T>::from_float(fine ? low : NAN);
    const float step = ElemTraits<T>::to_float(step_out);
    if (!(step > 0.0f)) return 0u;
    float x[8];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<T>::floats(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
    return numbers(x, low, step);
}

// One warp quantises two (token, KV head) vectors of K and of V.
template <typename T>
__global__ void __launch_bounds__(kStoreWarps * 32)
store_int4_kernel(const T* __restrict__ key, const T* __restrict__ value, uint32_t* __restrict__ k_cache, uint32_t* __restrict__ v_cache,
                  uint32_t* __restrict__ k_params, uint32_t* __restrict__ v_params, const IndexArray slot_mapping, uint32_t total, const FastDiv by_heads,
                  int64_t cache_rows) {
    pdl_wait_then_release();
    const uint32_t lane = threadIdx.x & 31u, sub = lane % kLanes;
    uint32_t work = (blockIdx.x * kStoreWarps + (threadIdx.x >> 5)) * 2 + lane / kLanes;   // (token, head)
    if (work >= total) work = total - 1;   // lanes past the end repeat the last vector: the shuffles stay full-warp
    const uint32_t token = by_heads.div(work), head = work - token * by_heads.d;
    const size_t src = static_cast<size_t>(work) * kDim + sub * 8;
    const uint4 kv = __ldcs(reinterpret_cast<const uint4*>(key + src));
    const uint4 vv = __ldcs(reinterpret_cast<const uint4*>(value + src));
    const int64_t slot = slot_mapping[token];
    uint32_t lo = join_lowest<T>(lowest2<T>(kv), lowest2<T>(vv)), hi = join_highest<T>(highest2<T>(kv), highest2<T>(vv));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
        lo = as_word(__hmin2_nan(as_pair<T>(lo), as_pair<T>(__shfl_xor_sync(0xffffffffu, lo, o))));
        hi = as_word(__hmax2_nan(as_pair<T>(hi), as_pair<T>(__shfl_xor_sync(0xffffffffu, hi, o))));
    }
    if (slot < 0 || slot >= cache_rows) return;
    const float2 low = Pair<T>::floats(lo), high = Pair<T>::floats(hi);
    const size_t row = static_cast<size_t>(slot) * by_heads.d + head;
    union { T e[2]; uint32_t w; } kp, vp;
    k_cache[row * kLanes + sub] = quantise<T>(kv, low.x, high.x, kp.e[0], kp.e[1]);
    v_cache[row * kLanes + sub] = quantise<T>(vv, low.y, high.y, vp.e[0], vp.e[1]);
    if (sub == 0) {
        k_params[row] = kp.w;
        v_params[row] = vp.w;
    }
}

template <typename T>
int launch_store_typed(const void* key, const void* value, void* k_cache, void* v_cache, void* k_params, void* v_params, const IndexArray& slots,
                       int64_t num_tokens, int num_kv_heads, int64_t cache_rows, cudaStream_t stream) {
    const int64_t work = num_tokens * num_kv_heads;
    if (work >= 0x7fffffffLL) return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int4: too many tokens");
    const int64_t blocks = (work + 2 * kStoreWarps - 1) / (2 * kStoreWarps);
    const cudaError_t e = launch_pdl(store_int4_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kStoreWarps * 32), 0, stream, static_cast<const T*>(key),
                                     static_cast<const T*>(value), static_cast<uint32_t*>(k_cache), static_cast<uint32_t*>(v_cache),
                                     static_cast<uint32_t*>(k_params), static_cast<uint32_t*>(v_params), slots, static_cast<uint32_t>(work),
                                     FastDiv(static_cast<uint32_t>(num_kv_heads)), cache_rows);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "store_int4_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("store_int4_kernel launch");
}

// ---- gather ----------------------------------------------------------------------------------------------------------------
constexpr int kGatherWarps = 8;
constexpr int kGatherRows = 32;           // dense rows of a block

struct GatherParams {
    const uint32_t* k_cache; const uint32_t* v_cache; const uint32_t* k_params; const uint32_t* v_params;
    void* key; void* value;
    IndexArray cu; IndexArray block_tables;
    int64_t num_seqs, total, max_blocks, num_cache_blocks;
    int block_size;
    FastDiv by_heads;
};

template <typename T> __device__ __forceinline__ uint4 dequantise(uint32_t word, uint32_t param) {
    const float2 p = Pair<T>::floats(param);   // (step, low)
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // 2^23 + n, exactly; n is exact, the product too, and low + step n is rounded once to fp32 and once to the type
        const float n0 = __uint_as_float(((word >> (8 * i)) & 15u) | 0x4b000000u) - 8388608.0f, n1 = __uint_as_float(((word >> (8 * i + 4)) & 15u) | 0x4b000000u) - 8388608.0f;
        out[i] = ElemTraits<T>::pack2(fmaf(p.x, n0, p.y), fmaf(p.x, n1, p.y));
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

template <typename T>
__global__ void __launch_bounds__(kGatherWarps * 32) gather_int4_kernel(const __grid_constant__ GatherParams p) {
    __shared__ int64_t s_row[kGatherRows];   // cache row of a dense row; -1: zeros
    pdl_wait_then_release();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kGatherRows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(kGatherRows), p.total - first));
    if (threadIdx.x < kGatherRows) {
        const int64_t r = first + threadIdx.x;
        int64_t lo = 0, hi = p.num_seqs;     // the last sequence that begins at or before r
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.cu[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int64_t pos = r - p.cu[lo];
        int64_t row = -1;
        if (pos >= 0 && r < p.cu[lo + 1] && pos < p.max_blocks * p.block_size) {
            const int64_t block = p.block_tables[lo * p.max_blocks + pos / p.block_size];
            if (block >= 0 && block < p.num_cache_blocks) row = block * p.block_size + pos % p.block_size;
        }
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, sub = lane % kLanes;
    const int vectors = rows * static_cast<int>(p.by_heads.d);
    uint4* key = static_cast<uint4*>(p.key) + first * p.by_heads.d * kLanes;
    uint4* value = static_cast<uint4*>(p.value) + first * p.by_heads.d * kLanes;
    for (int i = (threadIdx.x >> 5) * 2 + lane / kLanes; i < vectors; i += kGatherWarps * 2) {
        const int r = static_cast<int>(p.by_heads.div(i)), head = i - r * static_cast<int>(p.by_heads.d);
        const int64_t row = s_row[r];
        const bool there = row >= 0;
        const int64_t at = there ? row * p.by_heads.d + head : 0;
        const uint32_t k = there ? p.k_cache[at * kLanes + sub] : 0u, v = there ? p.v_cache[at * kLanes + sub] : 0u;
        const uint32_t kp = there ? p.k_params[at] : 0u, vp = there ? p.v_params[at] : 0u;
        key[static_cast<int64_t>(i) * kLanes + sub] = dequantise<T>(k, kp);
        value[static_cast<int64_t>(i) * kLanes + sub] = dequantise<T>(v, vp);
    }
}

}  // namespace

int launch_store_int4(const void* key, const void* value, void* k_cache, void* v_cache, void* k_params, void* v_params, const IndexArray& slots,
                      int64_t num_tokens, int num_kv_heads, int64_t cache_rows, int dtype, cudaStream_t stream) {
    return dtype == NVK_BF16 ? launch_store_typed<__nv_bfloat16>(key, value, k_cache, v_cache, k_params, v_params, slots, num_tokens, num_kv_heads, cache_rows, stream)
                             : launch_store_typed<__half>(key, value, k_cache, v_cache, k_params, v_params, slots, num_tokens, num_kv_heads, cache_rows, stream);
}

int launch_gather_int4(const void* k_cache, const void* v_cache, const void* k_params, const void* v_params, const IndexArray& cu, const IndexArray& tables,
                       int64_t num_seqs, int64_t total, int64_t max_blocks, int64_t num_cache_blocks, int num_kv_heads, int block_size, void* key,
                       void* value, int dtype, cudaStream_t stream) {
    const int64_t blocks = (total + kGatherRows - 1) / kGatherRows;
    if (blocks > 0x7fffffffLL || num_kv_heads > 0x7fffffff / kGatherRows) return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_int4: too many rows");
    const GatherParams p{static_cast<const uint32_t*>(k_cache), static_cast<const uint32_t*>(v_cache), static_cast<const uint32_t*>(k_params),
                         static_cast<const uint32_t*>(v_params), key, value, cu, tables, num_seqs, total, max_blocks, num_cache_blocks, block_size,
                         FastDiv(static_cast<uint32_t>(num_kv_heads))};
    const dim3 grid(static_cast<unsigned>(blocks)), block(kGatherWarps * 32);
    const cudaError_t e = dtype == NVK_BF16 ? launch_pdl(gather_int4_kernel<__nv_bfloat16>, grid, block, 0, stream, p)
                                            : launch_pdl(gather_int4_kernel<__half>, grid, block, 0, stream, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "gather_int4_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("gather_int4_kernel launch");
}

}  // namespace nvk
