// 4-bit paged KV cache for sm_100a: quantising store, and the gather of whole contexts into dense 16-bit rows.  (Decode attention over
// this cache: Cache4 in decode_body.cuh.)  No counterpart in the reference, whose smallest cache is the int8 one
// (src/kernels/kvcache.cu:222-296).
//
// Format: of a head vector x of 128 elements in F16 / BF16, with low = min x and step = (max x - min x) / 15 rounded to the type, the numbers
//   n = min(15, floor((x - low) / step + 1/2)), 0 where step is 0,
// two to a byte (element 2i in the low half of byte i), and the pair (step, low) in the type itself: x stands for low + step n, off by half a step
// at most (and by 15 / 2 of what the rounding of step took off it at the top).  low is an element of x, so that it needs no rounding.  A vector whose
// range is not finite gets a pair of NaN, and reads as NaN.
//
// The store should be HBM-bound (of an element two bytes are read and half a one is written) but is bound by issue: 36864 tokens of 8 heads, 192 MB, take 37.5 us, 5.1
// TB/s, with 80 % of the issue slots busy and DRAM at half.  The gather writes 3.8 times what it reads: 43008 rows of 8 heads, 223 MB, take 39 us, 5.7 TB/s.
#include "nvk_internal.cuh"

#include <type_traits>

namespace nvk {
namespace {

constexpr int kDim = 128;
constexpr int kLanes = kDim / 8;          // 16-byte pieces (eight elements) of a head vector
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

// Two floats in one instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 floats_of(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t fma2_up(uint64_t a, uint64_t b, uint64_t c) {   // rounded upwards
    uint64_t d;
    asm("fma.rp.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// The numbers of eight elements (pairs of the type, as loaded), as a word.  floor(q + 1/2) of the true quotient q = (x - low) / step, without a division:
// x / step - low / step - 1/4, each term rounded (off by less than 1/4, since |low| <= 2^11 ranges), rounds to that number or to the one before it, and it is
// the one after exactly if x >= low + (n + 1/2) step, which fma rounded upwards decides exactly, x being representable.
// CAREFUL: step is a subnormal number of the type: 1 / step may not be finite (all is multiplied by 2^100 first; elements are small as well, since low's own
// spacing is no larger than the range), and numbers above 15 come out where it was rounded down.
template <typename T, bool CAREFUL> __device__ __forceinline__ uint32_t numbers(const uint4& v, float low, float step) {
    const float scale = CAREFUL && step < 0x1p-100f ? 0x1p100f : 1.0f;
    if (CAREFUL) { low *= scale; step *= scale; }
    float inv;                              // (to within one unit in its last place)
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(inv) : "f"(step));
    constexpr float kMagic = 12582912.0f;   // 1.5 x 2^23: adding it rounds to a whole number, in the low bits of the sum
    const uint64_t inv2 = pair_of(inv, inv), from = pair_of(fmaf(-low, inv, -0.25f), fmaf(-low, inv, -0.25f)), low2 = pair_of(low, low), step2 = pair_of(step, step);
    const uint64_t magic = pair_of(kMagic, kMagic), back = pair_of(-kMagic, -kMagic), half = pair_of(0.5f, 0.5f);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 x = Pair<T>::floats(w[i]);
        if (CAREFUL) { x.x *= scale; x.y *= scale; }
        const uint64_t m = add2(fma2(pair_of(x.x, x.y), inv2, from), magic);
        const float2 border = floats_of(fma2_up(add2(add2(m, back), half), step2, low2)), whole = floats_of(m);
        // (whole numbers are 12582912 + n as bits too; what the 12582912 leave in the word goes at the end)
        uint32_t a = __float_as_uint(whole.x), b = __float_as_uint(whole.y);
        if (CAREFUL) {
            a = min((a & 0x3fu) + (x.x >= border.x ? 1u : 0u), 15u);
            b = min((b & 0x3fu) + (x.y >= border.y ? 1u : 0u), 15u);
        } else {
            if (x.x >= border.x) word += 1u << (8 * i);
            if (x.y >= border.y) word += 1u << (8 * i + 4);
        }
        word += (a << (8 * i)) + (b << (8 * i + 4));
    }
    constexpr uint32_t kBits = 0x4b400000u;
    return CAREFUL ? word : word - (kBits + (kBits << 4) + (kBits << 8));   // (beyond that the shifts leave nothing of them)
}

// x / 15, correctly rounded: a quotient from the rounded reciprocal, and one step with its exact remainder (Markstein, Computation of elementary functions on the
// IBM RISC System/6000 processor, 1990); small numbers, whose remainders may not be exact, are divided.
__device__ __forceinline__ float fifteenth(float x) {
    constexpr float kInv = 1.0f / 15.0f;
    const float q = __fmul_rn(x, kInv);
    return x >= 0x1p-100f ? __fmaf_rn(__fmaf_rn(-q, 15.0f, x), kInv, q) : __fdiv_rn(x, 15.0f);
}
// What is stored of a head vector beside its numbers: a pair (step, low).
template <typename T> __device__ __forceinline__ uint32_t params_of(float low, float high) {
    const float span = __fsub_rn(high, low);
    return fabsf(span) < INFINITY ? ElemTraits<T>::pack2(fifteenth(span), low) : ElemTraits<T>::pack2(NAN, NAN);
}
// A lane's two pieces of a head vector -> numbers.
template <typename T> __device__ __forceinline__ uint2 quantise(const uint4 (&v)[2], uint32_t params) {
    constexpr float kNormal = std::is_same<T, __half>::value ? 0x1p-14f : 0x1p-126f;
    const float2 p = Pair<T>::floats(params);
    if (p.x >= kNormal) return make_uint2(numbers<T, false>(v[0], p.y, p.x), numbers<T, false>(v[1], p.y, p.x));
    return p.x > 0.0f ? make_uint2(numbers<T, true>(v[0], p.y, p.x), numbers<T, true>(v[1], p.y, p.x)) : make_uint2(0u, 0u);
}

// One warp quantises four (token, KV head) vectors of K and of V, eight lanes to a vector, each with its pieces `sub` and `sub` + 8: what is done once for a vector
// is as much as what is done for eight elements (with 16 lanes to a vector 310 instructions a warp for 1024 elements, and 36864 tokens of 8 heads took
// 53 us; by 8 lanes 1.5 times as many for twice the elements).
constexpr int kStoreLanes = 8, kStoreVectors = 32 / kStoreLanes;
template <typename T>
__global__ void __launch_bounds__(kStoreWarps * 32)
store_int4_kernel(const T* __restrict__ key, const T* __restrict__ value, uint32_t* __restrict__ k_cache, uint32_t* __restrict__ v_cache,
                  uint32_t* __restrict__ k_params, uint32_t* __restrict__ v_params, const IndexArray slot_mapping, uint32_t total, const FastDiv by_heads,
                  int64_t cache_rows) {
    pdl_wait_then_release();
    const uint32_t lane = threadIdx.x & 31u, sub = lane % kStoreLanes;
    uint32_t work = (blockIdx.x * kStoreWarps + (threadIdx.x >> 5)) * kStoreVectors + lane / kStoreLanes;   // (token, head)
    if (work >= total) work = total - 1;   // lanes past the end repeat the last vector: the shuffles stay full-warp
    const uint32_t token = by_heads.div(work), head = work - token * by_heads.d;
    const uint4* k_src = reinterpret_cast<const uint4*>(key) + static_cast<size_t>(work) * kLanes + sub;
    const uint4* v_src = reinterpret_cast<const uint4*>(value) + static_cast<size_t>(work) * kLanes + sub;
    const uint4 kv[2] = {__ldcs(k_src), __ldcs(k_src + kStoreLanes)}, vv[2] = {__ldcs(v_src), __ldcs(v_src + kStoreLanes)};
    const IndexArray::Raw raw_slot = slot_mapping.raw(token);
    auto both = [](uint32_t a, uint32_t b, bool low) { return as_word(low ? __hmin2_nan(as_pair<T>(a), as_pair<T>(b)) : __hmax2_nan(as_pair<T>(a), as_pair<T>(b))); };
    uint32_t lo = join_lowest<T>(both(lowest2<T>(kv[0]), lowest2<T>(kv[1]), true), both(lowest2<T>(vv[0]), lowest2<T>(vv[1]), true));
    uint32_t hi = join_highest<T>(both(highest2<T>(kv[0]), highest2<T>(kv[1]), false), both(highest2<T>(vv[0]), highest2<T>(vv[1]), false));
#pragma unroll
    for (int o = kStoreLanes / 2; o > 0; o >>= 1) {
        lo = both(lo, __shfl_xor_sync(0xffffffffu, lo, o), true);
        hi = both(hi, __shfl_xor_sync(0xffffffffu, hi, o), false);
    }
    const int64_t slot = slot_mapping.value(raw_slot);
    if (slot < 0 || slot >= cache_rows) return;
    const float2 low = Pair<T>::floats(lo), high = Pair<T>::floats(hi);
    const size_t row = static_cast<size_t>(slot) * by_heads.d + head;
    const uint32_t kp = params_of<T>(low.x, high.x), vp = params_of<T>(low.y, high.y);
    const uint2 k = quantise<T>(kv, kp), v = quantise<T>(vv, vp);
    uint32_t *k_dst = k_cache + row * kLanes + sub, *v_dst = v_cache + row * kLanes + sub;
    k_dst[0] = k.x;
    k_dst[kStoreLanes] = k.y;
    v_dst[0] = v.x;
    v_dst[kStoreLanes] = v.y;
    if (sub == 0) {
        k_params[row] = kp;
        v_params[row] = vp;
    }
}

template <typename T>
int launch_store_typed(const void* key, const void* value, void* k_cache, void* v_cache, void* k_params, void* v_params, const IndexArray& slots,
                       int64_t num_tokens, int num_kv_heads, int64_t cache_rows, cudaStream_t stream) {
    const int64_t work = num_tokens * num_kv_heads;
    if (work >= 0x7fffffffLL) return fail(NVK_ERR_INVALID_ARGUMENT, "store_kvcache_int4: too many tokens");
    constexpr int kPerBlock = kStoreVectors * kStoreWarps;
    const int64_t blocks = (work + kPerBlock - 1) / kPerBlock;
    const cudaError_t e = launch_pdl(store_int4_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kStoreWarps * 32), 0, stream, static_cast<const T*>(key),
                                     static_cast<const T*>(value), static_cast<uint32_t*>(k_cache), static_cast<uint32_t*>(v_cache),
                                     static_cast<uint32_t*>(k_params), static_cast<uint32_t*>(v_params), slots, static_cast<uint32_t>(work),
                                     FastDiv(static_cast<uint32_t>(num_kv_heads)), cache_rows);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "store_int4_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("store_int4_kernel launch");
}

// ---- gather ----------------------------------------------------------------------------------------------------------------
constexpr int kGatherWarps = 8;
constexpr int kGatherRows = 32;           // dense rows of a block, at most
constexpr int kGatherAhead = 4;           // head vectors of K and of V that a lane has under way

struct GatherParams {
    const uint32_t* k_cache; const uint32_t* v_cache; const uint32_t* k_params; const uint32_t* v_params;
    void* key; void* value;
    IndexArray cu; IndexArray block_tables;
    int64_t num_seqs, total, max_blocks, num_cache_blocks;
    int block_size, rows;                 // `rows` of a block
    FastDiv by_heads;
};

// Numbers 2i and 2i + 1 of a word as a pair of the type: in the low bits of a mantissa, the constant above them taken off again, exactly.
template <typename T> __device__ __forceinline__ typename Pair<T>::type number_pair(uint32_t word, uint32_t upper, int i) {   // upper: word >> 4
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr uint32_t kBits = kHalf ? 0x64006400u : 0x43004300u;   // 1024, 128
    const uint32_t n = (__byte_perm(word, upper, 0x0400 + 0x0101 * i + (i << 12)) & 0x000f000fu) | kBits;
    return __hsub2(as_pair<T>(n), as_pair<T>(kBits));
}
template <typename T> __device__ __forceinline__ uint4 dequantise(uint32_t word, uint32_t param) {
    const uint32_t upper = word >> 4;
    const auto step = as_pair<T>(__byte_perm(param, 0, 0x1010)), low = as_pair<T>(__byte_perm(param, 0, 0x3232));
    uint32_t out[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = as_word(__hfma2(step, number_pair<T>(word, upper, i), low));   // (one rounding)
    return make_uint4(out[0], out[1], out[2], out[3]);
}

template <typename T>
__global__ void __launch_bounds__(kGatherWarps * 32) gather_int4_kernel(const __grid_constant__ GatherParams p) {
    __shared__ int64_t s_row[kGatherRows];   // cache row of a dense row; -1: zeros
    pdl_wait_then_release();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(p.rows), p.total - first));
    if (threadIdx.x < static_cast<unsigned>(rows)) {
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
    const int lane = threadIdx.x & 31, sub = lane % kLanes, heads = static_cast<int>(p.by_heads.d), vectors = rows * heads;
    uint4* key = static_cast<uint4*>(p.key) + first * heads * kLanes + sub;
    uint4* value = static_cast<uint4*>(p.value) + first * heads * kLanes + sub;
    constexpr int kStride = kGatherWarps * 2;
    for (int i0 = (threadIdx.x >> 5) * 2 + lane / kLanes; i0 < vectors; i0 += kStride * kGatherAhead) {
        uint32_t k[kGatherAhead], v[kGatherAhead], kp[kGatherAhead], vp[kGatherAhead];
#pragma unroll
        for (int u = 0; u < kGatherAhead; ++u) {
            const int i = min(i0 + u * kStride, vectors - 1), r = static_cast<int>(p.by_heads.div(i));
            const int64_t row = s_row[r];
            const int64_t at = row >= 0 ? row * heads + (i - r * heads) : 0;
            k[u] = __ldcs(p.k_cache + at * kLanes + sub);
            v[u] = __ldcs(p.v_cache + at * kLanes + sub);
            kp[u] = p.k_params[at];
            vp[u] = p.v_params[at];
            if (row < 0) k[u] = v[u] = kp[u] = vp[u] = 0u;
        }
#pragma unroll
        for (int u = 0; u < kGatherAhead; ++u) {
            const int i = i0 + u * kStride;
            if (i < vectors) {
                key[static_cast<int64_t>(i) * kLanes] = dequantise<T>(k[u], kp[u]);
                value[static_cast<int64_t>(i) * kLanes] = dequantise<T>(v[u], vp[u]);
            }
        }
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
    // Few rows are spread over the SMs.
    int rows = kGatherRows;
    while (rows > 1 && (total + rows - 1) / rows < 4 * kSmCount) rows >>= 1;
    const int64_t blocks = (total + rows - 1) / rows;
    if (blocks > 0x7fffffffLL || num_kv_heads > 0x7fffffff / kGatherRows) return fail(NVK_ERR_UNSUPPORTED, "gather_kvcache_int4: too many rows");
    const GatherParams p{static_cast<const uint32_t*>(k_cache), static_cast<const uint32_t*>(v_cache), static_cast<const uint32_t*>(k_params),
                         static_cast<const uint32_t*>(v_params), key, value, cu, tables, num_seqs, total, max_blocks, num_cache_blocks, block_size, rows,
                         FastDiv(static_cast<uint32_t>(num_kv_heads))};
    const dim3 grid(static_cast<unsigned>(blocks)), block(kGatherWarps * 32);
    const cudaError_t e = dtype == NVK_BF16 ? launch_pdl(gather_int4_kernel<__nv_bfloat16>, grid, block, 0, stream, p)
                                            : launch_pdl(gather_int4_kernel<__half>, grid, block, 0, stream, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "gather_int4_kernel launch: %s", cudaGetErrorString(e));
    return check_launch("gather_int4_kernel launch");
}

}  // namespace nvk
