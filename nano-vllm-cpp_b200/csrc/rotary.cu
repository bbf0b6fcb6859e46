// Rotary positions on query and key heads: any position, pairs of halves or of neighbours, all of a head or its first part, any frequencies.
//
// Beside the fused prologue (fused_prologue.cu), whose rotation is over halves of a whole head and goes by a table of cosines: here
//   (a, b) -> factor (a cos t - b sin t, b cos t + a sin t),   t = position * frequency of the pair,
// with pairs (i, i + rot / 2) or (2i, 2i + 1) of the first `rot` elements; the others are copied.  The reference rotates whole heads by halves
// (src/kernels/split_qkv.cu:62-154).
//
// Far out in a long context position * frequency has no bits left for the angle in 32 bits (position 2^20: off by up to 1/16), so the turns are taken in 64
// bits, and only their fraction goes on to sincospi in 32: off by 2^-53 of the number of turns, and by 2^-25 of a turn.  A row's angles are worked out once for all its
// heads: a handful of 64-bit operations for each pair of a row, next to Hq + Hkv times as many elements.
//
// Bound by HBM for many rows (every element is read and written once), by the trip to memory and the launch for few.  A thread takes two pieces of V elements of a head,
// whose V pairs lie in them whole, in either layout: pieces i and rot / 2 + i, or two next to each other.
#include "nvk_internal.cuh"

#include <algorithm>
#include <type_traits>

namespace nvk {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;         // items of a thread under way
constexpr int kMaxRows = 4;       // of a block

struct RotaryParams {
    const void* in[2]; void* out[2];                  // queries, keys
    int64_t in_stride[2], out_stride[2];              // elements from a row to the next
    IndexArray positions; const float* inv_freq;
    int64_t rows;
    float factor;
    int heads[2];
    int head_dim, rot, items;                         // items: of a head
    int block_rows;
    FastDiv by_items, by_heads, by_pairs;             // of a head, of a row (queries and keys), of the rotated part
};

template <int BYTES> struct Piece;
template <> struct Piece<16> { using type = uint4; };
template <> struct Piece<8> { using type = uint2; };
template <> struct Piece<4> { using type = uint32_t; };
template <> struct Piece<2> { using type = uint16_t; };

template <typename T, int V> union Elems {
    typename Piece<V * sizeof(T)>::type piece;
    T e[V];
};

// V: elements of a piece.  PAIRS: neighbours are pairs.
template <typename T, int V, bool PAIRS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    extern __shared__ float2 s_turn[];                // [row][pair]: (cos, sin) times the factor
    using P = typename Piece<V * sizeof(T)>::type;
    pdl_wait_then_release();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(p.block_rows), p.rows - row0));
    const int half = p.rot / 2, total = rows * static_cast<int>(p.by_heads.d) * p.items;
    const int turned = p.rot / (2 * V);               // items of a head that are rotated
    Elems<T, V> x[kAhead][2];
    // Where an item is: its two pieces, as loaded from or stored to.
    struct Place { int row, which, head, item, first, second; bool two; };
    auto place_of = [&](int i) {
        Place w;
        const int head = static_cast<int>(p.by_items.div(i));
        w.item = i - head * p.items;
        w.row = static_cast<int>(p.by_heads.div(head));
        w.head = head - w.row * static_cast<int>(p.by_heads.d);
        w.which = w.head >= p.heads[0] ? 1 : 0;
        if (w.which) w.head -= p.heads[0];
        const bool halves = !PAIRS && w.item < turned;
        w.first = halves ? w.item * V : w.item * 2 * V;
        w.second = halves ? w.first + half : w.first + V;
        w.two = w.second < p.head_dim;
        return w;
    };
    auto load = [&](int i, Elems<T, V> (&to)[2]) {
        const Place w = place_of(i);
        const T* from = static_cast<const T*>(p.in[w.which]) + (row0 + w.row) * p.in_stride[w.which] + static_cast<int64_t>(w.head) * p.head_dim;
        to[0].piece = *reinterpret_cast<const P*>(from + w.first);
        if (w.two) to[1].piece = *reinterpret_cast<const P*>(from + w.second);
    };
    // The first elements on their way while the angles are worked out.
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
        const int i = static_cast<int>(threadIdx.x) + u * kThreads;
        if (i < total) load(i, x[u]);
    }
    for (int i = threadIdx.x; i < rows * half; i += kThreads) {
        const int r = static_cast<int>(p.by_pairs.div(i)), pair = i - r * half;
        // (1 / 2 pi rounded to 64 bits: with the product's rounding 2^-52 of the turns)
        const double turns = static_cast<double>(p.positions[row0 + r]) * (static_cast<double>(p.inv_freq[pair]) * 0.15915494309189535);
        const float part = static_cast<float>(turns - rint(turns));
        float s, c;
        sincospif(2.0f * part, &s, &c);
        s_turn[i] = make_float2(c * p.factor, s * p.factor);
    }
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < total; i0 += kAhead * kThreads) {
        if (i0 >= kAhead * kThreads) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (i0 + u * kThreads < total) load(i0 + u * kThreads, x[u]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kThreads;
            if (i >= total) break;
            const Place w = place_of(i);
            if (w.item < turned) {
                const float2* turn = s_turn + w.row * half + w.item * V;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    // (pair k: elements k of both pieces, or 2k and 2k + 1 of the two together)
                    T& at_a = PAIRS ? x[u][2 * k / V].e[2 * k % V] : x[u][0].e[k];
                    T& at_b = PAIRS ? x[u][(2 * k + 1) / V].e[(2 * k + 1) % V] : x[u][1].e[k];
                    const float a = ElemTraits<T>::to_float(at_a), b = ElemTraits<T>::to_float(at_b);
                    const float2 t = turn[k];
                    at_a = ElemTraits<T>::from_float(fmaf(a, t.x, -(b * t.y)));
                    at_b = ElemTraits<T>::from_float(fmaf(b, t.x, a * t.y));
                }
            }
            T* to = static_cast<T*>(p.out[w.which]) + (row0 + w.row) * p.out_stride[w.which] + static_cast<int64_t>(w.head) * p.head_dim;
            *reinterpret_cast<P*>(to + w.first) = x[u][0].piece;
            if (w.two) *reinterpret_cast<P*>(to + w.second) = x[u][1].piece;
        }
    }
}

template <typename T, int V> int launch_width(const RotaryParams& in, bool pairs, bool in_place, cudaStream_t stream) {
    RotaryParams p = in;
    // In place only what is rotated is touched.
    p.items = p.rot / (2 * V) + (in_place ? 0 : (p.head_dim - p.rot + 2 * V - 1) / (2 * V));
    const int heads = p.heads[0] + p.heads[1];
    p.by_items = FastDiv(static_cast<uint32_t>(p.items));
    p.by_heads = FastDiv(static_cast<uint32_t>(heads));
    p.by_pairs = FastDiv(static_cast<uint32_t>(p.rot / 2));
    if (static_cast<int64_t>(heads) * p.items > (1 << 28)) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: too many heads");
    // Several rows to a block once there are blocks enough.
    p.block_rows = 1;
    while (p.block_rows < kMaxRows && p.rows >= 2 * p.block_rows * 8 * kSmCount) p.block_rows *= 2;
    const int64_t blocks = (p.rows + p.block_rows - 1) / p.block_rows;
    if (blocks > 0x7fffffffLL) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: too many rows");
    const size_t smem = static_cast<size_t>(p.block_rows) * (p.rot / 2) * sizeof(float2);
    const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
    const cudaError_t e = pairs ? launch_pdl(rotary_kernel<T, V, true>, grid, block, smem, stream, p) : launch_pdl(rotary_kernel<T, V, false>, grid, block, smem, stream, p);
    if (e != cudaSuccess) return fail(NVK_ERR_CUDA, "rotary_embedding kernel launch: %s", cudaGetErrorString(e));
    return check_launch("rotary_embedding kernel launch");
}

// The widest pieces that head, rotated part, strides and addresses allow.
template <typename T> int launch_typed(const RotaryParams& p, bool pairs, bool in_place, cudaStream_t stream) {
    auto allows = [&](int v) {
        if (p.head_dim % v != 0 || p.rot % (2 * v) != 0) return false;
        for (int i = 0; i < 2; ++i) {
            if (p.heads[i] > 0 && (p.in_stride[i] % v != 0 || p.out_stride[i] % v != 0 || !aligned_to(p.in[i], v * sizeof(T)) || !aligned_to(p.out[i], v * sizeof(T)))) return false;
        }
        return true;
    };
    if constexpr (sizeof(T) == 2) {
        if (allows(8)) return launch_width<T, 8>(p, pairs, in_place, stream);
    }
    if (allows(4)) return launch_width<T, 4>(p, pairs, in_place, stream);
    if (allows(2)) return launch_width<T, 2>(p, pairs, in_place, stream);
    return launch_width<T, 1>(p, pairs, in_place, stream);
}

}  // namespace

int launch_rotary(const RotaryArgs& a) {
    RotaryParams p{};
    p.in[0] = a.query; p.in[1] = a.key; p.out[0] = a.query_out; p.out[1] = a.key_out;
    p.in_stride[0] = a.query_stride; p.in_stride[1] = a.key_stride; p.out_stride[0] = a.query_out_stride; p.out_stride[1] = a.key_out_stride;
    p.positions = a.positions; p.inv_freq = a.inv_freq; p.rows = a.rows; p.factor = a.factor;
    p.heads[0] = a.num_q_heads; p.heads[1] = a.key != nullptr ? a.num_kv_heads : 0;
    p.head_dim = a.head_dim; p.rot = a.rotary_dim;
    const bool in_place = a.query_out == a.query && a.key_out == a.key;
    switch (a.dtype) {
        case NVK_BF16: return launch_typed<__nv_bfloat16>(p, a.interleaved, in_place, a.stream);
        case NVK_F16: return launch_typed<__half>(p, a.interleaved, in_place, a.stream);
        default: return launch_typed<float>(p, a.interleaved, in_place, a.stream);
    }
}

}  // namespace nvk
