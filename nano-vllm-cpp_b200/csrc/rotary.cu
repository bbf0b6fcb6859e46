// Rotary positions on query and key heads: any position, pairs of halves or of neighbours, all of a head or its first part, any frequencies.
//
// Beside the fused prologue (fused_prologue.cu), whose rotation is over halves of a whole head and goes by a table of cosines: here
//   (a, b) -> factor (a cos t - b sin t, b cos t + a sin t),   t = position * frequency of the pair,
// with pairs (i, i + rot / 2) or (2i, 2i + 1) of the first `rot` elements; the others are copied.  The reference rotates whole heads by halves
// (src/kernels/split_qkv.cu:62-154).
//
// Far out in a long context position * frequency has no bits left for the angle in 32 bits (position 2^20: off by up to 1/16), nor, further out, in 64 (2^40: by 2^-13 of a turn).  So the
// turns are taken as the sum of two 64-bit numbers, off by some 2^-104 of themselves, and only their fraction goes on to sincospi in 32: off by 2^-26 of a turn, whatever the position up to
// 2^53.  A row's angles are worked out once for all its heads: a handful of 64-bit operations for each pair of a row, next to Hq + Hkv times as many elements.
//
// Bound by HBM for many rows (every element is read and written once), by the trip to memory and the launch for few.  A thread takes two pieces of V elements of a head, i and rot / 2 + i,
// which hold V pairs whole in either layout, and the lanes' pieces lie next to each other (pairs of neighbours in two pieces next to each other: 59.2 instead of 53.9 us below, in F32 56.3 instead
// of 50.5).  Two pairs are turned by one instruction (f32x2), three items of a thread are under way at once, in 64 registers: 16384 rows of 32 / 8 heads of 128, BF16, halves, take 54.9 us
// (6.1 TB/s; one pair at a time 62.7, four items at once 57.0, two 58.1), neighbours 53.9, 4096 rows 13.1, one row 1.9.  Where half of the rotated part is no multiple of 16 bytes all of a
// head goes in the pieces that it allows, what is only copied too: 16384 rows of 32 / 8 heads of 80 with 20 rotated, BF16, 71.9 us (2.9 TB/s; in place, where nothing is copied, 22.8), of 96
// with 24 82.3 (3.1; 21.6), of 80 with 20 in F32 87.9 (4.8; 36.2).
#include "nvk_internal.cuh"

#include <algorithm>
#include <type_traits>

namespace nvk {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 3;         // items of a thread under way
constexpr int kMaxRows = 16;      // of a block

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
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(const __grid_constant__ RotaryParams p) {
    extern __shared__ __align__(16) float s_cos[];    // [row][pair], times the factor; the sines behind them
    constexpr bool kApart = !PAIRS || V >= 2;         // an item's pieces lie half of the rotated part from each other (neighbours of one element each: next to each other)
    constexpr int kEach = PAIRS && V >= 2 ? V / 2 : V;   // from the angles of an item to those of the next
    using P = typename Piece<V * sizeof(T)>::type;
    pdl_wait_then_release();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.block_rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(p.block_rows), p.rows - row0));
    const int half = p.rot / 2, total = rows * static_cast<int>(p.by_heads.d) * p.items;
    const int turned = p.rot / (2 * V);               // items of a head that are rotated
    float* s_sin = s_cos + p.block_rows * half;
    Elems<T, V> x[kAhead][2];
    // Where an item is; its two pieces lie `second` elements from each other, 0: it has only one.  (Worked out again for the store: to keep it costs more registers than there are.)
    struct Place { int row, which, off, second, angle; };
    auto place_of = [&](int i) {
        const int all = static_cast<int>(p.by_items.div(i)), item = i - all * p.items;
        const int row = static_cast<int>(p.by_heads.div(all)), head = all - row * static_cast<int>(p.by_heads.d);
        const bool halves = kApart && item < turned;
        Place w;
        w.row = row;
        w.which = head >= p.heads[0] ? 1 : 0;
        w.off = (head - (w.which ? p.heads[0] : 0)) * p.head_dim + (halves ? item * V : item * 2 * V);
        w.second = halves ? half : item * 2 * V + V < p.head_dim ? V : 0;
        w.angle = item < turned ? row * half + item * kEach : -1;
        return w;
    };
    auto load = [&](int i, Elems<T, V> (&v)[2]) {
        const Place w = place_of(i);
        const T* from = static_cast<const T*>(p.in[w.which]) + (row0 + w.row) * p.in_stride[w.which] + w.off;
        v[0].piece = *reinterpret_cast<const P*>(from);
        if (w.second != 0) v[1].piece = *reinterpret_cast<const P*>(from + w.second);
    };
    // The first elements on their way while the angles are worked out.
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
        const int i = static_cast<int>(threadIdx.x) + u * kThreads;
        if (i < total) load(i, x[u]);
    }
    for (int i = threadIdx.x; i < rows * half; i += kThreads) {
        const int r = static_cast<int>(p.by_pairs.div(i)), pair = i - r * half;
        // Turns as the sum of two numbers of 64 bits: the frequency's turns for a position, then for this one.
        constexpr double kTurn = 0.15915494309189535, kTurnRest = -9.839338337591243e-18;   // 1 / 2 pi
        const double f = static_cast<double>(p.inv_freq[pair]), at = static_cast<double>(p.positions[row0 + r]);
        const double each = f * kTurn, each_rest = fma(f, kTurnRest, fma(f, kTurn, -each));
        const double turns = at * each, rest = fma(at, each_rest, fma(at, each, -turns));
        const float part = static_cast<float>((turns - rint(turns)) + rest);
        float s, c;
        sincospif(2.0f * part, &s, &c);
        s_cos[i] = c * p.factor;
        s_sin[i] = s * p.factor;
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
            if (i0 + u * kThreads >= total) break;
            const Place w = place_of(i0 + u * kThreads);
            if (w.angle >= 0) {
                using E = ElemTraits<T>;
                // Pairs k and k + 1 of a piece, or of both; where their angles are.
                auto turn2 = [&](T& a0, T& b0, T& a1, T& b1, int angle) {
                    const float2 c = *reinterpret_cast<const float2*>(s_cos + angle), s = *reinterpret_cast<const float2*>(s_sin + angle);
                    const F2 c2 = f2_make(c.x, c.y), s2 = f2_make(s.x, s.y), n2 = f2_make(-s.x, -s.y);
                    const F2 a = f2_make(E::to_float(a0), E::to_float(a1)), b = f2_make(E::to_float(b0), E::to_float(b1));
                    float first, second;
                    f2_split(f2_fma(a, c2, f2_mul(b, n2)), first, second);
                    a0 = E::from_float(first);
                    a1 = E::from_float(second);
                    f2_split(f2_fma(b, c2, f2_mul(a, s2)), first, second);
                    b0 = E::from_float(first);
                    b1 = E::from_float(second);
                };
                auto turn1 = [&](T& a0, T& b0, int angle) {
                    const float a = E::to_float(a0), b = E::to_float(b0), c = s_cos[angle], s = s_sin[angle];
                    a0 = E::from_float(fmaf(a, c, -(b * s)));
                    b0 = E::from_float(fmaf(b, c, a * s));
                };
                if constexpr (!PAIRS && V >= 2) {
#pragma unroll
                    for (int k = 0; k < V; k += 2) turn2(x[u][0].e[k], x[u][1].e[k], x[u][0].e[k + 1], x[u][1].e[k + 1], w.angle + k);
                } else if constexpr (PAIRS && V >= 4) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int k = 0; k < V; k += 4) turn2(x[u][i].e[k], x[u][i].e[k + 1], x[u][i].e[k + 2], x[u][i].e[k + 3], w.angle + i * (half / 2) + k / 2);
                } else if constexpr (PAIRS && V == 2) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) turn1(x[u][i].e[0], x[u][i].e[1], w.angle + i * (half / 2));
                } else {
                    turn1(x[u][0].e[0], x[u][1].e[0], w.angle);
                }
            }
            T* out = static_cast<T*>(p.out[w.which]) + (row0 + w.row) * p.out_stride[w.which] + w.off;
            *reinterpret_cast<P*>(out) = x[u][0].piece;
            if (w.second != 0) *reinterpret_cast<P*>(out + w.second) = x[u][1].piece;
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
    // As many rows to a block as its threads have under way at once, once there are blocks enough.
    const int row_items = heads * p.items;
    p.block_rows = 1;
    while (p.block_rows < kMaxRows && (p.block_rows + 1) * row_items <= kAhead * kThreads && p.rows >= (p.block_rows + 1) * 8 * kSmCount) ++p.block_rows;
    const int64_t blocks = (p.rows + p.block_rows - 1) / p.block_rows;
    if (blocks > 0x7fffffffLL) return fail(NVK_ERR_UNSUPPORTED, "rotary_embedding: too many rows");
    const size_t smem = static_cast<size_t>(p.block_rows) * (p.rot / 2) * 2 * sizeof(float);
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
