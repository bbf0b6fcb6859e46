// Device code of paged decode attention on tensor cores (F16 / BF16 queries, head_dim 128; 16-bit, int8, e4m3 or 4-bit cache), shared
// by the decode kernels (decode_attn.cu) and the mixed prefill + decode kernel (prefill_attn_tc.cu).
//
// The op is HBM-bound: every K and V row of every context is read once.  A group of four warps (over a 4-bit cache also of eight) takes a range of the keys of one
// (sequence, KV head); the G = Hq / Hkv <= 8 query heads of the KV head are the columns of the MMA tile, so a K / V row is read once
// per KV head.  Each warp streams every fourth tile of 16 keys through a private ring of cp.async stages (no barrier in the main
// loop); at the end the four warps merge through shared memory.
//
// Three ways to share a sequence out, by the sizes the host knows:
//   chunks     ranges of `chunk_tokens` keys; where a context is longer than one, the ranges leave partial results (maximum, sum,
//              unnormalised output) in the workspace and a second kernel merges them;
//   per_seq    num_splits equal ranges of every sequence in one thread-block cluster, merged through distributed shared memory in
//              the same launch, without a workspace: for small steps;
//   halves     two chunks, each half of the table's row, in one cluster: a context that ends in the first is one block's alone.
//
// Cutting the whole batch's keys into equal runs that ignore sequence boundaries (each block sums up the contexts, warps or groups
// walk on from one sequence to the next with their rings full, a quarter of the work handed out dynamically) was built and measured:
// the main loop gains 2 to 15 %, but the pass over the contexts, the look-ups and three to eight partial results per sequence
// cost more: 48 us against 37 at 37 sequences of 100 to 2048 keys, 700 against 697 at 256 of 1024 to 8192.
#pragma once

#include "nvk_internal.cuh"

#include <type_traits>

namespace nvk {
namespace dec {

constexpr int kHeadDim = 128;
constexpr int kTileTokens = 16;
constexpr int kMaxGroup = 8;           // query heads per KV head
constexpr int kGroupWarps = 4;
constexpr int kGroupThreads = kGroupWarps * 32;
constexpr int kMergeWarps = 8;         // warps that merge the parts of one (sequence, head) where there are many

struct DecodeParams {
    const void* q; const void* k_cache; const void* v_cache;
    const __half* k_scale; const __half* v_scale;      // 8-bit caches: a scale; 4-bit ones: a pair (step, low) in the queries' type, one 32-bit word
    IndexArray context_lens; IndexArray block_tables;
    void* out; float* ws_o; float2* ws_ml;             // partial results: [sequence][KV head][split][group][128] and (maximum, sum)
    int64_t max_blocks, num_cache_blocks;
    int batch, num_heads, num_kv_heads, group, block_size;
    int chunk_tokens, num_splits;
    int per_seq;                                       // 1: num_splits equal ranges per sequence instead of chunks
    int longest_first;                                 // blocks take the sequences in order of falling context length
    int chunk_major;                                   // decode_split_kernel's grid: all sequences' first chunks, then all second ones, ...
    int split_shift;                                   // clusters: log2 of num_splits
    int beside;                                        // waits at its end (pdl_wait_beside)
    float* scores;                                     // where they are kept (F::kScores): [sequence][KV head][max_blocks * block_size][group], times log2(e)
    KeyWeights weights;                                // what becomes of them
    FastDiv by_block, by_kv_heads;
    float scale_log2;
};

// A context length, limited to what the block table can address (max_blocks * block_size), and not negative.
__device__ __forceinline__ int clamped_context(const DecodeParams& p, IndexArray::Raw raw) {
    const int64_t ctx = p.context_lens.value(raw);
    const int64_t cap = p.max_blocks * p.block_size;
    return static_cast<int>(ctx < 0 ? 0 : ctx < cap ? ctx : cap);
}
__device__ __forceinline__ int clamped_context(const DecodeParams& p, int b) { return clamped_context(p, p.context_lens.raw(b)); }
// Range i of a context has keys [i * len, min(ctx, (i + 1) * len)).
__device__ __forceinline__ int range_len(const DecodeParams& p, int ctx) {
    return p.per_seq ? (((ctx + p.num_splits - 1) >> p.split_shift) + kTileTokens - 1) / kTileTokens * kTileTokens : p.chunk_tokens;
}
// Lane i: entry base + i of a sequence's block table, as loaded.  Entries past the context are loaded and not used.
__device__ __forceinline__ IndexArray::Raw load_ids(const DecodeParams& p, int b, int base, int lane) {
    return p.block_tables.raw(b * p.max_blocks + base + lane, base + lane < p.max_blocks);
}

__device__ __forceinline__ void group_sync(int bar_id, int threads) { asm volatile("bar.sync %0, %1;\n" ::"r"(bar_id), "r"(threads) : "memory"); }

// ---- cache formats: how a tile is fetched and what a warp does with it ---------------------------------------------------
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void lds32x4(uint32_t addr, uint32_t (&w)[4]) {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}

// 8 x 8 matrix of 16-bit elements over a warp (lane (g, t): row g, columns 2t, 2t + 1), transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}

// Online-softmax state of a warp.  Lane (g, t) = (lane / 4, lane % 4) holds heads 2t and 2t + 1: columns of the accumulators, the
// maxima (equal over g) and, over the keys that the lane has seen, the sums.
struct SoftmaxState {
    float o[8][4];
    float m[2], l[2];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int i = 0; i < 8; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f; }
        m[0] = m[1] = -INFINITY; l[0] = l[1] = 0.0f;
    }
    // Scores of a tile: rescale where a maximum moves (a handful of tiles of a sequence; the branch is warp-uniform).  `extra`: further
    // columns that are scaled along.
    __device__ __forceinline__ void raise_max(const float (&sc)[4], float* extra) {
        float top[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
            float c[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
                const float m_new = fmaxf(m[h], top[h]);   // finite: the tile's first key is always valid
                c[h] = fast_exp2(m[h] - m_new);
                l[h] *= c[h];
                m[h] = m_new;
            }
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) { o[mt][0] *= c[0]; o[mt][1] *= c[1]; o[mt][2] *= c[0]; o[mt][3] *= c[1]; }
            if (extra != nullptr) { extra[0] *= c[0]; extra[1] *= c[1]; extra[2] *= c[0]; extra[3] *= c[1]; }
        }
    }
};

// Scores of lane (g, t): keys g (sc[0], sc[1]) and g + 8 (sc[2], sc[3]), heads 2t and 2t + 1 of each.  Keys past `valid` of a tile get no
// weight; only a sequence's last tile has any (warp-uniform branch).
__device__ __forceinline__ void mask_scores(float (&sc)[4], int g, int valid) {
    if (valid < kTileTokens) {
        if (g >= valid) sc[0] = sc[1] = -INFINITY;
        if (g + 8 >= valid) sc[2] = sc[3] = -INFINITY;
    }
}

// Scores that are kept: the warp's tiles are every fourth one, and a lane's place moves on with them.
struct ScoreOut {
    float* at;                                         // key g of the warp's next tile, head 2t
    __device__ __forceinline__ void start(const DecodeParams& p, int b, int kvh, int token, int lane) {
        const int64_t keys = p.max_blocks * p.block_size;
        at = p.scores + ((static_cast<int64_t>(b) * p.num_kv_heads + kvh) * keys + token + (lane >> 2)) * p.group + 2 * (lane & 3);
    }
    __device__ __forceinline__ void put16(const float (&sc)[4], int row0, int valid, int lane, int group) const {
        const int g = lane >> 2, h = 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (row0 + g + 8 * i < valid && h < group) {
                float* to = at + (row0 + 8 * i) * group;
                if ((group & 1) == 0) {
                    *reinterpret_cast<float2*>(to) = make_float2(sc[2 * i], sc[2 * i + 1]);
                } else {
                    to[0] = sc[2 * i];
                    if (h + 1 < group) to[1] = sc[2 * i + 1];
                }
            }
        }
    }
    __device__ __forceinline__ void put(const DecodeParams& p, const float (&sc)[4], int valid, int lane) {   // tiles of 16 keys
        put16(sc, 0, valid, lane, p.group);
        at += kGroupWarps * 16 * p.group;
    }
    __device__ __forceinline__ void put(const DecodeParams& p, const float (&sa)[4], const float (&sb)[4], int valid, int lane, int warps) {   // of 32
        put16(sa, 0, valid, lane, p.group);
        put16(sb, 16, valid, lane, p.group);
        at += warps * 32 * p.group;
    }
};

// 16-bit cache.  K and V tiles of 16 x 256 bytes, XOR-swizzled by row; S^T = K Q^T as mma.sync m16n8k16: the 16 keys are the rows,
// the (zero padded) query heads the 8 columns; O^T = V^T P^T with V^T taken straight from the row-major V tile by ldmatrix.trans and
// P^T from S^T by two 8 x 8 transposes.  (Heads as the 16 rows need no transpose but twice the MMAs, half of them on padding, in a
// chain twice as long.)  Even and odd k-steps have accumulators of their own: a step is a serial chain that few warps hide.
// Measured: 37 sequences of up to 2048 keys 34.8 -> 33.7 us; 100 int8 ones of up to 4096, where the step is closer to the bound, 97 -> 89.
// 8 warps per SM x 3 stages of 8 KiB: 128 KiB in flight.
template <typename T, bool SCORES = false>
struct Cache16 {
    static constexpr bool kScores = SCORES;
    static constexpr bool kFourBits = false;
    static constexpr int kWarps = kGroupWarps;
    static constexpr int kGroups = 2;   // resident per SM
    static constexpr int kSplitBlocks = kGroups;
    static constexpr int kRowBytes = kHeadDim * 2;
    static constexpr int kTileBytes = kTileTokens * kRowBytes;
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr int kStages = 3;
    static constexpr int kPartStride = kHeadDim + 8;

    SoftmaxState s;
    ScoreOut kept;       // (SCORES)
    uint32_t qa[8][2];   // head g of the 8-column B tile; zero from head G on

    __device__ __forceinline__ void start(const DecodeParams& p, int b, int kvh, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const bool live = g < p.group;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(
            static_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.num_heads + kvh * p.group + (live ? g : 0)) * kHeadDim);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            qa[ks][0] = live ? row[ks * 8 + t] : 0u;
            qa[ks][1] = live ? row[ks * 8 + 4 + t] : 0u;
        }
        s.reset();
    }
    // Rows row0 .. row0 + valid - 1 of the cache into a stage; the rest of the tile is zero-filled (stale cache contents, even NaN,
    // never reach the arithmetic).
    static __device__ __forceinline__ void issue(const DecodeParams& p, int kvh, int64_t row0, int valid, uint32_t stage, int lane) {
        const size_t stride = static_cast<size_t>(p.num_kv_heads) * kRowBytes;
        const int c = lane & 15, rhalf = lane >> 4;   // 16-byte piece c of rows 2 i + rhalf
        const size_t base = static_cast<size_t>(row0) * stride + static_cast<size_t>(kvh) * kRowBytes + c * 16;
        const unsigned char* kc = static_cast<const unsigned char*>(p.k_cache) + base;
        const unsigned char* vc = static_cast<const unsigned char*>(p.v_cache) + base;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 2 * i + rhalf;
            const int bytes = r < valid ? 16 : 0;
            const size_t src = bytes ? r * stride : 0;
            const uint32_t dst = stage + r * kRowBytes + ((c ^ (r & 7)) << 4);
            cp_async16(dst, kc + src, bytes);
            cp_async16(dst + kTileBytes, vc + src, bytes);
        }
    }
    __device__ __forceinline__ void step(const DecodeParams& p, uint32_t stage, int valid, int /*kvh*/, int lane) {
        // ldmatrix lane addressing.  K: matrices (tok 0-7, d lo), (tok 0-7, d hi), (tok 8-15, d lo), (tok 8-15, d hi) of one
        // 16-wide k-step.  V (transposed): the same of one 16-wide d-tile.
        const int row = ((lane >> 4) << 3) + (lane & 7), sel = (lane >> 3) & 1;
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            uint32_t k0, k1, k2, k3;
            ldmatrix_x4(k0, k1, k2, k3, stage + row * kRowBytes + (((2 * ks + sel) ^ (row & 7)) << 4));
            mma_16816<T>(ks & 1 ? s1 : s0, k0, k2, k1, k3, qa[ks][0], qa[ks][1]);
        }
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[i] = (s0[i] + s1[i]) * p.scale_log2;
        mask_scores(sc, lane >> 2, valid);
        if constexpr (SCORES) kept.put(p, sc, valid, lane);
        s.raise_max(sc, nullptr);
        const float p0 = fast_exp2(sc[0] - s.m[0]), p1 = fast_exp2(sc[1] - s.m[1]), p2 = fast_exp2(sc[2] - s.m[0]), p3 = fast_exp2(sc[3] - s.m[1]);
        s.l[0] += p0 + p2;
        s.l[1] += p1 + p3;
        const uint32_t pb0 = transpose_8x8(ElemTraits<T>::pack2(p0, p1)), pb1 = transpose_8x8(ElemTraits<T>::pack2(p2, p3));
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
            uint32_t a0, a1, a2, a3;
            ldmatrix_x4_trans(a0, a1, a2, a3, stage + kTileBytes + row * kRowBytes + (((2 * mt + sel) ^ (row & 7)) << 4));
            mma_16816<T>(s.o[mt], a0, a1, a2, a3, pb0, pb1);
        }
    }
    __device__ __forceinline__ void finish() {}   // (after the last tile, by the whole warp)
    // The warp's unnormalised output of head 2t + h.
    __device__ __forceinline__ void write_part(float* row, int h, int g) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) row[8 * i + g] = s.o[i >> 1][(i & 1) * 2 + h];
    }
};

// Two 8-bit cache elements -> two f16 (MMA operand halves).  int8: the byte glued under the exponent byte of 1024 (the word has
// had its sign bits flipped: value + 1152, taken out algebraically afterwards); e4m3: the hardware conversion, exact.
template <bool FP8> __device__ __forceinline__ uint32_t widen_pair_lo(uint32_t x) {   // bytes 0, 1
    if constexpr (FP8) {
        uint32_t d;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(d) : "h"(static_cast<unsigned short>(x & 0xffffu)));
        return d;
    } else {
        return __byte_perm(x, 0x64646464u, 0x4140);
    }
}
template <bool FP8> __device__ __forceinline__ uint32_t widen_pair_hi(uint32_t x) {   // bytes 2, 3
    if constexpr (FP8) {
        uint32_t d;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(d) : "h"(static_cast<unsigned short>(x >> 16)));
        return d;
    } else {
        return __byte_perm(x, 0x64646464u, 0x4342);
    }
}

// 8-bit cache (int8, the reference's format: src/kernels/attention.cu:746-842; or e4m3 of the same layout): per token and KV head
// 128 bytes of K, 128 of V and two fp16 scales.  The MMA fragments are built from the bytes in registers -- no widened copy in
// shared memory, no ldmatrix:
//   * an int8 x becomes the fp16 number 1024 + (x + 128) by gluing the byte (x ^ 0x80) under the exponent byte 0x64 (one PRMT per
//     pair); the constant 1152 is taken out afterwards: q . (k' - 1152) = q . k' - 1152 * sum(q), and P (v' - 1152) = P v' - 1152 *
//     sum(P), where sum(P) comes from one extra MMA per tile against a row of ones, i.e. from exactly the rounded probabilities the
//     other MMAs used;
//   * the MMAs contract over d (scores) and over keys (output); a contraction does not care in which order its index runs, and
//     neither does the output care which accumulator row holds which d, so every lane takes whole 16-byte pieces: for K, piece 4q + t
//     of key row g supplies its k-steps 4q .. 4q + 3 (the query fragment is loaded with the same permutation); for V, piece g of key
//     rows 2t, 2t+1, 2t+8, 2t+9 supplies all eight d-tiles after a byte interleave of row pairs (two PRMTs), and accumulator row g /
//     g + 8 of d-tile 2a + e holds d = 16 g + 4 a + 2 e (+ 1);
//   * pieces are XOR-swizzled in the ring so that those 16-byte reads are conflict free.
// The scales never touch the tiles: k_scale multiplies the score of its key after the first MMA, v_scale the probability of its key
// before the second (the row sum uses the unscaled probability).  MMAs run as f16 whatever the query type: the query is converted
// once, probabilities are <= 1.  12 warps per SM x 4 stages of 4.1 KiB: 148 KiB in flight.
template <typename T, bool FP8>
struct Cache8 {
    static constexpr bool kScores = false;
    static constexpr bool kFourBits = false;
    static constexpr int kWarps = kGroupWarps;
    static constexpr int kGroups = 3, kSplitBlocks = kGroups;
    static constexpr int kRowBytes = kHeadDim;
    static constexpr int kTileBytes = kTileTokens * kRowBytes;
    static constexpr int kScaleBytes = 2 * kTileTokens * 4;   // one 32-bit word per (K | V, token): the word that holds its fp16 scale
    static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes;
    static constexpr int kStages = 4;
    static constexpr int kPartStride = kHeadDim + 4;
    static constexpr float kOffset = FP8 ? 0.0f : 1152.0f;    // 1024 (exponent glue) + 128 (sign flip)
    static constexpr uint32_t kFlip = FP8 ? 0u : 0x80808080u; // int8: sign bits flipped before the glue

    SoftmaxState s;
    float osum[4];       // sum of the (scaled, rounded) probabilities per head, from the ones-row MMA
    float q_off[2];
    uint32_t qa[8][2];   // k-step ks = 4 q + w, positions {2t, 2t+1 | 2t+8, 2t+9} <- d = 64 q + 16 t + 4 w + {0, 1 | 2, 3}

    __device__ __forceinline__ void start(const DecodeParams& p, int b, int kvh, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const bool live = g < p.group;
        const T* row = static_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.num_heads + kvh * p.group + (live ? g : 0)) * kHeadDim;
        float qsum = 0.0f;   // of the f16-rounded query row g
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            const int d0 = 64 * (ks >> 2) + 16 * t + 4 * (ks & 3);
#pragma unroll
            for (int hlf = 0; hlf < 2; ++hlf) {
                const __half2 h2 = __floats2half2_rn(ElemTraits<T>::to_float(row[d0 + 2 * hlf]), ElemTraits<T>::to_float(row[d0 + 2 * hlf + 1]));
                qa[ks][hlf] = live ? *reinterpret_cast<const uint32_t*>(&h2) : 0u;
                if (live) qsum += __low2float(h2) + __high2float(h2);
            }
        }
        qsum += __shfl_xor_sync(0xffffffffu, qsum, 1);
        qsum += __shfl_xor_sync(0xffffffffu, qsum, 2);
        q_off[0] = kOffset * __shfl_sync(0xffffffffu, qsum, 8 * t);
        q_off[1] = kOffset * __shfl_sync(0xffffffffu, qsum, 8 * t + 4);
        osum[0] = osum[1] = osum[2] = osum[3] = 0.0f;
        s.reset();
    }
    static __device__ __forceinline__ void issue(const DecodeParams& p, int kvh, int64_t row0, int valid, uint32_t stage, int lane) {
        const size_t stride = static_cast<size_t>(p.num_kv_heads) * kRowBytes;
        const int c = lane & 7, rq = lane >> 3;   // 16-byte piece c of rows 4 i + rq; ring swizzles: K piece c ^ ((r & 1) << 2), V piece c ^ (r & 6)
        const size_t base = static_cast<size_t>(row0) * stride + static_cast<size_t>(kvh) * kRowBytes + c * 16;
        const unsigned char* kc = static_cast<const unsigned char*>(p.k_cache) + base;
        const unsigned char* vc = static_cast<const unsigned char*>(p.v_cache) + base;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * i + rq;
            const int bytes = r < valid ? 16 : 0;
            const size_t src = bytes ? r * stride : 0;
            cp_async16(stage + r * kRowBytes + ((c ^ ((r & 1) << 2)) << 4), kc + src, bytes);
            cp_async16(stage + kTileBytes + r * kRowBytes + ((c ^ (r & 6)) << 4), vc + src, bytes);
        }
        // the scale of token (lane & 15): lanes 0-15 K, lanes 16-31 V; copied as the aligned 32-bit word around it
        const int tr = lane & 15;
        const int sbytes = tr < valid ? 4 : 0;
        const size_t sidx = sbytes ? (static_cast<size_t>(row0) + tr) * p.num_kv_heads + kvh : 0;
        cp_async4(stage + 2 * kTileBytes + lane * 4, (lane < 16 ? p.k_scale : p.v_scale) + (sidx & ~static_cast<size_t>(1)), sbytes);
    }
    __device__ __forceinline__ void step(const DecodeParams& p, uint32_t stage, int valid, int kvh, int lane) {
        const int g = lane >> 2, t = lane & 3;
        // Scales of keys g and g + 8.  Which half of a copied word is the scale: cache rows of a tile start at an even row, so the parity of
        // row * Hkv + kvh is that of (token & Hkv & 1) + kvh.
        float2 kscale, vscale;
        {
            uint32_t w[4];
            const uint32_t at = stage + 2 * kTileBytes + g * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(w[i]) : "r"(at + i * 32));
            const uint32_t pick = (((g & p.num_kv_heads) ^ kvh) & 1) != 0 ? 0x7632u : 0x5410u;
            const uint32_t k2 = __byte_perm(w[0], w[1], pick), v2 = __byte_perm(w[2], w[3], pick);
            kscale = __half22float2(*reinterpret_cast<const __half2*>(&k2));
            vscale = __half22float2(*reinterpret_cast<const __half2*>(&v2));
            kscale.x *= p.scale_log2;
            kscale.y *= p.scale_log2;
        }
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            uint32_t w0[4], w1[4];
            lds32x4(stage + g * kRowBytes + (((4 * q + t) ^ ((g & 1) << 2)) << 4), w0);
            lds32x4(stage + (g + 8) * kRowBytes + (((4 * q + t) ^ ((g & 1) << 2)) << 4), w1);
#pragma unroll
            for (int wi = 0; wi < 4; ++wi) {
                const int ks = 4 * q + wi;
                const uint32_t x0 = w0[wi] ^ kFlip, x1 = w1[wi] ^ kFlip;
                mma_16816<__half>(ks & 1 ? s1 : s0, widen_pair_lo<FP8>(x0), widen_pair_lo<FP8>(x1), widen_pair_hi<FP8>(x0), widen_pair_hi<FP8>(x1), qa[ks][0],
                                  qa[ks][1]);
            }
        }
        float sc[4] = {(s0[0] + s1[0] - q_off[0]) * kscale.x, (s0[1] + s1[1] - q_off[1]) * kscale.x, (s0[2] + s1[2] - q_off[0]) * kscale.y,
                       (s0[3] + s1[3] - q_off[1]) * kscale.y};
        mask_scores(sc, g, valid);
        s.raise_max(sc, FP8 ? nullptr : osum);
        const float p0 = fast_exp2(sc[0] - s.m[0]), p1 = fast_exp2(sc[1] - s.m[1]), p2 = fast_exp2(sc[2] - s.m[0]), p3 = fast_exp2(sc[3] - s.m[1]);
        s.l[0] += p0 + p2;
        s.l[1] += p1 + p3;
        const uint32_t pb0 = transpose_8x8(ElemTraits<__half>::pack2(p0 * vscale.x, p1 * vscale.x));
        const uint32_t pb1 = transpose_8x8(ElemTraits<__half>::pack2(p2 * vscale.y, p3 * vscale.y));
        // output: V rows 2t, 2t+1, 2t+8, 2t+9, piece g (d = 16 g .. 16 g + 15)
        uint32_t v0[4], v1[4], v2[4], v3[4];
        const uint32_t vbase = stage + kTileBytes;
        lds32x4(vbase + (2 * t) * kRowBytes + ((g ^ ((2 * t) & 6)) << 4), v0);
        lds32x4(vbase + (2 * t + 1) * kRowBytes + ((g ^ ((2 * t + 1) & 6)) << 4), v1);
        lds32x4(vbase + (2 * t + 8) * kRowBytes + ((g ^ ((2 * t + 8) & 6)) << 4), v2);
        lds32x4(vbase + (2 * t + 9) * kRowBytes + ((g ^ ((2 * t + 9) & 6)) << 4), v3);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const uint32_t x0 = v0[a] ^ kFlip, x1 = v1[a] ^ kFlip, x2 = v2[a] ^ kFlip, x3 = v3[a] ^ kFlip;
            // bytes of one d from two consecutive keys, side by side
            const uint32_t lo01 = __byte_perm(x0, x1, 0x5140), hi01 = __byte_perm(x0, x1, 0x7362);
            const uint32_t lo23 = __byte_perm(x2, x3, 0x5140), hi23 = __byte_perm(x2, x3, 0x7362);
            mma_16816<__half>(s.o[2 * a], widen_pair_lo<FP8>(lo01), widen_pair_hi<FP8>(lo01), widen_pair_lo<FP8>(lo23), widen_pair_hi<FP8>(lo23), pb0, pb1);
            mma_16816<__half>(s.o[2 * a + 1], widen_pair_lo<FP8>(hi01), widen_pair_hi<FP8>(hi01), widen_pair_lo<FP8>(hi23), widen_pair_hi<FP8>(hi23), pb0, pb1);
        }
        constexpr uint32_t kOnes = 0x3C003C00u;   // {1.0, 1.0}
        if (!FP8) mma_16816<__half>(osum, kOnes, kOnes, kOnes, kOnes, pb0, pb1);
    }
    __device__ __forceinline__ void finish() {}
    __device__ __forceinline__ void write_part(float* row, int h, int g) const {
        const float off = kOffset * osum[h];
#pragma unroll
        for (int i = 0; i < 8; i += 2)
            *reinterpret_cast<float4*>(row + 16 * g + 2 * i) = make_float4(s.o[i][h] - off, s.o[i][2 + h] - off, s.o[i + 1][h] - off, s.o[i + 1][2 + h] - off);
    }
};

// 4-bit cache: per token and KV head 64 bytes of K, 64 of V (numbers n from 0 to 15, element 2i in the low half of byte i) and for each a
// pair (step, low) in the queries' type; an element is low + step n.  The MMA operands are made from the nibbles in registers: a nibble in bits 0 to 3
// of an f16 is the subnormal number n 2^-24, in bits 4 to 7 it is 16 n 2^-24, exactly, so that a word of eight nibbles gives its four registers for one shift
// and four ANDs, whatever the queries' type.  Queries are brought to f16 by a power of two, each head's own (exact but for
// elements below 2^-24 of the head's largest), those that meet a number times 16 divided by it; sums are fp32:
//   q . x         = step 2^24 (q . n 2^-24) + low sum(q)
//   sum_k p_k x_k = 2^E (2^24 sum_k p'_k n_k 2^-24 - 7.5 sum_k p'_k) + sum_k p_k (low_k + 7.5 step_k),   p'_k = p_k step_k 2^-E rounded to f16
// p' is the one rounding to 16 bits (as with the other caches).  With F16 results the middle of the range goes in the fp32 sum at the right, so that what the
// rounding touches is no larger than the values' spread, and sum(p') comes from an MMA against a row of ones, i.e. from exactly the p' that the others used;
// a BF16 result is rounded to an eighth of p''s precision, and the 7.5 and the MMA are left out.  2^E is each head's own and goes by p step: the largest p' is at
// least 1/8 when E is chosen, and all are held to 2^-22 of the largest or better.  (By the largest step alone, a key that hardly any attention went to could take the others' bits: one
// whose step was 2^20 times theirs cost them 10 to 20 %.)  E is chosen, and the sums are rescaled, where a score passes the last maximum by 8 or a step reaches 2^(7 + E): p' < 2^15.
// (At every new maximum, the ranges of 8 to 16 tiles a warp of few long contexts came there at nearly every tile.)
// As in Cache8 the order in which a contraction runs is free: of key row g lane t takes the 16-byte piece t, whose word w has the k-steps
// 2w and 2w + 1 (registers: elements {0, 4}, {1, 5}; {2, 6}, {3, 7}; the query fragment is loaded the same way).  Of V lane (g, t) takes 8 bytes,
// d = 16 g .. 16 g + 15, of keys 2t, 2t + 1, 2t + 8, 2t + 9; with halves of two keys' words side by side the same masks give both keys' numbers, and accumulator
// rows g / g + 8 of d-tile i hold d = 16 g + 2 i and d = 16 g + 2 i + 1 (times 16).  The two rows of a 128-byte line of V are swizzled by the line's number, so
// that these reads are conflict free.
// A quarter of the bytes, for as many MMAs: per warp and 32 keys some 570 cycles of a scheduler, of which the MMAs and the masks take most, and 64 sequences of 500 to
// 4096 keys, 32 / 8 heads, take 46.0 us where the bytes take 24.6.  No unit is near its limit then (issue slots 52 % busy, the ALU pipe 51 %, tensor 25 %, DRAM 47 %): blocks
// of uneven length leave SMs idle for a fifth of the time, and latency takes the rest.
// A warp takes 32 keys at a time, two chains of 16: the arithmetic of a tile is one long chain, and the four warps of a scheduler (three in clusters) do not hide it.  The cache
// rows of its next 16 tiles are worked out by the lanes, one half of a tile each, while the ids of the 16 after them are on their way.
template <int AT> __device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1], 16;\n" ::"r"(dst), "l"(src), "n"(AT));
}
template <int AT> __device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0+%2], [%1], 4;\n" ::"r"(dst), "l"(src), "n"(AT));
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126 <= e <= 127

template <typename T, bool SCORES = false, int WARPS = kGroupWarps>
struct Cache4 {
    using Eight = Cache4<T, SCORES, 8>;                       // eight warps to a block
    static constexpr bool kScores = SCORES;
    static constexpr bool kFourBits = true;
    static constexpr int kWarps = WARPS;
    static constexpr int kGroups = 3;                         // resident per SM in clusters; a step is shared out by it in chunks too, as with the 8-bit caches
    static constexpr int kSplitBlocks = 16 / WARPS;           // in chunks: the registers are there, and the chains are what a warp waits for
    static constexpr int kRowBytes = kHeadDim / 2;
    static constexpr int kKeys = 32;                          // of a stage
    static constexpr int kKeysAhead = 32 * 8 * kKeys + 16;    // two windows of 16 tiles, of eight warps at most, and a half: how far `run` counts beyond the last key
    static constexpr int kTileBytes = kKeys * kRowBytes;
    static constexpr int kStageBytes = 2 * kTileBytes + 2 * kKeys * 4;   // K, V, (step, low) of K and of V
    static constexpr int kStages = 3;
    static constexpr int kPartStride = kHeadDim + 4;
    static constexpr bool kCentred = std::is_same<T, __half>::value;
    static constexpr float kSlack = 8.0f;                     // by so much a score may pass s.m: p <= 2^8
    static constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u, kNone = 0xffffffffu;

    SoftmaxState s;
    ScoreOut kept;       // (SCORES)
    float ones[4];       // sum(p')
    float mid[2];        // sum(p (low + 7.5 step)) of heads 2t, 2t + 1 over the lane's keys
    float q_sum[2], step_scale[2];
    float down[2];       // 2^-E of heads 2t, 2t + 1
    float top_part[2];   // the largest log2(p step) so far, p without the maximum taken off
    uint32_t qa[8][2];   // k-step 2 w + e: elements 32 t + 8 w + 2 e + {0, 4 | 1, 5}

    __device__ __forceinline__ void start(const DecodeParams& p, int b, int kvh, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const bool live = g < p.group;
        const uint4* row = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) + (static_cast<int64_t>(b) * p.num_heads + kvh * p.group + (live ? g : 0)) * kHeadDim) + 4 * t;
        float sum = 0.0f, top = 0.0f;
        uint4 v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = live ? row[w] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t e[4] = {v[w].x, v[w].y, v[w].z, v[w].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2<T>(e[i]);
                sum += f.x + f.y;
                top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
        }
#pragma unroll
        for (int x = 1; x < 4; x *= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        }
        // the head's largest to [2^14, 2^15); (infinities and NaN stay what they are)
        const int up = top > 0.0f && top < INFINITY ? min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 100) : 0;
        const float even = power_of_two(up), odd = even * 0.0625f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 e01 = unpack2<T>(v[w].x), e23 = unpack2<T>(v[w].y), e45 = unpack2<T>(v[w].z), e67 = unpack2<T>(v[w].w);
            qa[2 * w][0] = ElemTraits<__half>::pack2(e01.x * even, e45.x * even);
            qa[2 * w][1] = ElemTraits<__half>::pack2(e01.y * odd, e45.y * odd);
            qa[2 * w + 1][0] = ElemTraits<__half>::pack2(e23.x * even, e67.x * even);
            qa[2 * w + 1][1] = ElemTraits<__half>::pack2(e23.y * odd, e67.y * odd);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            q_sum[h] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * h) * p.scale_log2;
            step_scale[h] = p.scale_log2 * 0x1p24f * power_of_two(-__shfl_sync(0xffffffffu, up, 8 * t + 4 * h));
        }
        ones[0] = ones[1] = ones[2] = ones[3] = mid[0] = mid[1] = 0.0f;
        down[0] = down[1] = 0x1p126f;
        top_part[0] = top_part[1] = -INFINITY;
        s.reset();
    }
    static __device__ __forceinline__ void lds64(uint32_t addr, uint2& v) { asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr)); }
    // Scores of 16 keys, rows `row0` on of a stage; their (step, low) of V.
    __device__ __forceinline__ void score(uint32_t stage, int row0, int lane, float (&sc)[4], float2 (&vp)[2]) const {
        const int g = lane >> 2, t = lane & 3;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w0[4], w1[4];
        uint2 w[2];
        lds32x4(stage + (row0 + g) * kRowBytes + t * 16, w0);
        lds32x4(stage + (row0 + g + 8) * kRowBytes + t * 16, w1);
#pragma unroll
        for (int i = 0; i < 2; ++i) lds64(stage + 2 * kTileBytes + (row0 + g + 8 * i) * 8, w[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x0 = w0[i] >> 8, x1 = w1[i] >> 8;
            mma_16816<__half>(acc, w0[i] & kLow, w1[i] & kLow, w0[i] & kHigh, w1[i] & kHigh, qa[2 * i][0], qa[2 * i][1]);
            mma_16816<__half>(acc, x0 & kLow, x1 & kLow, x0 & kHigh, x1 & kHigh, qa[2 * i + 1][0], qa[2 * i + 1][1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 kp = unpack2<T>(w[i].x);
            vp[i] = unpack2<T>(w[i].y);
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[2 * i + h] = fmaf(acc[2 * i + h], kp.x * step_scale[h], kp.y * q_sum[h]);
        }
    }
    __device__ __forceinline__ int exponent(int h) const { return 127 - static_cast<int>(__float_as_uint(down[h]) >> 23); }   // E
    // Where a score passes s.m by more than kSlack, or a p' could leave f16.  s.m is then the maximum, and E is chosen again: the largest p' of the tiles that came here is between
    // 1/8 and 1/4.
    __device__ __forceinline__ void raise(const float (&sa)[4], const float (&sb)[4], const float2 (&va)[2], const float2 (&vb)[2]) {
        const float a0 = __log2f(fabsf(va[0].x)), a1 = __log2f(fabsf(va[1].x)), b0 = __log2f(fabsf(vb[0].x)), b1 = __log2f(fabsf(vb[1].x));
        float c[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = fmaxf(fmaxf(sa[h], sa[2 + h]), fmaxf(sb[h], sb[2 + h])), part = fmaxf(fmaxf(sa[h] + a0, sa[2 + h] + a1), fmaxf(sb[h] + b0, sb[2 + h] + b1));
#pragma unroll
            for (int x = 4; x < 32; x *= 2) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                part = fmaxf(part, __shfl_xor_sync(0xffffffffu, part, x));
            }
            const float m_new = fmaxf(s.m[h], top);
            top_part[h] = fmaxf(top_part[h], part);
            const int was = exponent(h), e = static_cast<int>(fminf(fmaxf(ceilf(top_part[h] - m_new) + 2.0f, -126.0f), 126.0f));
            c[h] = s.m[h] == m_new ? 1.0f : fast_exp2(s.m[h] - m_new);
            s.l[h] *= c[h];
            mid[h] *= c[h];
            s.m[h] = m_new;
            c[h] *= power_of_two(min(max(was - e, -126), 127));   // (beyond that nothing is seen of what was there, or there was nothing)
            down[h] = power_of_two(-e);
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) { s.o[mt][0] *= c[0]; s.o[mt][1] *= c[1]; s.o[mt][2] *= c[0]; s.o[mt][3] *= c[1]; }
        ones[0] *= c[0]; ones[1] *= c[1]; ones[2] *= c[0]; ones[3] *= c[1];
    }
    // What 16 keys add to the sums.
    __device__ __forceinline__ void add(uint32_t stage, int row0, const float (&sc)[4], const float2 (&vp)[2], int lane) {
        const int g = lane >> 2, t = lane & 3;
        const float p0 = fast_exp2(sc[0] - s.m[0]), p1 = fast_exp2(sc[1] - s.m[1]), p2 = fast_exp2(sc[2] - s.m[0]), p3 = fast_exp2(sc[3] - s.m[1]);
        s.l[0] += p0 + p2;
        s.l[1] += p1 + p3;
        const float mid0 = kCentred ? fmaf(vp[0].x, 7.5f, vp[0].y) : vp[0].y, mid1 = kCentred ? fmaf(vp[1].x, 7.5f, vp[1].y) : vp[1].y;
        mid[0] = fmaf(p0, mid0, fmaf(p2, mid1, mid[0]));
        mid[1] = fmaf(p1, mid0, fmaf(p3, mid1, mid[1]));
        // (p first: where it is 0, 2^-E step need not be finite)
        const uint32_t pb0 = transpose_8x8(ElemTraits<__half>::pack2(p0 * down[0] * vp[0].x, p1 * down[1] * vp[0].x));
        const uint32_t pb1 = transpose_8x8(ElemTraits<__half>::pack2(p2 * down[0] * vp[1].x, p3 * down[1] * vp[1].x));
        // V rows 2t, 2t + 1 (line t) and 2t + 8, 2t + 9 (line t + 4), words 2g and 2g + 1: half of piece g / 2
        const uint32_t v_at = stage + kTileBytes + row0 * kRowBytes + t * 128 + (g & 1) * 8, even = ((g >> 1) ^ (t << 1)) << 4;
        uint2 x[4];
        lds64(v_at + even, x[0]);
        lds64(v_at + (even ^ 64), x[1]);
        lds64(v_at + 512 + even, x[2]);
        lds64(v_at + 512 + (even ^ 64), x[3]);
        auto four = [&](uint32_t k01, uint32_t k89, int i) {   // d-tiles i and i + 1 of two keys' halves side by side
            mma_16816<__half>(s.o[i], k01 & kLow, k01 & kHigh, k89 & kLow, k89 & kHigh, pb0, pb1);
            k01 >>= 8;
            k89 >>= 8;
            mma_16816<__half>(s.o[i + 1], k01 & kLow, k01 & kHigh, k89 & kLow, k89 & kHigh, pb0, pb1);
        };
        four(__byte_perm(x[0].x, x[1].x, 0x5410), __byte_perm(x[2].x, x[3].x, 0x5410), 0);
        four(__byte_perm(x[0].x, x[1].x, 0x7632), __byte_perm(x[2].x, x[3].x, 0x7632), 2);
        four(__byte_perm(x[0].y, x[1].y, 0x5410), __byte_perm(x[2].y, x[3].y, 0x5410), 4);
        four(__byte_perm(x[0].y, x[1].y, 0x7632), __byte_perm(x[2].y, x[3].y, 0x7632), 6);
        constexpr uint32_t kOnes = 0x3c003c00u;
        if (kCentred) mma_16816<__half>(ones, kOnes, kOnes, kOnes, kOnes, pb0, pb1);
    }
    // 32 keys, of which `valid` (more than none) are there.
    __device__ __forceinline__ void step(const DecodeParams& p, uint32_t stage, int valid, int lane) {
        float sa[4], sb[4];
        float2 va[2], vb[2];
        score(stage, 0, lane, sa, va);
        score(stage, 16, lane, sb, vb);
        if (valid < kKeys) {
            mask_scores(sa, lane >> 2, valid);
            mask_scores(sb, lane >> 2, valid - 16);
        }
        if constexpr (SCORES) kept.put(p, sa, sb, valid, lane, WARPS);
        const float top0 = fmaxf(fmaxf(sa[0], sa[2]), fmaxf(sb[0], sb[2])), top1 = fmaxf(fmaxf(sa[1], sa[3]), fmaxf(sb[1], sb[3]));
        const float top_step = fmaxf(fmaxf(fabsf(va[0].x), fabsf(va[1].x)), fmaxf(fabsf(vb[0].x), fabsf(vb[1].x)));
        if (__any_sync(0xffffffffu, fmaxf(top0 - s.m[0], top1 - s.m[1]) > kSlack || top_step * fmaxf(down[0], down[1]) >= 0x1p7f)) raise(sa, sb, va, vb);
        add(stage, 0, sa, va, lane);
        add(stage, 16, sb, vb, lane);
    }
    // One multiplication with a 64-bit sum: the ALU is the busiest pipe here.
    static __device__ __forceinline__ const void* row_at(uint32_t unit, const unsigned char* base) {
        uint64_t at;
        asm("mad.wide.u32 %0, %1, %2, %3;\n" : "=l"(at) : "r"(unit), "n"(kRowBytes), "l"(base));
        return reinterpret_cast<const void*>(at);
    }
    static __device__ __forceinline__ const void* word_at(uint32_t unit, const uint32_t* base) {
        uint64_t at;
        asm("mad.wide.u32 %0, %1, 4, %2;\n" : "=l"(at) : "r"(unit), "l"(base));
        return reinterpret_cast<const void*>(at);
    }

    // Keys [t0, t1): this warp's tiles of 32, every WARPS-th one.
    __device__ __forceinline__ void run(const DecodeParams& p, int b, int kvh, int t0, int t1, IndexArray::Raw raw_ids, int id_base, uint32_t ring, int warp, int lane) {
        const int tiles = (t1 - t0 + kKeys - 1) / kKeys, mine = tiles > warp ? (tiles - warp + WARPS - 1) / WARPS : 0;
        const int bs = p.block_size, first = t0 + warp * kKeys;
        constexpr int kStride = WARPS * kKeys;
        // Lane 2i + h: half h of tile i of a window of 16 tiles, the place of its first row among all head vectors of the cache.
        auto token_of = [&](int window) { return first + (window * 16 + (lane >> 1)) * kStride + (lane & 1) * 16; };
        auto load = [&](int window) {
            const int token = token_of(window);
            const int blk = static_cast<int>(p.by_block.div(token < t1 ? token : 0));
            return p.block_tables.raw(b * p.max_blocks + blk, token < t1);
        };
        auto unit_of = [&](int window, IndexArray::Raw raw) {
            const int token = token_of(window), off = token - static_cast<int>(p.by_block.div(token < t1 ? token : 0)) * bs;
            const int64_t id = p.block_tables.value(raw);
            return token < t1 && id >= 0 && id < p.num_cache_blocks ? (static_cast<uint32_t>(id) * bs + off) * p.num_kv_heads + kvh : kNone;
        };
        uint32_t units;
        {   // the first window from the ids that came with the context, if they reach that far
            const int token = token_of(0), at = static_cast<int>(p.by_block.div(token < t1 ? token : t0)) - id_base;
            IndexArray::Raw raw{__shfl_sync(0xffffffffu, raw_ids.lo, at), __shfl_sync(0xffffffffu, raw_ids.hi, at)};
            if (__any_sync(0xffffffffu, at >= 32)) raw = load(0);
            units = unit_of(0, raw);
        }
        IndexArray::Raw next = load(1);
        const int r = lane >> 2, c = lane & 3;
        const size_t row_bytes = static_cast<size_t>(p.num_kv_heads) * kRowBytes;
        const unsigned char* k_at = static_cast<const unsigned char*>(p.k_cache) + r * row_bytes + c * 16;
        const unsigned char* v_at = static_cast<const unsigned char*>(p.v_cache) + r * row_bytes + c * 16;
        const unsigned char *k8_at = k_at + 8 * row_bytes, *v8_at = v_at + 8 * row_bytes;
        const uint32_t* par_at = reinterpret_cast<const uint32_t*>(lane < 16 ? p.k_scale : p.v_scale) + static_cast<size_t>(lane & 15) * p.num_kv_heads;
        const uint32_t k_to = r * kRowBytes + c * 16, v_to = kTileBytes + (r >> 1) * 128 + (((((r & 1) << 2) + c) ^ (((r >> 1) & 3) << 1)) << 4);
        const uint32_t par_to = 2 * kTileBytes + (lane & 15) * 8 + (lane >> 4) * 4;
        int issued = 0, left = t1 - first;        // keys from the next tile on
        uint32_t istage = ring;
        auto issue = [&]() {
            if (issued < mine) {
                if ((issued & 15) == 0 && issued > 0) {
                    units = unit_of(issued >> 4, next);
                    next = load((issued >> 4) + 1);
                }
                const uint32_t u0 = __shfl_sync(0xffffffffu, units, 2 * issued), u1 = __shfl_sync(0xffffffffu, units, 2 * issued + 1);
                const uint32_t k_dst = istage + k_to, v_dst = istage + v_to, par_dst = istage + par_to;
                constexpr int kHalf = 16 * kRowBytes, kRow8 = 8 * kRowBytes;
                if (left >= kKeys && max(u0, u1) != kNone) {
                    cp_async16<0>(k_dst, row_at(u0, k_at));
                    cp_async16<kRow8>(k_dst, row_at(u0, k8_at));
                    cp_async16<kHalf>(k_dst, row_at(u1, k_at));
                    cp_async16<kHalf + kRow8>(k_dst, row_at(u1, k8_at));
                    cp_async16<0>(v_dst, row_at(u0, v_at));
                    cp_async16<kRow8>(v_dst, row_at(u0, v8_at));
                    cp_async16<kHalf>(v_dst, row_at(u1, v_at));
                    cp_async16<kHalf + kRow8>(v_dst, row_at(u1, v8_at));
                    cp_async4<0>(par_dst, word_at(u0, par_at));
                    cp_async4<128>(par_dst, word_at(u1, par_at));
                } else {   // what is not there reads as zeros (stale cache contents, even NaN, never reach the arithmetic)
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t unit = h == 0 ? u0 : u1;
                        const int valid = unit == kNone ? 0 : left - 16 * h;
                        const bool r0 = r < valid, r1 = r + 8 < valid, rp = (lane & 15) < valid;
                        nvk::cp_async16(k_dst + h * kHalf, r0 ? row_at(unit, k_at) : p.k_cache, r0 ? 16 : 0);
                        nvk::cp_async16(k_dst + h * kHalf + kRow8, r1 ? row_at(unit, k8_at) : p.k_cache, r1 ? 16 : 0);
                        nvk::cp_async16(v_dst + h * kHalf, r0 ? row_at(unit, v_at) : p.v_cache, r0 ? 16 : 0);
                        nvk::cp_async16(v_dst + h * kHalf + kRow8, r1 ? row_at(unit, v8_at) : p.v_cache, r1 ? 16 : 0);
                        dec::cp_async4(par_dst + h * 128, rp ? word_at(unit, par_at) : p.k_scale, rp ? 4 : 0);
                    }
                }
                ++issued;
                left -= kStride;
                istage = istage == ring + (kStages - 1) * kStageBytes ? ring : istage + kStageBytes;
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) issue();
        start(p, b, kvh, lane);
        if constexpr (SCORES) kept.start(p, b, kvh, first, lane);
        uint32_t cstage = ring;
        int here = t1 - first;
        for (int j = 0; j < mine; ++j) {
            issue();
            cp_async_wait<kStages - 1>();
            __syncwarp();
            step(p, cstage, here, lane);
            __syncwarp();   // the stage is refilled by other lanes' copies
            cstage = cstage == ring + (kStages - 1) * kStageBytes ? ring : cstage + kStageBytes;
            here -= kStride;
        }
    }
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) mid[h] += __shfl_xor_sync(0xffffffffu, mid[h], x);
        }
    }
    __device__ __forceinline__ void write_part(float* row, int h, int g) const {
        const float up = power_of_two(exponent(h)), off = kCentred ? fmaf(ones[h] * -7.5f, up, mid[h]) : mid[h];
        auto even = [&](int i) { return fmaf(s.o[i][h] * 0x1p24f, up, off); };
        auto odd = [&](int i) { return fmaf(s.o[i][2 + h] * 0x1p20f, up, off); };
#pragma unroll
        for (int i = 0; i < 8; i += 2) *reinterpret_cast<float4*>(row + 16 * g + 2 * i) = make_float4(even(i), odd(i), even(i + 1), odd(i + 1));
    }
};

// ---- a group's range of keys ---------------------------------------------------------------------------------------------
template <class F>
struct alignas(128) GroupSmem {
    union Warp {
        unsigned char ring[F::kStages * F::kStageBytes];
        struct {                                       // what the warp leaves for the merge, when its ring is idle
            float o[kMaxGroup * F::kPartStride];       // head 2 t + h in row 4 h + t: the lanes of a store hit different banks
            float2 ml[kMaxGroup];
        } part;
    } warps[F::kWarps];
};

// The warp's tiles of keys [t0, t1), every fourth one, through its ring.
template <class F>
__device__ __forceinline__ void stream_tiles(const DecodeParams& p, int b, int kvh, int t0, int t1, IndexArray::Raw raw_ids, int id_base, uint32_t ring, int warp,
                                             int lane, F& st) {
    const int bs = p.block_size;
    const int num_tiles = (t1 - t0 + kTileTokens - 1) / kTileTokens;
    const int my_tiles = num_tiles > warp ? (num_tiles - warp + kGroupWarps - 1) / kGroupWarps : 0;
    // The issuing end: this warp's next tile begins at row `off` of table entry `blk`.  Lane i holds the cache block of entry
    // id_base + i (-1: outside the cache, reads as zeros).
    int tok = t0 + warp * kTileTokens;
    int blk = static_cast<int>(p.by_block.div(tok)), off = tok - blk * bs, ids;
    auto take_ids = [&](IndexArray::Raw raw) {
        const int64_t id = p.block_tables.value(raw);
        ids = (id >= 0 && id < p.num_cache_blocks) ? static_cast<int>(id) : -1;
    };
    auto move_window = [&]() {
        if (blk - id_base >= 32 && tok < t1) {
            id_base = blk;
            take_ids(load_ids(p, b, id_base, lane));
        }
    };
    take_ids(raw_ids);
    move_window();   // (a warp may begin just past what was loaded)
    uint32_t istage = ring;
    auto issue = [&]() {
        if (tok < t1) {
            const int phys = __shfl_sync(0xffffffffu, ids, blk - id_base);
            F::issue(p, kvh, phys < 0 ? 0 : static_cast<int64_t>(phys) * bs + off, phys < 0 ? 0 : t1 - tok, istage, lane);
            istage = istage == ring + (F::kStages - 1) * F::kStageBytes ? ring : istage + F::kStageBytes;
            tok += kGroupWarps * kTileTokens;
            for (off += kGroupWarps * kTileTokens; off >= bs; off -= bs) ++blk;
            move_window();
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < F::kStages - 1; ++s) issue();

    st.start(p, b, kvh, lane);
    if constexpr (F::kScores) st.kept.start(p, b, kvh, t0 + warp * kTileTokens, lane);
    uint32_t cstage = ring;
    int left = t1 - t0 - warp * kTileTokens;   // keys from this warp's tile on
    for (int j = 0; j < my_tiles; ++j) {
        issue();
        cp_async_wait<F::kStages - 1>();
        __syncwarp();
        st.step(p, cstage, left, kvh, lane);
        __syncwarp();   // the stage is refilled by other lanes' copies
        cstage = cstage == ring + (F::kStages - 1) * F::kStageBytes ? ring : cstage + F::kStageBytes;
        left -= kGroupWarps * kTileTokens;
    }
}

// Keys [t0, t1) of sequence b (t0 < t1), one KV head.  sink(h, quad, o, m, l) takes elements 4 quad .. 4 quad + 3 of head h: unnormalised
// output, maximum and sum.  `tid`: 0..127 inside the group, `bar_id`: its named barrier; all its threads call it.  `raw_ids`: block
// table entries `id_base` + lane as loaded.  The four warps' parts come together in one trip over all heads, after one barrier (a warp writes
// its part over its own ring; before, two barriers and a loop over the heads, a trip each).
template <class F, class Sink>
__device__ __forceinline__ void attend_range(const DecodeParams& p, int b, int kvh, int t0, int t1, IndexArray::Raw raw_ids, int id_base, GroupSmem<F>& sm,
                                             int tid, int bar_id, Sink sink) {
    const int warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = smem_u32(sm.warps[warp].ring);
    F st;
    if constexpr (F::kFourBits) st.run(p, b, kvh, t0, t1, raw_ids, id_base, ring, warp, lane);
    else stream_tiles(p, b, kvh, t0, t1, raw_ids, id_base, ring, warp, lane, st);
    cp_async_wait<0>();
    __syncwarp();                              // this warp's ring is idle from here on
    st.finish();
    const int g = lane >> 2, t = lane & 3;
    auto& part = sm.warps[warp].part;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float l = st.s.l[h];
#pragma unroll
        for (int x = 4; x < 32; x *= 2) l += __shfl_xor_sync(0xffffffffu, l, x);
        if (2 * t + h < p.group) {
            if (g == 0) part.ml[2 * t + h] = make_float2(st.s.m[h], l);
            st.write_part(part.o + (4 * h + t) * F::kPartStride, h, g);
        }
    }
    group_sync(bar_id, F::kWarps * 32);
    for (int h = warp; h < p.group; h += F::kWarps) {
        float4 o[F::kWarps];
        float2 ml[F::kWarps];
#pragma unroll
        for (int w = 0; w < F::kWarps; ++w) {
            const auto& from = sm.warps[w].part;
            ml[w] = from.ml[h];
            o[w] = *reinterpret_cast<const float4*>(from.o + (4 * (h & 1) + (h >> 1)) * F::kPartStride + 4 * lane);
        }
        float mx = ml[0].x, sum = 0.0f;
        float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 1; w < F::kWarps; ++w) mx = fmaxf(mx, ml[w].x);
#pragma unroll
        for (int w = 0; w < F::kWarps; ++w) {
            const float f = fast_exp2(ml[w].x - mx);   // 0 for a warp without a tile
            total.x = fmaf(f, o[w].x, total.x); total.y = fmaf(f, o[w].y, total.y); total.z = fmaf(f, o[w].z, total.z); total.w = fmaf(f, o[w].w, total.w);
            sum = fmaf(f, ml[w].y, sum);
        }
        sink(h, lane, total, mx, sum);
    }
}

template <typename T> __device__ __forceinline__ void write_quad(T* at, const float4& v) {   // four elements of a result
    *reinterpret_cast<uint2*>(at) = make_uint2(ElemTraits<T>::pack2(v.x, v.y), ElemTraits<T>::pack2(v.z, v.w));
}
__device__ __forceinline__ float4 scaled(const float4& v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

// Keys [t0, t1) of (b, kvh): new = old + sum over the heads of exp2(score - M) / L, with (M, 1 / L) of the whole context in `ml`.  By the block that has these keys'
// scores, which come back from L2: a kernel of its own after it took 9 us of 105 for 64 sequences of 500 to 4096 keys, 32 / 8 heads.
template <int THREADS>
__device__ __forceinline__ void add_key_weights(const DecodeParams& p, int b, int kvh, int t0, int t1, const float2* ml, int tid) {
    const KeyWeights& w = p.weights;
    const int64_t row = w.rows != nullptr ? w.rows[b] : b;
    if (row < 0 || row >= w.num_rows) return;
    const int group = p.group;
    const float* scores = p.scores + (static_cast<int64_t>(b) * p.num_kv_heads + kvh) * p.max_blocks * p.block_size * group;
    const int64_t at = (row * p.num_kv_heads + kvh) * w.row_keys;
    float2 heads[kMaxGroup];
#pragma unroll
    for (int h = 0; h < kMaxGroup; ++h) heads[h] = h < group ? ml[h] : make_float2(0.0f, 0.0f);
    constexpr int kAhead = 4;
    auto trip = [&](auto load, auto count) {   // `count` heads of a key by load(key, to)
        for (int k0 = t0 + tid; k0 < t1; k0 += kAhead * THREADS) {
            float sc[kAhead][count.value], old[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int k = min(k0 + i * THREADS, t1 - 1);
                load(scores + static_cast<int64_t>(k) * group, sc[i]);
                old[i] = w.old_weights != nullptr ? w.old_weights[at + k] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                float sum = 0.0f;
#pragma unroll
                for (int h = 0; h < count.value; ++h)
                    if (h < group) sum = fmaf(fast_exp2(sc[i][h] - heads[h].x), heads[h].y, sum);
                if (k0 + i * THREADS < t1) w.new_weights[at + k0 + i * THREADS] = old[i] + sum;
            }
        }
    };
    if (group == 4) {
        trip([](const float* from, float* to) {
            const float4 v = *reinterpret_cast<const float4*>(from);
            to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        }, std::integral_constant<int, 4>());
    } else if (group == 2) {
        trip([](const float* from, float* to) {
            const float2 v = *reinterpret_cast<const float2*>(from);
            to[0] = v.x; to[1] = v.y;
        }, std::integral_constant<int, 2>());
    } else {
        trip([group](const float* from, float* to) {
#pragma unroll
            for (int h = 0; h < kMaxGroup; ++h) to[h] = from[h < group ? h : 0];
        }, std::integral_constant<int, kMaxGroup>());
    }
}

// Range `split` of (b, kvh): the result if it is all of the context, else a part in the workspace.  `heads`: room for (M, 1 / L) of every head (F::kScores).
template <class F, typename T>
__device__ __forceinline__ void run_split(const DecodeParams& p, int b, int kvh, int split, GroupSmem<F>& sm, int tid, int bar_id, float2* heads = nullptr) {
    const int lane = tid & 31;
    const IndexArray::Raw raw_ctx = p.context_lens.raw(b);
    // The first range's block ids on their way with the context: a trip to memory less.  Further chunks look whether they have keys first: with tables
    // much wider than the contexts nearly all blocks are of this kind (256 sequences of 100 to 300 keys, 8 KV heads, 32768-key tables, 32768
    // blocks: 82 us a pass, 106 with ids for all), and they leave before anything else (128 such sequences: 56.7 -> 50.8 us a call).
    const bool early = p.per_seq || split == 0;
    int id_base = 0;
    IndexArray::Raw raw_ids{0, 0};
    if (early) raw_ids = load_ids(p, b, 0, lane);
    const int ctx = clamped_context(p, raw_ctx);
    if (!p.per_seq && split > 0 && static_cast<int64_t>(split) * p.chunk_tokens >= ctx) return;
    const int len = range_len(p, ctx), t0 = split * len, t1 = min(ctx, t0 + len);
    if (!early) {
        id_base = static_cast<int>(p.by_block.div(t0));
        raw_ids = load_ids(p, b, id_base, lane);
    }
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.num_heads + kvh * p.group) * kHeadDim;
    if (t0 >= t1) {
        if (ctx == 0 && split == 0) {
            for (int i = tid; i < p.group * kHeadDim; i += F::kWarps * 32) out[i] = ElemTraits<T>::from_float(0.0f);
        }
        return;
    }
    const size_t part = (static_cast<size_t>(b) * p.num_kv_heads + kvh) * p.num_splits + split;
    attend_range<F>(p, b, kvh, t0, t1, raw_ids, id_base, sm, tid, bar_id, [&](int h, int quad, const float4& o, float m, float l) {
        if (ctx <= len) {
            write_quad(out + h * kHeadDim + 4 * quad, scaled(o, 1.0f / l));   // (rounded as write_merged does)
        } else {
            reinterpret_cast<float4*>(p.ws_o + (part * p.group + h) * kHeadDim)[quad] = o;
            if (!F::kScores && quad == 0) p.ws_ml[part * p.group + h] = make_float2(m, l);
        }
        if (F::kScores && quad == 0) {   // (the weights of the keys need them, however many parts there are)
            if (p.num_splits == 1) heads[h] = make_float2(m, 1.0f / l);
            else p.ws_ml[part * p.group + h] = make_float2(m, l);
        }
    });
    if constexpr (F::kScores) {
        if (p.num_splits == 1) {
            group_sync(bar_id, F::kWarps * 32);
            add_key_weights<F::kWarps * 32>(p, b, kvh, t0, t1, heads, tid);
        }
    }
}

// ---- merging the parts of a sequence -------------------------------------------------------------------------------------
// HG heads of one (sequence, KV head) at a time.  Where there can be few parts one warp takes them in order, otherwise they are
// dealt over kMergeWarps warps.
struct PartRef { const float* o; const float2* ml; };   // head 0 of a part
struct Merged {                                         // elements 4 lane .. 4 lane + 3 of a head's output, maximum and row sum
    float4 o;
    float m, l;
    // Four parts at a time (every merge in the same order, so that who merges makes no difference to a bit); one that is not there: zeros, with a
    // maximum of minus infinity.
    __device__ __forceinline__ void add(const float4 (&v)[4], const float2 (&ml)[4]) {
        const float mx = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x))), f = fast_exp2(m - mx);
        o = scaled(o, f);
        l *= f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float w = fast_exp2(ml[u].x - mx);
            o.x = fmaf(w, v[u].x, o.x); o.y = fmaf(w, v[u].y, o.y); o.z = fmaf(w, v[u].z, o.z); o.w = fmaf(w, v[u].w, o.w);
            l = fmaf(w, ml[u].y, l);
        }
        m = mx;
    }
};
__device__ __forceinline__ Merged nothing_merged() { return Merged{make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.0f}; }

// Heads h0 .. h0 + HG - 1 (clamped to the group) over parts first, first + stride, ...
template <int HG, class Get>
__device__ __forceinline__ void sum_parts(Get get, int n, int first, int stride, int h0, int group, int lane, Merged (&acc)[HG]) {
    constexpr int U = HG == 4 ? 4 : 8;   // parts in flight
#pragma unroll
    for (int h = 0; h < HG; ++h) acc[h] = nothing_merged();
    for (int i0 = first; i0 < n; i0 += U * stride) {
        float2 ml[U][HG];
        float4 v[U][HG];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const PartRef r = get(min(i0 + u * stride, n - 1));   // (loads without branches, so that all are in flight at once)
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                const int hh = min(h0 + h, group - 1);
                ml[u][h] = r.ml[hh];
                v[u][h] = *reinterpret_cast<const float4*>(r.o + hh * kHeadDim + 4 * lane);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u += 4) {
            if (i0 + u * stride < n) {
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    float4 four[4];
                    float2 ml4[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool there = i0 + (u + k) * stride < n;
                        four[k] = there ? v[u + k][h] : make_float4(0.f, 0.f, 0.f, 0.f);
                        ml4[k] = there ? ml[u + k][h] : make_float2(-INFINITY, 0.0f);
                    }
                    acc[h].add(four, ml4);
                }
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void write_merged(T* row, const Merged& a, int lane) {
    const float inv = a.l > 0.0f ? 1.0f / a.l : 0.0f;
    write_quad(row + 4 * lane, scaled(a.o, inv));
}
// Heads h0 .. h0 + HG - 1 of the group, rows of `out`, by one warp.
template <typename T, int HG, class Get>
__device__ __forceinline__ void merge_by_warp(Get get, int n, int h0, int group, T* out, int lane) {
    Merged acc[HG];
    sum_parts<HG>(get, n, 0, 1, h0, group, lane, acc);
#pragma unroll
    for (int h = 0; h < HG; ++h)
        if (h0 + h < group) write_merged<T>(out + (h0 + h) * kHeadDim, acc[h], lane);
}
// One head, by the whole block; the first kMergeWarps warps work.
struct MergeScratch { float4 o[kMergeWarps][32]; float2 ml[kMergeWarps]; };
template <typename T, class Get>
__device__ __forceinline__ void merge_by_block(Get get, int n, int head, int group, T* row, MergeScratch& sm, int warp, int lane) {
    if (warp < kMergeWarps) {
        Merged acc[1];
        sum_parts<1>(get, n, warp, kMergeWarps, head, group, lane, acc);
        sm.o[warp][lane] = acc[0].o;
        if (lane == 0) sm.ml[warp] = make_float2(acc[0].m, acc[0].l);
    }
    __syncthreads();
    if (warp == 0) {
        Merged a = nothing_merged();
#pragma unroll
        for (int w = 0; w < kMergeWarps; w += 4)
            a.add({sm.o[w][lane], sm.o[w + 1][lane], sm.o[w + 2][lane], sm.o[w + 3][lane]}, {sm.ml[w], sm.ml[w + 1], sm.ml[w + 2], sm.ml[w + 3]});
        write_merged<T>(row, a, lane);
    }
    __syncthreads();
}

}  // namespace dec
}  // namespace nvk
