// Attention of several query rows per sequence on the matrix cores: the body
// shared by prompt attention (contiguous K/V, attention_prompt.hip) and tree
// attention (paged K/V, attention_tree.hip).
//
// Mathematics.  A row is one (token i, query head) pair; the G = n_heads /
// n_kv heads that share a K/V head are packed, row r = i G + head, so that a
// tile of rows reads every K/V byte once for all of them.  Per row, over its
// attended keys j: s_j = q . k_j, p_j = exp2(c (s_j - m)) with c = scale log2 e,
// out = sum p_j v_j / sum p_j, the maximum m and the sum running in f32.
//
// Layout.  A wavefront owns 32 rows and walks tiles of KT keys staged in LDS:
//  * S^T = K Q^T by v_mfma_f32_32x32x16: A = K (lane: key lane % 32, 8 dims),
//    B = Q^T held in registers.  Lane (n, h) = (lane % 32, lane / 32) then has
//    the scores of row n with keys 8 (i / 4) + 4 h + i % 4, i = 0..15: maximum
//    and sum are lane-local up to one exchange between the halves.
//  * O^T = V^T P^T: p is rounded to 16 bits where it is, in the B layout; the
//    order of keys inside a contraction is free, so V^T is read in the order
//    the scores came in, by ds_read_b64_tr_b16 (4 keys x 16 dims transposed
//    per 16 lanes).  O^T has its row in the lane too: rescaling is per lane.
//  * K and V go to LDS straight from memory (buffer loads with lds), double
//    buffered, one barrier per tile; keys past the end are out of the
//    resource's range and arrive as zeros.  The 16-byte pieces of a key row are
//    permuted by a bijection of the key's low bits (swizzle) that spreads both
//    the 16-key reads of K and the 4-key x 32-dim reads of V over all banks.
//  * The running maximum is raised only when a row's new maximum exceeds it by
//    more than kLazy (in log2): p stays below 2^kLazy, and most tiles skip the
//    rescaling of O.
// A masked score is -inf before the exp; a masked V that is not finite makes
// 0 x inf = NaN in the product, so rows whose result is not finite (or whose
// sum is zero though they attend keys) are computed again key by key, over their
// attended keys alone.  A row without keys is zero.
#pragma once

#include "common.hpp"

namespace fellm {
namespace rows_attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
using Rsrc = __amdgpu_buffer_rsrc_t;

constexpr uint32_t kRows = 32;         // rows of a wavefront
constexpr uint32_t kBlockTokens = 16;  // tokens of a cache block

// K/V element policies.  kBias: log2 added to every exponent, so that small
// probabilities stay normal f16 numbers; it cancels in out = O / l.
struct ElemF16 {
    using A = F16;
    static constexpr int kQParts = 2, kPParts = 2;  // parts that hold f32 operands
    static constexpr float kBias = 4.0f, kBiasParts = 15.0f;
    __device__ static f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    // Two values rounded to nearest even and packed; the remainders replace them.
    __device__ static uint32_t part(float &x, float &y) {
        typedef _Float16 half2 __attribute__((ext_vector_type(2)));
        const half2 h = {(_Float16)x, (_Float16)y};
        x -= (float)h[0];
        y -= (float)h[1];
        return __builtin_bit_cast(uint32_t, h);
    }
};
struct ElemBF16 {
    using A = BF16;
    static constexpr int kQParts = 3, kPParts = 3;
    static constexpr float kBias = 0.0f, kBiasParts = 0.0f;
    __device__ static f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ static uint32_t part(float &x, float &y) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        const bf2 h = {(__bf16)x, (__bf16)y};
        const uint32_t u = __builtin_bit_cast(uint32_t, h);
        x -= __uint_as_float(u << 16);
        y -= __uint_as_float(u & 0xffff0000u);
        return u;
    }
};

// Division by a number fixed at the launch, by a multiplication with its
// rounded-up reciprocal (Granlund and Montgomery, 1994).
struct Divisor {
    uint32_t d, m, s1, s2;
    Divisor() = default;
    explicit Divisor(uint32_t n) : d(n) {
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < n) ++l;
        m = (uint32_t)((((1ull << l) - n) << 32) / n + 1);
        s1 = l < 1 ? l : 1;
        s2 = l < 1 ? 0 : l - 1;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const {
        const uint32_t t = __umulhi(m, x);
        return (t + ((x - t) >> s1)) >> s2;
    }
};

struct Args {
    const void *q;
    void *out;
    const uint8_t *k, *v;   // contiguous K/V, 16-bit elements
    uint32_t k_stride, v_stride, q_stride, out_stride;  // elements per token row
    uint32_t q_dtype, out_dtype;
    const uint32_t *cu;     // [n_seqs + 1] first token of each sequence
    const uint32_t *before; // [n_seqs] cached keys before a sequence's first token, or null
    const uint32_t *mask;   // [tokens, mask_words] bits of the sequence's own tokens, or null
    uint32_t mask_words, n_seqs, tokens, n_heads, n_kv, group;
    Divisor by_group;
    float c;                // scale log2 e
    uint32_t causal, window;
    uint32_t max_before;    // bound that `before` is clamped to
    // paged K/V
    const uint8_t *arena;
    uint64_t arena_len, block_bytes, n_table;
    const uint32_t *table;
    uint32_t n_logical, n_layers, layer, stride;
    // the launch's share of the rounds of keys (paged): at least this many a
    // workgroup, the records of tiles that several share (null: whole tiles)
    uint32_t min_rounds;
    float *part;
};

// A tile of rows: sequence, its tokens and the keys before them.
struct Tile {
    uint32_t seq, row0;      // first packed row inside the sequence
    uint32_t first, n;       // first token in the packed tensors, tokens
    uint32_t before;
};

// Tiles are numbered so that no prefix sum over the sequences is needed:
// sequence b's first tile is floor(cu[b] G / BM) + b, which leaves room for its
// ceil(n_b G / BM) tiles; numbers past a sequence's rows are empty.
template <uint32_t BM>
__device__ __forceinline__ Tile find_tile(const Args &a, uint32_t t) {
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t lo = 0, len = a.n_seqs;
    while (len > 1) {
        const uint32_t step = (len + kWave - 1) / kWave, b = lane * step;
        const bool le = b < len && min(a.cu[lo + min(b, len - 1)], a.tokens) * a.group / BM + lo + b <= t;
        const uint32_t below = max(1u, (uint32_t)__popcll(__ballot(le)));
        lo += (below - 1) * step;
        len = min(step, len - (below - 1) * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    Tile r;
    r.seq = lo;
    r.first = min(a.cu[lo], a.tokens);
    const uint32_t end = min(a.cu[lo + 1], a.tokens);
    r.n = end > r.first ? end - r.first : 0;
    r.row0 = (t - (r.first * a.group / BM + lo)) * BM;
    r.before = a.before ? min(a.before[lo], a.max_before) : 0;
    if (r.row0 >= r.n * a.group) r.n = 0;
    return r;
}

// Sum of v over the wavefront, uniform.
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
    v += dpp_u32<0x140>(v);
    v += dpp_u32<0x141>(v);
    v += dpp_u32<0x4E>(v);
    v += dpp_u32<0xB1>(v);
    return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) +
           __builtin_amdgcn_readlane(v, 48);
}

__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    v = dpp_max_group<16>(v);
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// The tile of the given rank when the tiles of all sequences are ordered by
// their place in the sequence, the last first: under a causal mask those have
// the most keys, and workgroups that start last should have the least to do.
// (Seventeen f16 prompts of 128 to 2048 tokens, 28/4 heads of 128: 146 us with
// the tiles in the order of the sequences.)  It also numbers the tiles without
// gaps: workgroups are dealt to the shader engines in turn, and with every
// second one empty half of the CUs had no work (16 drafted tokens behind 32768,
// 32/8 heads of 128: 95 us).  Up to 64 sequences, one a lane: the level is
// found by search over sum_b max(0, T_b - level).
template <uint32_t BM>
__device__ __forceinline__ Tile ranked_tile(const Args &a, uint32_t rank) {
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t first = 0, n = 0;
    if (lane < a.n_seqs) {
        first = min(a.cu[lane], a.tokens);
        const uint32_t end = min(a.cu[lane + 1], a.tokens);
        n = end > first ? end - first : 0;
    }
    const uint32_t tiles = (n * a.group + BM - 1) / BM;
    Tile r{0, 0, 0, 0, 0};
    uint32_t level, seq = 0;
    if (a.n_seqs == 1) {
        const uint32_t t0 = __builtin_amdgcn_readfirstlane(tiles);
        if (rank >= t0) return r;
        level = t0 - 1 - rank;
    } else {
        if (wave_total(tiles) <= rank) return r;
        // tiles at levels >= lo: more than rank; >= hi: `above`, at most rank
        uint32_t lo = 0, hi = wave_most(tiles), above = 0;
        while (hi - lo > 1) {
            const uint32_t step = max(1u, (hi - lo) / 4);
            uint32_t c[3];
#pragma unroll
            for (uint32_t i = 0; i < 3; ++i) {
                const uint32_t at = lo + (i + 1) * step;
                c[i] = wave_total(tiles > at ? tiles - at : 0);
            }
            const uint32_t base = lo, top = hi;
#pragma unroll
            for (uint32_t i = 0; i < 3; ++i) {
                const uint32_t at = base + (i + 1) * step;
                if (at >= top) continue;
                if (c[i] > rank) lo = at;
                else if (at < hi) hi = at, above = c[i];
            }
        }
        level = lo;
        uint64_t at = __ballot(tiles > level);
        for (uint32_t k = rank - above; k; --k) at &= at - 1;
        seq = (uint32_t)__builtin_ctzll(at);
    }
    r.seq = seq;
    r.first = __builtin_amdgcn_readlane(first, seq);
    r.n = __builtin_amdgcn_readlane(n, seq);
    r.row0 = level * BM;
    r.before = a.before ? min(a.before[seq], a.max_before) : 0;
    return r;
}

template <uint32_t BM>
__device__ __forceinline__ Tile tile_of(const Args &a, uint32_t rank, uint32_t tiles) {
    return a.n_seqs <= kWave ? ranked_tile<BM>(a, rank) : find_tile<BM>(a, tiles - 1 - rank);
}

// Attended keys of token i: [lo, hi), all of them or, at and past `before`, those with a bit.
struct KeyRange {
    uint32_t lo, hi;
};
__device__ __forceinline__ KeyRange row_keys(const Args &a, const Tile &t, uint32_t i) {
    const uint32_t all = t.before + t.n;
    KeyRange r{0, all};
    if (a.mask) return r;
    if (a.causal) {
        r.hi = t.before + i + 1;
        if (a.window && r.hi > a.window) r.lo = r.hi - a.window;
    } else if (a.window) {
        r.lo = i >= a.window ? i - a.window + 1 : 0;
        r.hi = a.window < all - i ? i + a.window : all;
    }
    return r;
}

// Bit b: key kb + b (b < 64) is attended by the row.
__device__ __forceinline__ uint64_t key_bits(const Args &a, const Tile &t, uint32_t token, KeyRange r, uint32_t kb) {
    auto below = [&](uint32_t end) -> uint64_t {  // bits of keys < end
        const uint32_t n = end > kb ? end - kb : 0;
        return n >= 64 ? ~0ull : (1ull << n) - 1;
    };
    uint64_t bits = below(r.hi) & ~below(r.lo);
    if (a.mask && kb + 64 > t.before) {
        const uint64_t prefix = below(t.before);
        // the 64 mask bits from own token kb - before on (negative: none yet)
        const uint32_t *row = a.mask + (size_t)(t.first + token) * a.mask_words;
        const int64_t at = (int64_t)kb - (int64_t)t.before;
        const int32_t w = (int32_t)(at >> 5);
        const uint32_t sh = (uint32_t)(at & 31);
        uint32_t x[3];
#pragma unroll
        for (int e = 0; e < 3; ++e) x[e] = w + e >= 0 && (uint32_t)(w + e) < a.mask_words ? row[w + e] : 0;
        const uint64_t lo = x[0] | (uint64_t)x[1] << 32;
        const uint64_t own = sh ? lo >> sh | (uint64_t)x[2] << (64 - sh) : lo;
        bits &= prefix | own;
    }
    return bits;
}

// Table entry of cache block `blk` of the sequence, ~0 where the table has none,
// and the block's address, null where the arena has none.
__device__ __forceinline__ uint32_t block_entry(const Args &a, const Tile &t, uint32_t blk) {
    const size_t ti = ((size_t)t.seq * a.n_layers + a.layer) * a.n_logical + blk;
    return blk < a.n_logical && ti < a.n_table ? a.table[ti] : ~0u;
}
__device__ __forceinline__ const uint8_t *block_ptr(const Args &a, uint32_t entry) {
    return ((uint64_t)entry + 1) * a.block_bytes <= a.arena_len ? a.arena + entry * a.block_bytes : nullptr;
}

// Element pointers of key j (byte address), or null where the cache has no such block.
template <bool PAGED>
__device__ __forceinline__ const uint8_t *key_ptr(const Args &a, const Tile &t, uint32_t g, uint32_t hd, uint32_t j,
                                                  bool is_v) {
    if constexpr (PAGED) {
        const uint8_t *at = block_ptr(a, block_entry(a, t, j / kBlockTokens));
        return at ? at + ((uint64_t)(j % kBlockTokens + (is_v ? kBlockTokens : 0)) * a.stride + (uint64_t)g * hd) * 2 : nullptr;
    } else {
        const uint32_t stride = is_v ? a.v_stride : a.k_stride;
        return (is_v ? a.v : a.k) + ((size_t)(t.first + j) * stride + (size_t)g * hd) * 2;
    }
}

__device__ __forceinline__ void store_elem(void *p, uint32_t dtype, size_t i, float v) {
    if (dtype == FELLM_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == FELLM_DTYPE_F16) static_cast<_Float16 *>(p)[i] = F16::store(v);
    else static_cast<uint16_t *>(p)[i] = BF16::store(v);
}

// One row over the keys [k0, k1), by one wavefront: only attended keys count,
// whatever the others hold.  A lane scores a key, then owns dims lane + 64 e.
// Unnormalised sums in acc, m, l, all times 2^bias as the tiles' are; the row has
// an attended key here.  The loads
// of several keys are on their way together: a batch whose values all are NaN
// takes this path everywhere.
template <typename E, int HD, bool PAGED>
__device__ void careful_row(const Args &a, const Tile &t, uint32_t g, uint32_t token, uint32_t head, uint32_t k0,
                            uint32_t k1, float bias, float (&acc)[HD / 64], float &m, float &l) {
    using T = typename E::A::T;
    const uint32_t lane = threadIdx.x % kWave;
    const KeyRange r = row_keys(a, t, token);
    const size_t q0 = (size_t)(t.first + token) * a.q_stride + (size_t)head * HD;
    auto score = [&](uint32_t j) -> float {
        const T *kp = reinterpret_cast<const T *>(key_ptr<PAGED>(a, t, g, HD, j, false));
        float s = 0.0f;
#pragma unroll 4
        for (int d = 0; d < HD; d += 8) {
            float k8[8], q8[8];
            if (kp) {
                load_f32<typename E::A, 8>(kp + d, k8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) k8[e] = 0.0f;
            }
            if (a.q_dtype == FELLM_DTYPE_F32) load_f32<F32, 8>(static_cast<const float *>(a.q) + q0 + d, q8);
            else if (a.q_dtype == FELLM_DTYPE_F16) load_f32<F16, 8>(static_cast<const _Float16 *>(a.q) + q0 + d, q8);
            else load_f32<BF16, 8>(static_cast<const uint16_t *>(a.q) + q0 + d, q8);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(q8[e], k8[e], s);
        }
        return s;
    };
    auto attended = [&](uint32_t kb) -> uint64_t {
        const uint64_t bits = key_bits(a, t, token, r, kb);
        return kb + 64 > k1 ? bits & ((1ull << (k1 - kb)) - 1) : bits;
    };
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) acc[e] = 0.0f;
#pragma unroll 1
    for (uint32_t kb = k0; kb < k1; kb += 64) {
        const uint64_t bits = attended(kb);
        if (bits >> lane & 1) {
            const float s = score(kb + lane);
            m = s > m || s != s ? s : m;
        }
    }
    float top = m;
    const bool nan = m != m;
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    // scores that all are -inf: the lowest finite maximum keeps p = 0 and l = 0, so
    // that the row is 0 / 0 alone and nothing next to other shares of its keys
    m = __any(nan) ? __builtin_nanf("") : fmaxf(top, -3.402823466e38f);
#pragma unroll 1
    for (uint32_t kb = k0; kb < k1; kb += 64) {
        const uint64_t bits = attended(kb);
        if (!bits) continue;
        const float p = bits >> lane & 1 ? __builtin_amdgcn_exp2f((score(kb + lane) - m) * a.c + bias) : 0.0f;
        l += p;
#pragma unroll 1
        for (uint32_t b0 = 0; b0 < 64 && kb + b0 < k1; b0 += 8) {
            float v[8][HD / 64];
#pragma unroll
            for (uint32_t b = 0; b < 8; ++b) {
                const T *vp = reinterpret_cast<const T *>(key_ptr<PAGED>(a, t, g, HD, min(kb + b0 + b, k1 - 1), true));
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) v[b][e] = vp ? E::A::load(vp[lane + 64 * e]) : 0.0f;
            }
#pragma unroll
            for (uint32_t b = 0; b < 8; ++b) {
                if (!(bits >> (b0 + b) & 1)) continue;
                const float pb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), b0 + b));
#pragma unroll
                for (int e = 0; e < HD / 64; ++e) acc[e] = fmaf(pb, v[b][e], acc[e]);
            }
        }
    }
    l = wave_sum(l);
}

// The bijection of a key's low four (HD 64: bits 1 to 3) bits that its 16-byte
// pieces are permuted by.
template <int HD>
__device__ __forceinline__ uint32_t swizzle(uint32_t key) {
    if constexpr (HD == 64) return (key >> 1 & 1) << 2 | (key >> 2 & 1) << 1 | (key >> 3 & 1);
    return (key & 3) << 2 | (key >> 2 & 1) << 1 | (key >> 3 & 1);
}

__device__ __forceinline__ float halves_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// 32 dims of a row, lane h with dims 8 i + 4 h + e in v[4 i + e], as 16-bit
// numbers: the row's two lanes exchange 4-dim pieces and store 8 dims each.
template <typename O>
__device__ __forceinline__ void store_tile(typename O::T *to, const f32x16 &v, uint32_t h) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        using H = typename HwStore<O>::type;
        const typename O::T pair[2] = {H::store(v[2 * i]), H::store(v[2 * i + 1])};
        memcpy(&w[i], pair, 4);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const auto a = __builtin_amdgcn_permlane32_swap(w[4 * j], w[4 * j + 2], false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(w[4 * j + 1], w[4 * j + 3], false, false);
        *reinterpret_cast<u32x4 *>(to + 16 * j + 8 * h) = u32x4{a[0], b[0], a[1], b[1]};
    }
}

// A split's partial record of one row: HD unnormalised sums, m, l, two unused.
template <int HD>
constexpr uint32_t kRec = HD + 4;

// Keys of a tile of rows: [begin, end), begin a multiple of 64.
struct Keys {
    uint32_t begin, end;
};
template <uint32_t BM>
__device__ __forceinline__ Keys tile_keys(const Args &a, const Tile &t) {
    const uint32_t i0 = a.by_group(t.row0), i1 = min(t.n, a.by_group(t.row0 + BM - 1) + 1);
    return Keys{row_keys(a, t, i0).lo / 64 * 64, row_keys(a, t, i1 - 1).hi};
}

// Inclusive sum over the wavefront's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);  // row_shr:1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    const uint32_t a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31),
                   c = b + __builtin_amdgcn_readlane(v, 47), row = threadIdx.x % kWave / 16;
    return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

// How a paged launch shares its work.  The rounds of TK keys of every tile, tiles
// in the order of the sequences, are one line for each K/V head, which the head's
// `ids` workgroups cut into pieces, so that sequences of any lengths keep every
// workgroup busy and all of them are resident at once.
//  * Where there are workgroups enough a piece is a part of one tile: `per` rounds.
//  * Else the line is cut into equal shares, and a workgroup walks the tiles that
//    its share touches, of which the first and the last can be shared with others:
//    two records.  (Measured against tiles cut at fixed numbers of keys: 32 trees
//    of up to 32 tokens behind 616 .. 8192 keys, 64/8 heads of 128, bf16, 124 and
//    118 us; 16 drafted tokens behind 32768 keys, 16/4 heads of 256, 125 and 58.)
//  * EVEN, for launches of many tiles: every tile begins with
//    kStart units without keys, what its start costs in rounds, and the tiles of a
//    causal chunk have rounds that rise with their place in the sequence, tile k
//    the first one's and k BM / (G TK) more, rounded so that the first k tiles have
//    floor(k (k - 1) / 2 BM / (G TK)) more than k times the first; the last piece
//    of a tile takes what is left of its keys.  Shares of it are used where a piece
//    would be kJoin rounds longer, which is what joining every tile costs.  (8192
//    tokens behind 8192, 64/8 heads of 128: 4610 -> 3940 us; the 32 trees 118 ->
//    113.  Its arithmetic costs a launch of few rounds 0.7 of 12 us.)
// Lane b holds sequence c + b.
template <uint32_t BM, uint32_t TK, bool EVEN>
struct Line {
    static constexpr uint32_t kStart = 5, kJoin = 24;
    const Args &a;
    struct Lane {
        uint32_t first, n, before, tiles;
    } l0;
    uint32_t per = 1;       // rounds of a unit of the line
    uint32_t share, units;  // units of a workgroup, of the line
    uint32_t start = 0;     // units without keys that a tile begins with
    bool rising = false;

    __device__ __forceinline__ Line(const Args &args, uint32_t ids) : a(args), l0(lane(0)) {
        units = total();
        share = (units + ids - 1) / ids;
        if (!a.part) return;
        const uint32_t least = max(share, a.min_rounds);
        per = least;
        units = total();
        if (units > ids) {
            // two rounds more than an equal share cost less than a second tile's start
            per = least + 2;
            units = total();
        }
        const bool apart = units <= ids;
        if constexpr (!EVEN) {
            if (apart) {
                share = 1;
            } else {
                per = 1;
                units = total();
                share = least;
            }
            return;
        }
        const uint32_t parts = units, was = per;
        rising = !a.mask && !a.window;
        // (rising rounds are at least half of all)
        if (!apart || (rising && least / 2 + kJoin < per + kStart)) {
            per = 1;
            start = kStart;
            units = total();
            share = max((units + ids - 1) / ids, a.min_rounds);
            if (!apart || share + kJoin < was + kStart) return;
        }
        rising = false;
        per = was;
        start = 0;
        units = parts;
        share = 1;
    }
    __device__ __forceinline__ Lane lane(uint32_t c) const {
        const uint32_t b = c + threadIdx.x % kWave;
        Lane l{0, 0, 0, 0};
        if (b < a.n_seqs) {
            l.first = min(a.cu[b], a.tokens);
            const uint32_t end = min(a.cu[b + 1], a.tokens);
            l.n = end > l.first ? end - l.first : 0;
            l.before = min(a.before[b], a.max_before);
        }
        l.tiles = (l.n * a.group + BM - 1) / BM;
        return l;
    }
    // Units of the sequence's first tile.
    __device__ __forceinline__ uint32_t first_units(const Lane &l) const {
        if (!a.part || !l.n) return 1;
        uint32_t keys = l.before + (rising ? min(l.n, a.by_group(BM - 1) + 1) : l.n);
        // the last keys of the tile's first token, its other tokens, the alignment
        if (a.window) keys = min(keys, min(a.window, 1u << 30) + BM + 63);
        const uint32_t rounds = (keys + TK - 1) / TK;
        return per == 1 ? rounds + start : (rounds + per - 1) / per;
    }
    // Units of a sequence's first k tiles, u those of the first.
    __device__ __forceinline__ uint32_t upto(uint32_t u, uint32_t k) const {
        if (!EVEN || !rising) return k * u;
        const uint32_t pairs = k ? k * (k - 1) / 2 : 0;
        return k * u + a.by_group(BM >= TK ? pairs * (BM / TK) : pairs / (TK / BM));
    }
    __device__ __forceinline__ uint32_t total() const {
        const uint32_t here = upto(first_units(l0), l0.tiles);
        if (a.n_seqs == 1) return __builtin_amdgcn_readfirstlane(here);
        uint32_t sum = wave_total(here);
        for (uint32_t c = kWave; c < a.n_seqs; c += kWave) {
            const Lane l = lane(c);
            sum += wave_total(upto(first_units(l), l.tiles));
        }
        return sum;
    }
    // The tile, of `tiles`, that holds unit y of its sequence.
    __device__ __forceinline__ uint32_t tile_at(uint32_t u, uint32_t tiles, uint32_t y) const {
        if (!EVEN || !rising) return y / u;
        // k u + k^2 / 2 step = y to within a tile or two, then exactly
        const float step = (float)BM / (float)(a.group * TK), b = (float)u - 0.5f * step;
        const float root = __builtin_amdgcn_sqrtf(fmaf(b, b, 2.0f * step * (float)y));
        uint32_t k = min(tiles - 1, (uint32_t)fmaxf((root - b) / step, 0.0f));
        k = __builtin_amdgcn_readfirstlane(k);
        while (k && upto(u, k) > y) --k;
        while (k + 1 < tiles && upto(u, k + 1) <= y) ++k;
        return k;
    }
    struct Spot {
        Tile t;
        uint32_t units, at;  // of the tile, and where it begins on the line
    };
    // BY_TILE: tile number x; else the tile that holds unit x.  n = 0: none.
    template <bool BY_TILE>
    __device__ __forceinline__ Spot find(uint32_t x) const {
        Spot s{Tile{0, 0, 0, 0, 0}, 1, 0};
        uint32_t tiles = 0, at = 0;
        for (uint32_t c = 0; c < a.n_seqs; c += kWave) {
            const Lane l = c ? lane(c) : l0;
            const uint32_t u0 = first_units(l), v = upto(u0, l.tiles);
            const bool one = a.n_seqs == 1;
            const uint32_t vi = one ? v : wave_scan(v), ti = !BY_TILE ? 0 : one ? l.tiles : wave_scan(l.tiles);
            const uint64_t past = __ballot((BY_TILE ? tiles + ti : at + vi) > x);
            if (past) {
                const uint32_t b = (uint32_t)__builtin_ctzll(past);
                auto of = [&](uint32_t value) { return (uint32_t)__builtin_amdgcn_readlane(value, b); };
                const uint32_t begin = at + of(vi - v), u = of(u0);
                const uint32_t k = BY_TILE ? x - (tiles + of(ti - l.tiles)) : tile_at(u, of(l.tiles), x - begin);
                s.t = Tile{c + b, k * BM, of(l.first), of(l.n), of(l.before)};
                s.at = begin + upto(u, k);
                s.units = upto(u, k + 1) - upto(u, k);
                return s;
            }
            if (BY_TILE) tiles += __builtin_amdgcn_readlane(ti, kWave - 1);
            at += __builtin_amdgcn_readlane(vi, kWave - 1);
        }
        return s;
    }
};

// A buffer resource in scalar registers: everything it is made of is the same in
// all lanes, but where the compiler does not see that it would loop over lanes
// for every load (a chunk of 512 tokens behind 32256 keys: 340 us).
__device__ __forceinline__ Rsrc uniform_rsrc(const uint8_t *p, uint32_t range) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint64_t u = (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 |
                       (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, (int)__builtin_amdgcn_readfirstlane(range),
                                             0x00020000);
}

// E: K/V policy, HD: head dim, RW: wavefronts that own 32 rows each, KW:
// wavefronts that share those rows and take every KW-th key tile, KT: keys of
// a wavefront's tile (32 or 64), PARTS: q and p held to f32 accuracy in several
// 16-bit parts (q or out in f32, or q of another 16-bit type than K/V).
// OCC: wavefronts per SIMD the registers are kept for.  EVEN: see Line.  (Three tiles in LDS
// instead of two, two of them on their way, measured the same within 1%.)
template <typename E, int HD, int RW, int KW, int KT, bool PAGED, bool PARTS, int OCC, bool EVEN = false>
__global__ __launch_bounds__(kWave *RW *KW, OCC) void rows_kernel(Args a) {
    constexpr int NW = RW * KW, NS = HD / 16, NU = KT / 32, ND = HD / 32;
    constexpr int QP = PARTS ? E::kQParts : 1, PP = PARTS ? E::kPParts : 1;
    constexpr uint32_t BM = kRows * RW, TK = KT * KW, SK = TK / NW;  // keys a wavefront stages per round
    constexpr uint32_t CH = HD / 8, RB = HD * 2;                      // 16-byte pieces, bytes of a key row
    constexpr uint32_t KPI = kWave / CH;                              // keys per load instruction
    constexpr float kBias = PARTS ? E::kBiasParts : E::kBias;
    constexpr float kLazy = PARTS ? 0.0f : 8.0f;
    static_assert(SK % KPI == 0 && (SK <= kBlockTokens || SK % kBlockTokens == 0) && 64 % SK == 0);
    using T = typename E::A::T;

    // Separate arrays: the compiler then knows that a read of one need not wait
    // for loads to another.
    __shared__ __align__(16) uint8_t k_lds0[TK * RB], v_lds0[TK * RB], k_lds1[TK * RB], v_lds1[TK * RB];

    const uint32_t lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t rw = wave % RW, kw = wave / RW;
    const uint32_t n = lane % 32, h = lane / 32;
    // Neighbouring workgroups take the K/V heads in turn (one XCD sees few of them).
    const uint32_t g = blockIdx.x % a.n_kv, id = blockIdx.x / a.n_kv, ids = gridDim.x / a.n_kv;
    // this workgroup's piece [x, x_end) of the line (contiguous K/V: its one tile)
    const auto line = [&] {
        if constexpr (PAGED) return Line<BM, TK, EVEN>(a, ids);
        else return 0;
    }();
    uint32_t x = 0, x_end = 1;
    if constexpr (PAGED) {
        if ((uint64_t)id * line.share >= line.units) return;
        x = id * line.share;
        x_end = min(line.units, x + line.share);
    }
    for (uint32_t again = 0; x < x_end; again = 1) {
        Tile t;
        Keys sh;
        bool direct = true;
        float *part = nullptr;  // the tile's records where others share it
        if constexpr (PAGED) {
            const auto spot = line.template find<false>(x);
            t = spot.t;
            if (t.n == 0) break;  // offsets that are none: nothing more to find
            sh = tile_keys<BM>(a, t);
            const uint32_t u0 = x - spot.at, u1 = min(spot.units, u0 + x_end - x);
            x += u1 - u0;
            if (u1 <= line.start) break;  // the share ends before the tile's keys
            direct = u0 <= line.start && u1 == spot.units;
            if (!direct) {
                part = a.part + (size_t)(2 * (g * ids + id) + again) * BM * kRec<HD>;
                const uint32_t lo = sh.begin;
                if (u0 > line.start) sh.begin = lo + (u0 - line.start) * line.per * TK;
                if (u1 < spot.units) sh.end = min(sh.end, lo + (u1 - line.start) * line.per * TK);
            }
            if (again) __syncthreads();  // the buffers may still be read for the tile before
        } else {
            t = tile_of<BM>(a, id, ids);
            if (t.n == 0) return;
            sh = tile_keys<BM>(a, t);
            ++x;
        }

        const uint32_t row = t.row0 + rw * kRows + n;
        const bool valid = row < t.n * a.group;
        const uint32_t rrow = valid ? row : t.n * a.group - 1;
        const uint32_t token = a.by_group(rrow), head = g * a.group + rrow - token * a.group;
        const KeyRange mine = row_keys(a, t, token);
        // keys that every row of this wavefront attends, and that any does
        const uint32_t w0 = min(t.row0 + rw * kRows, t.n * a.group - 1), w1 = min(w0 + kRows - 1, t.n * a.group - 1);
        const KeyRange rf = row_keys(a, t, a.by_group(w0)), rl = row_keys(a, t, a.by_group(w1));
        const uint32_t full_lo = rl.lo, full_hi = a.mask ? t.before : rf.hi, any_lo = rf.lo, any_hi = rl.hi;

        f32x16 acc[ND];
        float m = -__builtin_inff(), l = 0.0f;
        bool some = false;  // the row attends a key of this share
    #pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = f32x16(0.0f);

        // ---- staging: SK keys from kb + wave SK on
        const uint32_t skey = lane / CH, spos = lane % CH;
        constexpr uint32_t BK = SK < kBlockTokens ? SK : kBlockTokens;  // keys of a piece, of one cache block
        // Table entries of the pieces of the tile that is requested next (paged): read
        // a tile ahead, so that their latency does not stand before the request.
        uint32_t entry[SK / BK];
        auto look_up = [&](uint32_t kb) __attribute__((always_inline)) {
            if constexpr (PAGED) {
    #pragma unroll
                for (uint32_t b = 0; b < SK / BK; ++b) {
                    // through a vector load: a scalar one on its way would turn every
                    // wait for an LDS read into a wait for all of them
                    uint32_t blk = (kb + wave * SK + b * BK) / kBlockTokens;
                    __asm__("" : "+v"(blk));
                    entry[b] = block_entry(a, t, blk);
                }
            }
        };
        auto stage = [&](uint32_t kb, uint8_t *lds, bool is_v) __attribute__((always_inline)) {
    #pragma unroll
            for (uint32_t b0 = 0; b0 < SK; b0 += BK) {
                const uint32_t j = kb + wave * SK + b0;
                const uint32_t have = j < sh.end ? min(BK, sh.end - j) : 0;
                const uint32_t stride = (PAGED ? a.stride : is_v ? a.v_stride : a.k_stride) * 2;
                const uint8_t *src;
                if constexpr (PAGED) {
                    const uint8_t *at = block_ptr(a, __builtin_amdgcn_readfirstlane(entry[b0 / BK]));
                    src = at ? at + (j % kBlockTokens + (is_v ? kBlockTokens : 0)) * stride + g * RB : nullptr;
                } else {
                    src = key_ptr<PAGED>(a, t, g, HD, j, is_v);
                }
                const Rsrc rs = uniform_rsrc(src, src && have ? (have - 1) * stride + RB : 0);
    #pragma unroll
                for (uint32_t i = 0; i < BK / KPI; ++i) {
                    const uint32_t key = i * KPI + skey;  // inside the piece of BK keys
                    const uint32_t c = (spos ^ swizzle<HD>(wave * SK + b0 + key)) * 16;
                    using L = __attribute__((address_space(3))) void;
                    const uint32_t at = (wave * SK + b0 + i * KPI) * RB;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (L *)(lds + at), 16, key * stride + c, 0, 0, 0);
                }
            }
        };
        auto request = [&](uint32_t kb, uint8_t *kl, uint8_t *vl) __attribute__((always_inline)) {
            if (kb >= sh.end) return;
            stage(kb, kl, false);
            stage(kb, vl, true);
            look_up(kb + TK);
        };

        look_up(sh.begin);
        request(sh.begin, k_lds0, v_lds0);

        // Q^T as the B operand: row n, dims 16 st + 8 h .. +7
        u32x4 qf[NS][QP];
        {
            const size_t q0 = (size_t)(t.first + token) * a.q_stride + (size_t)head * HD + 8 * h;
            if constexpr (!PARTS) {
                const T *qp = static_cast<const T *>(a.q) + q0;
    #pragma unroll
                for (int s = 0; s < NS; ++s) qf[s][0] = *reinterpret_cast<const u32x4 *>(qp + 16 * s);
            } else {
    #pragma unroll
                for (int s = 0; s < NS; ++s) {
                    float x[8];
                    if (a.q_dtype == FELLM_DTYPE_F32) load_f32<F32, 8>(static_cast<const float *>(a.q) + q0 + 16 * s, x);
                    else if (a.q_dtype == FELLM_DTYPE_F16) load_f32<F16, 8>(static_cast<const _Float16 *>(a.q) + q0 + 16 * s, x);
                    else load_f32<BF16, 8>(static_cast<const uint16_t *>(a.q) + q0 + 16 * s, x);
    #pragma unroll
                    for (int p = 0; p < QP; ++p)
    #pragma unroll
                        for (int w = 0; w < 4; ++w) qf[s][p][w] = E::part(x[2 * w], x[2 * w + 1]);
                }
            }
        }

        // ---- a tile of KT keys from kb on, in three parts
        f32x16 s[NU];          // scores of row n
        u32x4 pf[KT / 16][PP]; // probabilities, as the second product takes them
        const uint32_t kbase = kw * KT * RB + n * RB, ksw = (h ^ swizzle<HD>(n)) * 16;
        auto scores = [&](const uint8_t *kl) __attribute__((always_inline)) {
            // Piece x: dims 16 (x / NU) .. of keys 32 (x % NU) ...  Each is read kAhead
            // products early and the order is fixed: left to itself the compiler reads
            // a piece right before its product and waits for the LDS every time (one
            // prompt of 16384 tokens, 32/4 heads of 128, bf16: 2114 -> 1939 us).
            constexpr int N = NS * NU, kAhead = 4;
            auto piece = [&](int x) {
                return *reinterpret_cast<const u32x4 *>(kl + kbase + x % NU * 32 * RB + (ksw ^ (x / NU * 32)));
            };
            u32x4 kf[kAhead];
    #pragma unroll
            for (int x = 0; x < kAhead; ++x) kf[x] = piece(x);
    #pragma unroll
            for (int u = 0; u < NU; ++u) s[u] = f32x16(0.0f);
    #pragma unroll
            for (int x = 0; x < N; ++x) {
                __builtin_amdgcn_sched_barrier(0);
    #pragma unroll
                for (int p = 0; p < QP; ++p) s[x % NU] = E::mfma(kf[x % kAhead], qf[x / NU][p], s[x % NU]);
                if (x + kAhead < N) kf[x % kAhead] = piece(x + kAhead);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto weights = [&](uint32_t kb) __attribute__((always_inline)) {
            if (!(kb >= full_lo && kb + KT <= full_hi && kb + KT <= sh.end)) {
                uint64_t bits = key_bits(a, t, token, mine, kb);
                if (kb + 64 > sh.end) bits &= (1ull << (sh.end - kb)) - 1;
                some |= (KT == 64 ? bits : (uint32_t)bits) != 0;
                bits >>= 4 * h;
    #pragma unroll
                for (int u = 0; u < NU; ++u)
    #pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(bits >> (32 * u + 8 * (i / 4) + i % 4) & 1)) s[u][i] = -__builtin_inff();
            } else {
                some = true;
            }
            float top = s[0][0];
    #pragma unroll
            for (int u = 0; u < NU; ++u)
    #pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
            top = halves_max(top);
            if (__any((top - m) * a.c > kLazy)) {
                const float mn = fmaxf(m, top);
                const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * a.c);
                m = mn;
                l *= f;
    #pragma unroll
                for (int d = 0; d < ND; ++d)
    #pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= f;
            }
            const float base = (m == -__builtin_inff() ? 0.0f : -m * a.c) + kBias;
            float sum = 0.0f;
    #pragma unroll
            for (int k = 0; k < KT / 16; ++k) {
                float x[8];
    #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(fmaf(s[k / 2][8 * (k % 2) + e], a.c, base));
                    sum += x[e];
                }
    #pragma unroll
                for (int p = 0; p < PP; ++p)
    #pragma unroll
                    for (int w = 0; w < 4; ++w) pf[k][p][w] = E::part(x[2 * w], x[2 * w + 1]);
            }
            l += sum;
        };
        // V^T pieces: lane group of 16 reads keys 4 h + .. of dims 16 (group % 2) ..
        const uint32_t vkey = 4 * h + lane % 16 / 4, vpc = lane / 16 % 2 * 2 + lane % 4 / 2;
        const uint32_t vbase = kw * KT * RB + vkey * RB + lane % 2 * 8;
        const uint32_t vsw0 = (vpc ^ swizzle<HD>(vkey)) * 16, vsw1 = (vpc ^ swizzle<HD>(vkey + 8)) * 16;
        auto products = [&](const uint8_t *vl) __attribute__((always_inline)) {
            using L4 = __attribute__((address_space(3))) s16x4;
    #pragma unroll
            for (int k = 0; k < KT / 16; ++k)
    #pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const uint32_t off = k * 16 * RB + vbase;
                    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4 *)(vl + off + (vsw0 ^ (d * 64))));
                    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L4 *)(vl + off + 8 * RB + (vsw1 ^ (d * 64))));
                    const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
                    const u32x4 vf = {lo2[0], lo2[1], hi2[0], hi2[1]};
    #pragma unroll
                    for (int p = 0; p < PP; ++p) acc[d] = E::mfma(vf, pf[k][p], acc[d]);
                }
        };
        const uint32_t hi_here = t.row0 + rw * kRows < t.n * a.group ? min(sh.end, any_hi) : 0;  // 0: no row of its own
        auto mine_at = [&](uint32_t kb) { return kb < hi_here && kb + KT > any_lo; };

        // The tile's loads to LDS are done, then everyone's.  The wait is written out:
        // a barrier alone does not imply it, and the one the compiler puts before the
        // reads cannot know of other wavefronts' loads.
        auto arrived = [&]() __attribute__((always_inline)) {
            __asm__ volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
            __asm__ volatile("" ::: "memory");
            __syncthreads();
        };
        // kn and vn: the buffers of the tile before, which no wavefront reads any more after the barrier
        auto round = [&](uint32_t kb, const uint8_t *kl, const uint8_t *vl, uint8_t *kn, uint8_t *vn)
                         __attribute__((always_inline)) {
            if (kb >= sh.end) return;
            arrived();
            request(kb + TK, kn, vn);
            const uint32_t my = kb + kw * KT;
            if (mine_at(my)) {
                scores(kl);
                weights(my);
                products(vl);
            }
        };
        for (uint32_t kb = sh.begin; kb < sh.end; kb += 2 * TK) {
            round(kb, k_lds0, v_lds0, k_lds1, v_lds1);
            round(kb + TK, k_lds1, v_lds1, k_lds0, v_lds0);
        }
        l = halves_sum(l);

        float probe = 0.0f;  // NaN if any sum is not finite
    #pragma unroll
        for (int d = 0; d < ND; ++d)
    #pragma unroll
            for (int i = 0; i < 16; ++i) probe = fmaf(acc[d][i], 0.0f, probe);
        probe = halves_sum(probe) + l * 0.0f;

        // ---- wavefronts that share rows: every one leaves its sums in LDS and
        // joins (and stores) the tiles d = kw, kw + KW, .. of all of them
        if constexpr (KW > 1) {
            static_assert(16 * RW <= KT, "the sums of all wavefronts fit the four buffers");
            __shared__ float state_lds[NW][4][kWave];
            auto sum_at = [&](uint32_t w, int x) -> float & {  // x-th of a lane's 16 ND sums
                uint8_t *buf = x < 4 * ND ? k_lds0 : x < 8 * ND ? v_lds0 : x < 12 * ND ? k_lds1 : v_lds1;
                return reinterpret_cast<float *>(buf)[(w * 4 * ND + x % (4 * ND)) * kWave + lane];
            };
            __syncthreads();
    #pragma unroll
            for (int d = 0; d < ND; ++d)
    #pragma unroll
                for (int i = 0; i < 16; ++i) sum_at(wave, d * 16 + i) = acc[d][i];
            state_lds[wave][0][lane] = m;
            state_lds[wave][1][lane] = l;
            state_lds[wave][2][lane] = probe;
            state_lds[wave][3][lane] = some ? 1.0f : 0.0f;
            __syncthreads();
            float f[KW];
            m = -__builtin_inff();
    #pragma unroll
            for (int w = 0; w < KW; ++w) m = fmaxf(m, state_lds[rw + w * RW][0][lane]);
            l = probe = 0.0f;
    #pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float mw = state_lds[rw + w * RW][0][lane];
                f[w] = mw == m ? 1.0f : __builtin_amdgcn_exp2f((mw - m) * a.c);
                l = fmaf(state_lds[rw + w * RW][1][lane], f[w], l);
                probe += state_lds[rw + w * RW][2][lane];
                some |= state_lds[rw + w * RW][3][lane] != 0.0f;
            }
    #pragma unroll
            for (int d = 0; d < ND; ++d) {
                if (d % KW != (int)kw) continue;
    #pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float v = 0.0f;
    #pragma unroll
                    for (int w = 0; w < KW; ++w) v = fmaf(sum_at(rw + w * RW, d * 16 + i), f[w], v);
                    acc[d][i] = v;
                }
            }
        }

        // ---- results
        const bool bad = valid && some && !(probe == 0.0f && l > 0.0f);
        // exchanges between a row's two lanes follow: both take part or neither, as
        // valid and bad are the row's
        if (valid && !bad) {
            const float inv = !direct ? 1.0f : some ? 1.0f / l : 0.0f;
            const size_t o0 = (size_t)(t.first + token) * a.out_stride + (size_t)head * HD;
            float *rec = part + (size_t)(rw * kRows + n) * kRec<HD>;
    #pragma unroll
            for (int d = 0; d < ND; ++d) {
                if (KW > 1 && d % KW != (int)kw) continue;
    #pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= inv;
                if (!direct || (PARTS && a.out_dtype == FELLM_DTYPE_F32)) {
                    float *to = direct ? static_cast<float *>(a.out) + o0 : rec;
    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v[4] = {acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
                        store_f32<F32, 4>(to + 32 * d + 8 * i + 4 * h, v);
                    }
                } else if constexpr (!PARTS) {
                    store_tile<typename E::A>(static_cast<T *>(a.out) + o0 + 32 * d, acc[d], h);
                } else if (a.out_dtype == FELLM_DTYPE_F16) {
                    store_tile<F16>(static_cast<_Float16 *>(a.out) + o0 + 32 * d, acc[d], h);
                } else {
                    store_tile<BF16>(static_cast<uint16_t *>(a.out) + o0 + 32 * d, acc[d], h);
                }
            }
            if (!direct && h == 0 && kw == 0) {
                rec[HD] = m;
                rec[HD + 1] = l;
            }
        }
        uint64_t redo = kw ? 0 : __ballot(bad) & 0xffffffffull;
        while (redo) {
            const uint32_t r = (uint32_t)__builtin_ctzll(redo);
            redo &= redo - 1;
            const uint32_t pr = t.row0 + rw * kRows + r, tk = a.by_group(pr), hd = g * a.group + pr - tk * a.group;
            float sums[HD / 64], m1, l1;
            careful_row<E, HD, PAGED>(a, t, g, tk, hd, sh.begin, sh.end, kBias, sums, m1, l1);
            float *rec = part + (size_t)(rw * kRows + r) * kRec<HD>;
    #pragma unroll
            for (int e = 0; e < HD / 64; ++e) {
                if (direct)
                    store_elem(a.out, a.out_dtype, (size_t)(t.first + tk) * a.out_stride + (size_t)hd * HD + lane + 64 * e,
                               sums[e] / l1);
                else rec[lane + 64 * e] = sums[e];
            }
            if (!direct && lane == 0) {
                rec[HD] = m1;
                rec[HD + 1] = l1;
            }
        }
    }
}

// Joins the records of tiles that several workgroups shared: 16 lanes a row read
// one record, Q groups of 16 lanes every Q-th.  ids: the workgroups per K/V head
// of the launch before.
constexpr uint32_t kJoinThreads = 256;
template <int HD, uint32_t BM, uint32_t TK, int Q, bool EVEN>
__global__ __launch_bounds__(kJoinThreads) void rows_combine(Args a, uint32_t ids) {
    constexpr uint32_t ROWS = kJoinThreads / 16 / Q;  // of a workgroup
    const uint32_t id = blockIdx.x / (BM / ROWS), g = id % a.n_kv;
    const uint32_t r = blockIdx.x % (BM / ROWS) * ROWS + threadIdx.x / (16 * Q);
    const uint32_t col = threadIdx.x % 16, part = threadIdx.x / 16 % Q;
    const Line<BM, TK, EVEN> line(a, ids);
    const auto spot = line.template find<true>(id / a.n_kv);
    const Tile t = spot.t;
    if (t.n == 0 || spot.units == 1 || t.row0 + r >= t.n * a.group) return;
    // (offsets that are no offsets could name workgroups that there are none of)
    const uint32_t w0 = (spot.at + line.start) / line.share, w1 = min((spot.at + spot.units - 1) / line.share, ids - 1);
    if (w0 >= w1) return;
    // Workgroup w's first record if its piece begins inside the tile or with it, else its second.
    auto record = [&](uint32_t w) {
        const uint32_t slot = 2 * (g * ids + w) + (w * line.share >= spot.at ? 0 : 1);
        return a.part + ((size_t)slot * BM + r) * kRec<HD>;
    };
    float top = -__builtin_inff();
    for (uint32_t w = w0 + col + 16 * part; w <= w1; w += 16 * Q) top = fmaxf(top, record(w)[HD]);
#pragma unroll
    for (int off = 8 * Q; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    constexpr int PD = HD / 64;  // four dims from 4 (col + 16 e) on
    float acc[PD][4] = {}, l = 0.0f;
#pragma unroll 4
    for (uint32_t w = w0 + part; w <= w1; w += Q) {
        const float *rz = record(w);
        const float mz = rz[HD], lz = rz[HD + 1];
        const float f = mz == top ? 1.0f : __builtin_amdgcn_exp2f((mz - top) * a.c);
        l = fmaf(lz, f, l);
#pragma unroll
        for (int e = 0; e < PD; ++e) {
            float v[4];
            load_f32<F32, 4>(rz + 4 * (col + 16 * e), v);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[e][i] = fmaf(v[i], f, acc[e][i]);
        }
    }
#pragma unroll
    for (int off = 16; off < 16 * Q; off <<= 1) {
        l += __shfl_xor(l, off);
#pragma unroll
        for (int e = 0; e < PD; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[e][i] += __shfl_xor(acc[e][i], off);
    }
    if (part) return;
    const uint32_t pr = t.row0 + r, tk = a.by_group(pr), hd = g * a.group + pr - tk * a.group;
    const float inv = 1.0f / l;
    const bool none = top == -__builtin_inff() && l == 0.0f;  // no attended key
    const size_t o0 = (size_t)(t.first + tk) * a.out_stride + (size_t)hd * HD;
#pragma unroll
    for (int e = 0; e < PD; ++e) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[e][i] = none ? 0.0f : acc[e][i] * inv;
        const size_t o = o0 + 4 * (col + 16 * e);
        if (a.out_dtype == FELLM_DTYPE_F32) store_f32<F32, 4>(static_cast<float *>(a.out) + o, acc[e]);
        else if (a.out_dtype == FELLM_DTYPE_F16) store_f32<F16, 4>(static_cast<_Float16 *>(a.out) + o, acc[e]);
        else store_f32<BF16, 4>(static_cast<uint16_t *>(a.out) + o, acc[e]);
    }
}

}  // namespace rows_attn
}  // namespace fellm
