// Attention of packed whole prompts: causal self-attention of the tokens of
// each sequence, grouped heads, contiguous 16-bit q, k and v.  The kernel is
// rows_kernel of attention_rows.hpp.
#include "attention_rows.hpp"

namespace fellm {
namespace {
using namespace rows_attn;

template <typename E, int HD, int RW, int KW, int KT, int OCC>
int launch_prompt(Args a, hipStream_t st) {
    constexpr uint32_t BM = kRows * RW;
    const uint64_t rows = (uint64_t)a.tokens * a.group, tiles = a.n_seqs == 1 ? (rows + BM - 1) / BM : rows / BM + a.n_seqs;
    if (tiles * a.n_kv > 0xffffffffull / (kWave * RW * KW)) return FELLM_ERR_SHAPE;
    FELLM_LAUNCH((rows_kernel<E, HD, RW, KW, KT, false, false, OCC>), dim3((uint32_t)tiles * a.n_kv),
                 dim3(kWave * RW * KW), 0, st, a);
    return launch_status();
}

// Layouts (wavefronts that own rows, wavefronts that share them, keys of a
// tile, wavefronts per SIMD) by the tiles of 128 rows that the launch could
// have, w.  Few tiles: 64 rows a workgroup, two wavefronts on alternate keys,
// which halves the longest walk.  Measured in us, the layouts compared in the
// order of the lines below:
//  64:  one prompt of 1024 tokens (32/8 heads, w 256) 15.4, 22.0; of 2048 (512)
//       31.2, 40.3; of 4096 (1024) 91.9, 88.8; 16 of 256 (1024) 23.3, 17.4
//  128: one prompt of 512 tokens (32/8 heads, w 128) 13.4, 16.9, 20.8, 20.9; of
//       2048 (512) 55.4, 52.2, 65.4, 62.2; of 4096 (1024) 165, 151, 153, 142; 17
//       of 128 .. 2048 (28/4, 2707) 194, 144, 134, 151; one of 16384 (32/4) 2357,
//       2010, 2007, 1999
//  256: one prompt of 1024 tokens (16/4 heads, w 128) 43, 63; of 2048 (256) 88,
//       112; of 4096 (512) 290, 219; of 16384 (2048) 4073, 1941
// Whole prompts of 16384 rows and more on average keep eight wavefronts busy on
// the same keys; shorter ones gain more from a third workgroup on a CU, which
// covers the others' starts and ends.
template <typename E>
int prompt_heads(uint32_t head_dim, const Args &a, hipStream_t st) {
    const uint64_t rows = (uint64_t)a.tokens * a.group, w = (rows + 127) / 128 * a.n_kv;
    if (head_dim == 64) {
        if (w < 1024) return launch_prompt<E, 64, 2, 2, 32, 4>(a, st);
        return launch_prompt<E, 64, 4, 1, 64, 2>(a, st);
    }
    if (head_dim == 128) {
        if (w < 512) return launch_prompt<E, 128, 2, 2, 32, 2>(a, st);
        if (w < 1024) return launch_prompt<E, 128, 4, 1, 64, 2>(a, st);
        if (rows / a.n_seqs < 16384) return launch_prompt<E, 128, 4, 1, 32, 3>(a, st);
        return launch_prompt<E, 128, 8, 1, 64, 2>(a, st);
    }
    if (w <= 256) return launch_prompt<E, 256, 2, 2, 32, 1>(a, st);
    return launch_prompt<E, 256, 8, 1, 32, 2>(a, st);
}

}  // namespace
}  // namespace fellm

extern "C" int fellm_rocm_prompt_attention(const void *q, uint32_t q_stride, const void *k, uint32_t k_stride,
                                           const void *v, uint32_t v_stride, void *out, uint32_t dtype,
                                           const uint32_t *cu_seqlens, uint32_t n_seqs, uint32_t tokens,
                                           uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, float scale,
                                           uint32_t causal, uint32_t window, void *stream) {
    using namespace fellm;
    if (dtype != FELLM_DTYPE_F16 && dtype != FELLM_DTYPE_BF16) return FELLM_ERR_DTYPE;
    if (!n_kv_heads || !n_heads || n_heads % n_kv_heads) return FELLM_ERR_SHAPE;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return FELLM_ERR_SHAPE;
    if (n_seqs == 0 || tokens == 0) return FELLM_OK;
    if (!q || !k || !v || !out || !cu_seqlens) return FELLM_ERR_ARITY;
    const uint64_t qw = (uint64_t)n_heads * head_dim, kw = (uint64_t)n_kv_heads * head_dim;
    if (qw > 0x7fffffffull || (uint64_t)tokens * n_heads > 0x7fffffffull) return FELLM_ERR_SHAPE;
    if (q_stride < qw || k_stride < kw || v_stride < kw) return FELLM_ERR_SHAPE;
    // 16-byte pieces, and 16 rows of a tile inside a buffer resource's 31 bits
    if (q_stride % 8 || k_stride % 8 || v_stride % 8 || k_stride > (1u << 26) || v_stride > (1u << 26)) return FELLM_ERR_SHAPE;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 16)) return FELLM_ERR_SHAPE;
    if (!(scale > 0.0f)) scale = 1.0f / sqrtf((float)head_dim);
    rows_attn::Args a{};
    a.q = q;
    a.out = out;
    a.k = static_cast<const uint8_t *>(k);
    a.v = static_cast<const uint8_t *>(v);
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.out_stride = (uint32_t)qw;
    a.q_dtype = a.out_dtype = dtype;
    a.cu = cu_seqlens;
    a.n_seqs = n_seqs;
    a.tokens = tokens;
    a.n_heads = n_heads;
    a.n_kv = n_kv_heads;
    a.group = n_heads / n_kv_heads;
    a.by_group = rows_attn::Divisor(a.group);
    a.c = scale * 1.4426950408889634f;
    a.causal = causal;
    a.window = window;
    hipStream_t st = as_stream(stream);
    return dtype == FELLM_DTYPE_BF16 ? prompt_heads<rows_attn::ElemBF16>(head_dim, a, st)
                                     : prompt_heads<rows_attn::ElemF16>(head_dim, a, st);
}
