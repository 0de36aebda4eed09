// Attention of several new tokens per sequence over the paged KV cache: the
// verification of a tree of drafted tokens (each token attends the cached
// prefix and the drafted tokens its mask names), or a chunk of a prompt behind
// a cached prefix (no mask: causal).  The new tokens' K and V are in the cache
// already, after the prefix.  The kernel is rows_kernel of attention_rows.hpp;
// long caches of few rows are split over the keys and joined by rows_combine.
#include "attention_rows.hpp"

#include <algorithm>
#include <type_traits>

namespace fellm {
namespace {
using namespace rows_attn;

struct Plan {
    uint32_t rw;  // wavefronts that own rows: tiles of 32 rw rows
    uint64_t tiles;
    uint32_t splits, keys_per_split;
};

// Tiles of 32, 64 or 128 rows, the smallest that holds a sequence's rows: the
// wavefronts without rows of their own share the keys.  The keys are split until
// the launch has kTargetGroups workgroups, in parts of at least kMinKeys; the
// keys of several sequences, whose lengths differ, in parts of at most kMaxKeys.
#ifndef FELLM_TREE_GROUPS
#define FELLM_TREE_GROUPS 512
#endif
#ifndef FELLM_TREE_MIN
#define FELLM_TREE_MIN 192
#endif
#ifndef FELLM_TREE_MAX
#define FELLM_TREE_MAX 2048
#endif
#ifndef FELLM_TREE_MANY
#define FELLM_TREE_MANY 1024
#endif
constexpr uint32_t kTargetMany = FELLM_TREE_MANY;
constexpr uint32_t kTargetGroups = FELLM_TREE_GROUPS, kMinKeys = FELLM_TREE_MIN, kMaxKeys = FELLM_TREE_MAX;

Plan plan(uint32_t n_seqs, uint32_t tokens, uint32_t group, uint32_t n_kv, uint32_t max_nodes, uint32_t max_prefix) {
    Plan p;
    max_nodes = std::min(std::max(max_nodes, 1u), tokens);
    const uint64_t rows = (uint64_t)max_nodes * group;
    p.rw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    const uint32_t bm = kRows * p.rw;
    // one sequence: exactly its tiles; more: the most that tokens rows can need
    p.tiles = n_seqs == 1 ? ((uint64_t)tokens * group + bm - 1) / bm : (uint64_t)tokens * group / bm + n_seqs;
    const uint64_t used = std::min<uint64_t>(p.tiles, (uint64_t)n_seqs * ((rows + bm - 1) / bm)) * n_kv;
    const uint64_t keys = (uint64_t)max_prefix + max_nodes;
    uint64_t splits = std::min<uint64_t>(((n_seqs > 1 ? kTargetMany : kTargetGroups) + used - 1) / std::max<uint64_t>(used, 1), (keys + kMinKeys - 1) / kMinKeys);
    splits = std::max<uint64_t>(splits, n_seqs > 1 ? (keys + kMaxKeys - 1) / kMaxKeys : 1);
    if (splits == 1) {
        p.splits = 1;
        p.keys_per_split = 0x7fffffc0u;
        return p;
    }
    p.keys_per_split = (uint32_t)(((keys + splits - 1) / splits + 63) / 64 * 64);
    p.splits = (uint32_t)((keys + p.keys_per_split - 1) / p.keys_per_split);
    // a share starts at a multiple of 64 below its first key
    if (p.splits == 1) p.keys_per_split = 0x7fffffc0u;
    return p;
}

uint64_t part_bytes(const Plan &p, uint32_t n_kv, uint32_t head_dim) {
    return p.splits <= 1 ? 0 : p.tiles * n_kv * p.splits * kRows * p.rw * (head_dim + 4) * 4;
}

#ifndef CFG4
#define CFG4 64, 2, 2
#endif
#ifndef OCC12
#define OCC12 2
#endif
#ifndef CFG4P
#define CFG4P 32, 2, 2
#endif
template <int KT_, int OCC_, int NST_> struct Layout { static constexpr int KT = KT_, OCC = OCC_, NST = NST_; };
template <typename E, int HD, int RW, bool PARTS>
int launch_tree(const Plan &p, const Args &a, hipStream_t st) {
    constexpr int KW = RW == 4 ? 1 : HD == 256 || RW == 2 ? 2 : 4;
    using L = std::conditional_t<RW == 4 && HD != 256, std::conditional_t<PARTS, Layout<CFG4P>, Layout<CFG4>>, Layout<32, HD == 256 || (RW == 1 && HD == 128) ? 1 : OCC12, 2>>;
    constexpr uint32_t BM = kRows * RW;
    const uint64_t grid = p.tiles * a.n_kv * a.splits, join = p.tiles * a.n_kv * (BM / kJoinRows);
    // a launch has fewer than 2^32 threads
    if (std::max(grid, join) > 0xffffffffull / (4 * kWave)) return FELLM_ERR_SHAPE;
    FELLM_LAUNCH((rows_kernel<E, HD, RW, KW, L::KT, true, PARTS, L::OCC, L::NST>), dim3((uint32_t)grid), dim3(kWave * RW * KW), 0, st, a);
    int rc = launch_status();
    if (rc != FELLM_OK || a.splits == 1) return rc;
    FELLM_LAUNCH((rows_combine<HD, BM>), dim3((uint32_t)join), dim3(kJoinRows * 16), 0, st, a);
    return launch_status();
}

template <typename E, int HD, bool PARTS>
int tree_rows(const Plan &p, const Args &a, hipStream_t st) {
    return p.rw == 1 ? launch_tree<E, HD, 1, PARTS>(p, a, st)
                     : p.rw == 2 ? launch_tree<E, HD, 2, PARTS>(p, a, st) : launch_tree<E, HD, 4, PARTS>(p, a, st);
}

template <typename E, bool PARTS>
int tree_heads(uint32_t head_dim, const Plan &p, const Args &a, hipStream_t st) {
    if (head_dim == 64) return tree_rows<E, 64, PARTS>(p, a, st);
    if (head_dim == 128) return tree_rows<E, 128, PARTS>(p, a, st);
    return tree_rows<E, 256, PARTS>(p, a, st);
}

bool tree_heads_ok(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    return n_kv_heads && n_heads && n_heads % n_kv_heads == 0 && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace
}  // namespace fellm

extern "C" uint64_t fellm_rocm_paged_tree_attention_workspace(uint32_t n_seqs, uint32_t tokens, uint32_t n_heads,
                                                              uint32_t n_kv_heads, uint32_t head_dim,
                                                              uint32_t max_nodes, uint32_t max_prefix) {
    using namespace fellm;
    if (!tree_heads_ok(n_heads, n_kv_heads, head_dim) || !n_seqs || !tokens) return 0;
    const Plan p = plan(n_seqs, tokens, n_heads / n_kv_heads, n_kv_heads, max_nodes, max_prefix);
    return part_bytes(p, n_kv_heads, head_dim);
}

extern "C" int fellm_rocm_paged_tree_attention(const void *q, uint32_t q_dtype, void *out, uint32_t out_dtype,
                                               const uint32_t *cu_nodes, const uint32_t *prefix_lengths,
                                               uint32_t n_seqs, uint32_t tokens, const uint32_t *tree_mask,
                                               uint32_t mask_words, uint32_t n_heads, uint32_t n_kv_heads,
                                               uint32_t head_dim, uint32_t max_nodes, uint32_t max_prefix, float scale,
                                               uint32_t window, const FellmRocmPagedKv *kv, float *workspace,
                                               uint64_t workspace_bytes, void *stream) {
    using namespace fellm;
    if (!kv) return FELLM_ERR_ARITY;
    if (!tree_heads_ok(n_heads, n_kv_heads, head_dim)) return FELLM_ERR_SHAPE;
    if (kv->kv_dtype != FELLM_DTYPE_F16 && kv->kv_dtype != FELLM_DTYPE_BF16) return FELLM_ERR_DTYPE;
    if (!act_bytes(q_dtype) || (out_dtype != q_dtype && out_dtype != FELLM_DTYPE_F32)) return FELLM_ERR_DTYPE;
    if (n_seqs == 0 || tokens == 0) return FELLM_OK;
    if (!q || !out || !cu_nodes || !prefix_lengths || !kv->arena || !kv->block_table) return FELLM_ERR_ARITY;
    if ((tree_mask != nullptr) != (mask_words != 0) || (tree_mask && window)) return FELLM_ERR_SHAPE;
    if ((uint64_t)n_kv_heads * head_dim != kv->stride || kv->block_size != rows_attn::kBlockTokens || kv->stride > (1u << 26))
        return FELLM_ERR_SHAPE;
    if (kv->block_bytes < 2ull * kv->block_size * kv->stride * 2 || kv->block_bytes % 16) return FELLM_ERR_SHAPE;
    if (kv->layer >= kv->n_layers || kv->n_logical_blocks > (1u << 26)) return FELLM_ERR_SHAPE;
    if ((uint64_t)tokens * n_heads > 0x3fffffffull || (uint64_t)n_heads * head_dim > 0x7fffffffull)
        return FELLM_ERR_SHAPE;
    if (!aligned_to(kv->arena, 16) || !aligned_to(q, 16) || !aligned_to(out, 16)) return FELLM_ERR_SHAPE;
    if (workspace && !aligned_to(workspace, 16)) return FELLM_ERR_SHAPE;
    if (!(scale > 0.0f)) scale = 1.0f / sqrtf((float)head_dim);
    rows_attn::Args a{};
    a.q = q;
    a.out = out;
    a.q_stride = a.out_stride = n_heads * head_dim;
    a.q_dtype = q_dtype;
    a.out_dtype = out_dtype;
    a.cu = cu_nodes;
    a.before = prefix_lengths;
    a.max_before = kv->n_logical_blocks * rows_attn::kBlockTokens;
    a.mask = tree_mask;
    a.mask_words = mask_words;
    a.n_seqs = n_seqs;
    a.tokens = tokens;
    a.n_heads = n_heads;
    a.n_kv = n_kv_heads;
    a.group = n_heads / n_kv_heads;
    a.c = scale * 1.4426950408889634f;
    a.causal = 1;
    a.window = window;
    a.arena = static_cast<const uint8_t *>(kv->arena);
    a.arena_len = kv->arena_len;
    a.block_bytes = kv->block_bytes;
    a.n_table = kv->n_block_table;
    a.table = kv->block_table;
    a.n_logical = kv->n_logical_blocks;
    a.n_layers = kv->n_layers;
    a.layer = kv->layer;
    a.stride = kv->stride;
    Plan p = plan(n_seqs, tokens, a.group, n_kv_heads, max_nodes, max_prefix);
    if (p.splits > 1 && (!workspace || workspace_bytes < part_bytes(p, n_kv_heads, head_dim))) {
        p.splits = 1;
        p.keys_per_split = 0x7fffffc0u;
    }
    a.splits = p.splits;
    a.keys_per_split = p.keys_per_split;
    a.part = workspace;
    hipStream_t st = as_stream(stream);
    const bool parts = q_dtype != kv->kv_dtype || out_dtype != kv->kv_dtype;
    if (kv->kv_dtype == FELLM_DTYPE_BF16)
        return parts ? tree_heads<rows_attn::ElemBF16, true>(head_dim, p, a, st)
                     : tree_heads<rows_attn::ElemBF16, false>(head_dim, p, a, st);
    return parts ? tree_heads<rows_attn::ElemF16, true>(head_dim, p, a, st)
                 : tree_heads<rows_attn::ElemF16, false>(head_dim, p, a, st);
}
