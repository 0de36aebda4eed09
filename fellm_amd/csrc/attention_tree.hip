// Attention of several new tokens per sequence over the paged KV cache: the
// verification of a tree of drafted tokens (each token attends the cached
// prefix and the drafted tokens its mask names), or a chunk of a prompt behind
// a cached prefix (no mask: causal).  The new tokens' K and V are in the cache
// already, after the prefix.  The kernel is rows_kernel of attention_rows.hpp;
// tiles that several workgroups share are joined by rows_combine.
#include "attention_rows.hpp"

#include <algorithm>
#include <type_traits>

namespace fellm {
namespace {
using namespace rows_attn;

// Layouts by the rows of a sequence: tiles of 32, 64 or 128 rows, the smallest
// that holds them; the wavefronts without rows of their own share the keys.
// KW: those wavefronts; KT: keys of a wavefront's tile; OCC: wavefronts per SIMD.
template <int HD, int RW, bool PARTS>
struct Layout {
    static constexpr int KW = RW == 4 ? 1 : HD == 256 || RW == 2 ? 2 : 4;
    static constexpr int KT = RW == 4 && HD != 256 && !PARTS ? 64 : 32;
    static constexpr int OCC = HD == 256 || (RW == 1 && HD == 128) ? 1 : 2;
    static constexpr uint32_t BM = kRows * RW, TK = KT * KW;
    // Workgroups that are resident at once, and the rounds of the least keys that
    // one takes, below which the joining costs more than the walk.  Least keys 192,
    // 128, 64, us: two tokens behind 445 (f32 q, 32/8 heads of 128) 16.4, 14.1,
    // 14.0; two of 57 behind 330 (64/8) 24.0, 22.6, 27.2; eleven of 21 behind up to
    // 985 (32/8) 24.7, 26.3, 27.4
    static constexpr uint32_t kSlots = 256 * OCC, kMinRounds = (128 + TK - 1) / TK;
};

struct Plan {
    uint64_t tiles;       // of all sequences, at most
    uint32_t ids;         // workgroups per K/V head
    uint64_t part_bytes;  // their records
};

template <int HD, int RW, bool PARTS>
Plan plan(uint32_t n_seqs, uint32_t tokens, uint32_t group, uint32_t n_kv, uint32_t max_nodes, uint32_t max_prefix) {
    using L = Layout<HD, RW, PARTS>;
    Plan p;
    // one sequence: exactly its tiles; more: the most that tokens rows can need
    const uint64_t all = (uint64_t)tokens * group;
    p.tiles = n_seqs == 1 ? (all + L::BM - 1) / L::BM : all / L::BM + n_seqs;
    const uint64_t used = std::min<uint64_t>(p.tiles, (uint64_t)n_seqs * (((uint64_t)max_nodes * group + L::BM - 1) / L::BM));
    const uint64_t rounds = used * (((uint64_t)max_prefix + max_nodes + L::TK - 1) / L::TK);
    const uint64_t most = std::max<uint64_t>((rounds + L::kMinRounds - 1) / L::kMinRounds + used, 1);
    p.ids = (uint32_t)std::min<uint64_t>(std::max(L::kSlots / n_kv, 1u), most);
    p.part_bytes = p.ids == 1 ? 0 : (uint64_t)p.ids * n_kv * 2 * L::BM * kRec<HD> * 4;
    return p;
}

template <typename Fn>
auto with_layout(uint32_t head_dim, uint64_t rows, bool parts, Fn &&f) {
    auto pick_rows = [&]<int HD, bool PARTS>() {
        if (rows <= 32) return f.template operator()<HD, 1, PARTS>();
        if (rows <= 64) return f.template operator()<HD, 2, PARTS>();
        return f.template operator()<HD, 4, PARTS>();
    };
    auto pick_head = [&]<bool PARTS>() {
        if (head_dim == 64) return pick_rows.template operator()<64, PARTS>();
        if (head_dim == 128) return pick_rows.template operator()<128, PARTS>();
        return pick_rows.template operator()<256, PARTS>();
    };
    return parts ? pick_head.template operator()<true>() : pick_head.template operator()<false>();
}

template <typename E, int HD, int RW, bool PARTS, bool EVEN>
int launch_tree(const Plan &p, Args a, hipStream_t st) {
    using L = Layout<HD, RW, PARTS>;
    const uint64_t grid = (uint64_t)p.ids * a.n_kv, rows = p.tiles * a.n_kv * L::BM;
    // a launch has fewer than 2^32 threads; positions on the line are 32 bits
    if (std::max(grid * 4 * kWave, rows * 64) > 0xffffffffull) return FELLM_ERR_SHAPE;
    if (p.tiles * (((uint64_t)a.max_before + a.tokens) / L::TK + 1) > 0x3fffffffull) return FELLM_ERR_SHAPE;
    a.min_rounds = L::kMinRounds;
    FELLM_LAUNCH((rows_kernel<E, HD, RW, L::KW, L::KT, true, PARTS, L::OCC, EVEN>), dim3((uint32_t)grid),
                 dim3(kWave * RW * L::KW), 0, st, a);
    int rc = launch_status();
    if (rc != FELLM_OK || !a.part) return rc;
    // 64 lanes a row where a tile can have many records (one sequence of 32768
    // keys, 28/4 heads: 44.0 -> 38.1 us; eight of up to 1000 the other way 22.5, 24.6)
    auto join = [&]<int Q>() {
        FELLM_LAUNCH((rows_combine<HD, L::BM, L::TK, Q, EVEN>), dim3((uint32_t)(rows / (kJoinThreads / 16 / Q))),
                     dim3(kJoinThreads), 0, st, a, p.ids);
    };
    if (p.ids > 4 * p.tiles) join.template operator()<4>();
    else join.template operator()<1>();
    return launch_status();
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
    const uint32_t group = n_heads / n_kv_heads, nodes = std::min(std::max(max_nodes, 1u), tokens);
    uint64_t need = 0;
    for (bool parts : {false, true})
        need = std::max(need, with_layout(head_dim, (uint64_t)nodes * group, parts, [&]<int HD, int RW, bool PARTS>() {
                            return plan<HD, RW, PARTS>(n_seqs, tokens, group, n_kv_heads, nodes, max_prefix).part_bytes;
                        }));
    return need;
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
    if ((uint64_t)n_kv_heads * head_dim != kv->stride || kv->block_size != rows_attn::kBlockTokens || kv->stride > (1u << 25))
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
    a.by_group = rows_attn::Divisor(a.group);
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
    hipStream_t st = as_stream(stream);
    const bool parts = q_dtype != kv->kv_dtype || out_dtype != kv->kv_dtype;
    const uint32_t nodes = std::min(std::max(max_nodes, 1u), tokens);
    return with_layout(head_dim, (uint64_t)nodes * a.group, parts, [&]<int HD, int RW, bool PARTS>() {
        const Plan p = plan<HD, RW, PARTS>(n_seqs, tokens, a.group, n_kv_heads, nodes, max_prefix);
        a.part = p.part_bytes && workspace && workspace_bytes >= p.part_bytes ? workspace : nullptr;
        auto launch = [&]<bool EVEN>() {
            return kv->kv_dtype == FELLM_DTYPE_BF16 ? launch_tree<rows_attn::ElemBF16, HD, RW, PARTS, EVEN>(p, a, st)
                                                    : launch_tree<rows_attn::ElemF16, HD, RW, PARTS, EVEN>(p, a, st);
        };
        // rows for at least a tile to three workgroups, which ragged trees double
        // (and below 32768 tiles: the sums of Line::upto stay below 2^32)
        const uint64_t whole = (uint64_t)tokens * a.group / (rows_attn::kRows * RW);
        if constexpr (RW == 4)
            if (a.part && 3 * whole >= p.ids && whole < 32768) return launch.template operator()<true>();
        return launch.template operator()<false>();
    });
}
