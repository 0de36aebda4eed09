// Slots of the paged KV cache and the shapes of a rotation, as the kernels that
// rotate rows and append them to the cache share them.
#pragma once

#include "common.hpp"

namespace fellm {

constexpr uint32_t kMaxHalf = 512;  // rope_dim <= 1024

struct KvDev {
    uint8_t *arena;
    uint64_t arena_len;
    const uint32_t *table;
    uint64_t n_table;
    uint32_t n_logical, n_layers, layer, block_size;
    uint64_t block_bytes;
    uint32_t stride;
};

// Byte offset of (batch row, position)'s K row, or UINT64_MAX if the slot lies
// outside the table or the arena.  V rows sit block_size rows further on.
__device__ __forceinline__ uint64_t kv_slot_offset(const KvDev &kv, uint32_t row, uint32_t pos) {
    const uint32_t logical = pos / kv.block_size;
    const uint32_t slot = pos % kv.block_size;
    if (logical >= kv.n_logical) return ~0ull;
    const uint64_t idx = ((uint64_t)row * kv.n_layers + kv.layer) * kv.n_logical + logical;
    if (idx >= kv.n_table) return ~0ull;
    const uint64_t phys = kv.table[idx];
    const uint64_t row_bytes = (uint64_t)kv.stride * 2;
    const uint64_t base = phys * kv.block_bytes + (uint64_t)slot * row_bytes;
    if (base + (uint64_t)kv.block_size * row_bytes + row_bytes > kv.arena_len) return ~0ull;
    return base;
}

inline bool make_kv(const FellmRocmPagedKv *p, KvDev &kv) {
    if (!p || !p->arena || !p->block_table || p->block_size == 0 || p->stride == 0 || p->n_layers == 0 ||
        p->n_logical_blocks == 0 || p->layer >= p->n_layers)
        return false;
    // A block holds block_size K rows then block_size V rows of 2-byte elements.
    if (p->block_bytes < (uint64_t)2 * p->block_size * p->stride * 2 || p->block_bytes % 4) return false;
    kv = KvDev{(uint8_t *)p->arena, p->arena_len, p->block_table, p->n_block_table, p->n_logical_blocks,
               p->n_layers, p->layer, p->block_size, p->block_bytes, p->stride};
    return true;
}

template <typename Fn>
int dispatch_cache(uint32_t kv_dtype, Fn &&f) {
    if (kv_dtype == FELLM_DTYPE_F16) return f.template operator()<F16>();
    if (kv_dtype == FELLM_DTYPE_BF16) return f.template operator()<BF16>();
    return FELLM_ERR_DTYPE;
}

inline int check_rope_shape(uint32_t head_dim, uint32_t rope_dim, uint32_t pairing) {
    if (head_dim == 0 || head_dim % 2) return FELLM_ERR_SHAPE;
    if (rope_dim % 2 || rope_dim > head_dim || rope_dim / 2 > kMaxHalf) return FELLM_ERR_SHAPE;
    if (pairing > 2) return FELLM_ERR_SHAPE;
    return FELLM_OK;
}

}  // namespace fellm
