"""Attention of drafted trees and prompt chunks over the paged cache against
the 64-bit formula (tolerances: attention_util.attend)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attention_util import attend, causal_mask, check  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from fellm_amd import ops as _ops

    return _ops


def tolerance_args(act, kv, out):
    """Rounding of a probability: one 16-bit number, or parts of f32 accuracy
    (f16: two parts, 2^-22 of values above 2^-17, 2^-40 absolute; bf16: three, 2^-24)."""
    if act == kv == out:
        return {"f16": dict(p_half=2.0 ** -11, p_floor=2.0 ** -29), "bf16": dict(p_half=2.0 ** -8)}[kv]
    return {"f16": dict(p_half=2.0 ** -22, p_floor=2.0 ** -40), "bf16": dict(p_half=2.0 ** -24)}[kv]


class Case:
    """Sequences with a prefix and new tokens, their K/V in a paged cache whose
    other slots and blocks hold NaN."""

    def __init__(self, ops, dev, nodes, prefix, heads, kv_heads, hd, act, kv, *, n_layers=1, layer=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.nodes, self.prefix, self.heads, self.kv_heads, self.hd, self.dev = nodes, prefix, heads, kv_heads, hd, dev
        self.q = (1.5 * torch.randn(sum(nodes), heads * hd, generator=g)).to(DT[act])
        keys = [p + n for p, n in zip(prefix, nodes)]
        self.k, self.v = ([torch.randn(s, kv_heads, hd, generator=g).to(DT[kv]) for s in keys] for _ in range(2))
        need = [(s + 15) // 16 for s in keys]
        stride, n_logical = kv_heads * hd, max(max(need), 1) + 1
        blocks = sum(need) + 2
        arena = torch.full((blocks, 2, 16, stride), float("nan"), dtype=DT[kv])
        order = torch.randperm(blocks, generator=g)
        table = torch.full((len(nodes), n_layers, n_logical), 0x7fffffff, dtype=torch.int32)
        at = 0
        for b, s in enumerate(keys):
            for j in range(need[b]):
                table[b, layer, j] = order[at]
                part = slice(16 * j, min(16 * j + 16, s))
                arena[order[at], 0, :part.stop - part.start] = self.k[b][part].flatten(1)
                arena[order[at], 1, :part.stop - part.start] = self.v[b][part].flatten(1)
                at += 1
        self.cache = ops.PagedKvCache(arena=arena.view(torch.uint8).flatten().to(dev), block_table=table.to(dev),
                                      n_layers=n_layers, n_logical_blocks=n_logical, block_size=16,
                                      block_bytes=64 * stride, stride=stride, kv_dtype=DT[kv])
        self.cu = torch.tensor([sum(nodes[:i]) for i in range(len(nodes) + 1)], dtype=torch.int32)
        self.plen = torch.tensor(prefix, dtype=torch.int32)
        self.layer, self.act, self.kv = layer, act, kv

    def run(self, ops, *, bits=None, out_dtype=None, words=None, **kw):
        """bits: for each sequence a bool [n, n]."""
        mask = None
        if bits is not None:
            words = words or (max(self.nodes) + 31) // 32
            mask = torch.zeros(sum(self.nodes), words, dtype=torch.int64)
            at = 0
            for b in bits:
                for j in range(min(b.shape[1], 32 * words)):
                    mask[at:at + b.shape[0], j // 32] |= b[:, j].long() << (j % 32)
                at += b.shape[0]
            mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32).to(self.dev)
        kw = {"max_nodes": max(self.nodes), "max_prefix": max(self.prefix), **kw}
        return ops.paged_tree_attention(self.q.to(self.dev), self.cu.to(self.dev), self.plen.to(self.dev), self.cache,
                                        tree_mask=mask, n_heads=self.heads, n_kv_heads=self.kv_heads, head_dim=self.hd,
                                        layer=self.layer, out_dtype=DT[out_dtype] if out_dtype else None, **kw)

    def check(self, got, *, bits=None, window=0, out_dtype=None, scale=None):
        out = out_dtype or self.act
        at = 0
        for b, (n, p) in enumerate(zip(self.nodes, self.prefix)):
            if bits is None:
                allow = causal_mask(n, p, window)
            else:
                allow = torch.cat([torch.ones(n, p, dtype=torch.bool), bits[b]], 1)
            if n:
                want, tol = attend(self.q[at:at + n].view(n, self.heads, self.hd), self.k[b], self.v[b], allow, scale,
                                   out_dtype=DT[out], **tolerance_args(self.act, self.kv, out))
                assert torch.isfinite(want).all()
                check(got[at:at + n].view(n, self.heads, self.hd), want, tol, f"sequence {b}")
            at += n


def tree_bits(nodes, seed=0):
    """Ancestors and self of a random tree."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in nodes:
        b = torch.eye(n, dtype=torch.bool)
        for i in range(1, n):
            b[i] |= b[int(torch.randint(0, i, (1,), generator=g))]
        out.append(b)
    return out


HEADS = [(32, 8, 64), (8, 8, 64), (8, 2, 128), (28, 4, 128), (7, 1, 128), (16, 1, 128), (4, 2, 256), (16, 1, 256)]


@pytest.mark.parametrize("act,kv,out", [("f16", "f16", None), ("bf16", "bf16", None), ("f32", "f16", None),
                                        ("f32", "bf16", None), ("f16", "f16", "f32"), ("bf16", "f16", None),
                                        ("f16", "bf16", None), ("bf16", "bf16", "f32")])
@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
def test_trees(ops, dev, heads, kv_heads, hd, act, kv, out):
    c = Case(ops, dev, [1, 9, 33, 5], [100, 0, 17, 333], heads, kv_heads, hd, act, kv, seed=hd + heads)
    bits = tree_bits(c.nodes)
    c.check(c.run(ops, bits=bits, out_dtype=out), bits=bits, out_dtype=out)


@pytest.mark.parametrize("n", [1, 2, 4, 8, 9, 16, 31, 32, 33, 63, 64, 65, 100, 129])
@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f32", "f16")])
def test_tree_sizes(ops, dev, n, act, kv):
    """Every number of row tiles: four heads share a K/V head."""
    c = Case(ops, dev, [n, 3], [50, 15], 8, 2, 128, act, kv, seed=n)
    bits = tree_bits(c.nodes, n)
    c.check(c.run(ops, bits=bits), bits=bits)


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 31, 32, 48, 63, 64, 65, 127, 1000])
@pytest.mark.parametrize("nodes", [1, 8, 40])
def test_prefix_lengths(ops, dev, prefix, nodes):
    c = Case(ops, dev, [nodes, nodes], [prefix, prefix // 2], 8, 2, 128, "f16", "f16", seed=prefix)
    bits = tree_bits(c.nodes, prefix)
    c.check(c.run(ops, bits=bits), bits=bits)
    c.check(c.run(ops))


@pytest.mark.parametrize("window", [0, 1, 16, 100, 5000])
@pytest.mark.parametrize("act,kv,hd", [("bf16", "bf16", 128), ("f32", "f16", 64), ("f16", "f16", 256)])
def test_chunks(ops, dev, window, act, kv, hd):
    c = Case(ops, dev, [150, 1, 64], [200, 999, 0], 8, 2, hd, act, kv, seed=window)
    c.check(c.run(ops, window=window), window=window)


def test_rows_without_keys_are_zero(ops, dev):
    c = Case(ops, dev, [6, 3], [0, 40], 8, 2, 128, "bf16", "bf16")
    bits = tree_bits(c.nodes)
    bits[0][2] = False
    bits[0][5] = False
    bits[1][1] = False  # the prefix stays
    got = c.run(ops, bits=bits)
    assert (got[2] == 0).all() and (got[5] == 0).all()
    c.check(got, bits=bits)


def test_more_heads_than_a_tile_has_rows(ops, dev):
    c = Case(ops, dev, [3, 1, 5], [20, 300, 0], 40, 1, 64, "bf16", "bf16")
    bits = tree_bits(c.nodes)
    c.check(c.run(ops, bits=bits), bits=bits)


@pytest.mark.parametrize("act,kv,hd", [("bf16", "bf16", 128), ("f32", "f16", 64), ("f16", "f16", 256)])
def test_pieces_that_span_tiles(ops, dev, act, kv, hd):
    """More tiles than workgroups: each walks several, shared at both ends."""
    n = 96
    c = Case(ops, dev, [1 + (7 * i) % 40 for i in range(n)], [(131 * i) % 700 for i in range(n)], 16, 8, hd, act, kv)
    bits = tree_bits(c.nodes)
    got = c.run(ops, bits=bits)
    c.check(got, bits=bits)
    assert torch.equal(c.run(ops, bits=bits), got)


@pytest.mark.parametrize("nodes,prefix,heads,kv_heads,hd", [
    ([2100], [0], 24, 4, 64), ([1500, 1, 0, 700], [0, 50, 9, 333], 16, 2, 128), ([1030], [600], 7, 1, 256),
    ([9] * 70, [40] * 70, 64, 8, 64)])
def test_long_chunks(ops, dev, nodes, prefix, heads, kv_heads, hd):
    """Causal chunks whose tiles have rising numbers of keys, in shares of equal work."""
    c = Case(ops, dev, nodes, prefix, heads, kv_heads, hd, "bf16", "bf16")
    got = c.run(ops)
    c.check(got)
    assert torch.equal(c.run(ops), got)


@pytest.mark.parametrize("act,kv,hd,heads", [("bf16", "bf16", 128, 8), ("f16", "f16", 64, 8), ("f32", "bf16", 128, 4)])
def test_attended_scores_of_minus_infinity(ops, dev, act, kv, hd, heads):
    """Keys whose scores are -inf weigh nothing, also where they fill a whole share
    of the keys; a row that has no others is 0 / 0."""
    n, p = 4, 5000
    c = Case(ops, dev, [n], [p], heads, 2, hd, act, kv)
    c.q.view(n, heads, hd)[:, :, 0] = c.q.view(n, heads, hd)[:, :, 0].abs() + 0.25
    arena = c.cache.arena.view(DT[kv]).view(-1, 2, 16, 2 * hd)
    blocks = c.cache.block_table.long()[0, 0]

    def hide(first, last):
        for j in range(first, last):
            arena[blocks[j // 16], 0, j % 16].view(2, hd)[:, 0] = float("-inf")

    hide(640, 3200)
    allow = causal_mask(n, p)
    allow[:, 640:3200] = False
    want, tol = attend(c.q.view(n, heads, hd), c.k[0], c.v[0], allow, out_dtype=DT[act], **tolerance_args(act, kv, act))
    check(c.run(ops).view(n, heads, hd), want, tol)
    hide(0, p + n)
    assert torch.isnan(c.run(ops)).all()


def test_any_mask(ops, dev):
    """Bits above the diagonal, without the token itself, over several words."""
    g = torch.Generator().manual_seed(3)
    c = Case(ops, dev, [90, 70], [33, 5], 4, 1, 128, "bf16", "bf16")
    bits = [torch.rand(n, n, generator=g) < 0.2 for n in c.nodes]
    c.check(c.run(ops, bits=bits), bits=bits)


def test_fewer_mask_words_than_tokens(ops, dev):
    c = Case(ops, dev, [70, 10], [20, 3], 4, 1, 64, "f16", "f16")
    bits = tree_bits(c.nodes)
    got = c.run(ops, bits=bits, words=1)
    for b in bits:
        b[:, 32:] = False
    c.check(got, bits=bits)


@pytest.mark.parametrize("heads,kv_heads,hd,nodes", [(8, 2, 128, [4, 1]), (8, 2, 128, [16, 3]), (28, 4, 128, [20, 31]),
                                                     (4, 4, 64, [7, 2]), (4, 2, 256, [9, 40]), (2, 1, 256, [12])])
@pytest.mark.parametrize("act,kv", [("bf16", "bf16"), ("f32", "f16")])
def test_long_prefixes_are_split(ops, dev, heads, kv_heads, hd, nodes, act, kv):
    prefix = [5000, 70][:len(nodes)]
    c = Case(ops, dev, nodes, prefix, heads, kv_heads, hd, act, kv, seed=7)
    from fellm_amd import lib
    assert lib().fellm_rocm_paged_tree_attention_workspace(len(nodes), sum(nodes), heads, kv_heads, hd, max(nodes),
                                                           max(prefix)) > 0
    bits = tree_bits(nodes)
    split = c.run(ops, bits=bits)
    c.check(split, bits=bits)
    whole = c.run(ops, bits=bits, workspace=torch.empty(0, dtype=torch.float32, device=dev))
    c.check(whole, bits=bits)
    for _ in range(3):
        assert torch.equal(c.run(ops, bits=bits), split)
    # launches chosen for other bounds than the device's lengths
    c.check(c.run(ops, bits=bits, max_prefix=20000), bits=bits)
    c.check(c.run(ops, bits=bits, max_prefix=600), bits=bits)
    c.check(c.run(ops, bits=bits, max_nodes=1), bits=bits)
    c.check(c.run(ops, bits=bits, max_nodes=4096), bits=bits)


def test_window_over_splits(ops, dev):
    c = Case(ops, dev, [40, 3], [4000, 900], 8, 2, 128, "f16", "f16", seed=1)
    for window in (5, 700, 2500):
        c.check(c.run(ops, window=window), window=window)


def test_layers_and_many_sequences(ops, dev):
    n = 150
    c = Case(ops, dev, [1 + i % 3 for i in range(n)], [(7 * i) % 60 for i in range(n)], 4, 2, 64, "f16", "f16",
             n_layers=3, layer=1)
    bits = tree_bits(c.nodes)
    c.check(c.run(ops, bits=bits), bits=bits)


def test_empty_sequences(ops, dev):
    c = Case(ops, dev, [0, 5, 0, 0, 2, 0], [10, 20, 0, 30, 40, 5], 4, 2, 64, "f16", "f16")
    c.check(c.run(ops))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_masked_nodes_do_not_count(ops, dev, value):
    """A drafted token that no other token attends may hold anything."""
    c = Case(ops, dev, [12], [30], 8, 2, 128, "bf16", "bf16")
    bits = [torch.tril(torch.ones(12, 12, dtype=torch.bool))]
    bits[0][:, 4] = False
    kv = c.cache.arena.view(torch.bfloat16).view(-1, 2, 16, 256)
    phys = int(c.cache.block_table.flatten()[34 // 16])
    kv[phys, :, 34 % 16] = value
    c.check(c.run(ops, bits=bits), bits=bits)
    bits[0][9, 4] = True
    got = c.run(ops, bits=bits)
    assert torch.isnan(got[9]).all()
    keep = [i for i in range(12) if i != 9]
    assert torch.isfinite(got[keep]).all()


def test_other_stream_and_graph(ops, dev):
    from fellm_amd import graph, lib

    c = Case(ops, dev, [8, 5], [3000, 50], 8, 2, 128, "bf16", "bf16")
    q, cu, plen = c.q.to(dev), c.cu.to(dev), c.plen.to(dev)
    kw = dict(n_heads=8, n_kv_heads=2, head_dim=128, max_nodes=8, max_prefix=3000)
    need = lib().fellm_rocm_paged_tree_attention_workspace(2, 13, 8, 2, 128, 8, 3000)
    assert need
    ws = torch.empty(need // 4, dtype=torch.float32, device=dev)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), graph.GraphCapture(stream) as cap:
        ops.paged_tree_attention(q, cu, plen, c.cache, out=out, workspace=ws, **kw)
    for lens in ([3000, 50], [2000, 10], [1, 0]):
        plen.copy_(torch.tensor(lens, dtype=torch.int32))
        want = ops.paged_tree_attention(q, cu, plen, c.cache, **kw)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cap.graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(ops, dev):
    from fellm_amd import FellmRocmError

    c = Case(ops, dev, [4], [10], 4, 2, 64, "f16", "f16")
    with pytest.raises(FellmRocmError):
        c.run(ops, bits=tree_bits([4]), window=3)
    with pytest.raises(FellmRocmError):
        c.run(ops, out_dtype="bf16")
    with pytest.raises(ValueError):
        c.run(ops, out=torch.empty(4, 64, dtype=torch.float16, device=dev))
    q, cu, plen = c.q.to(dev), c.cu.to(dev), c.plen.to(dev)
    kw = dict(n_heads=4, n_kv_heads=2, head_dim=64, max_nodes=4, max_prefix=10)
    with pytest.raises(ValueError):
        ops.paged_tree_attention(q[:, :64], cu, plen, c.cache, **kw)
    with pytest.raises(ValueError):
        ops.paged_tree_attention(q, cu, torch.zeros(2, dtype=torch.int32, device=dev), c.cache, **kw)
    with pytest.raises(TypeError):
        ops.paged_tree_attention(q, cu, plen.long(), c.cache, **kw)
    with pytest.raises(ValueError):
        ops.paged_tree_attention(q, cu, plen, c.cache, tree_mask=torch.zeros(3, 1, dtype=torch.int32, device=dev), **kw)
    with pytest.raises(TypeError):
        ops.paged_tree_attention(q, cu, plen, c.cache, tree_mask=torch.ones(4, 1, dtype=torch.int64, device=dev), **kw)
    with pytest.raises(FellmRocmError):
        ops.paged_tree_attention(q, cu, plen, c.cache, **{**kw, "n_kv_heads": 4})
    with pytest.raises(ValueError):
        ops.paged_tree_attention(q, cu.cpu(), plen, c.cache, **kw)
