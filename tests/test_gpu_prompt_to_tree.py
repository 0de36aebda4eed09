"""A prompt, then a drafted tree, as a serving loop runs them: norm + rotation
with the append, prompt attention, the tree's norm + append, tree attention."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attention_util import attend, causal_mask, check  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
FLOOR = {"f16": 2.0 ** -29, "bf16": 0.0}
PARENTS = [[-1, 0, 0, 1, 1, 2, 5, 3, 6], [-1, 0, 1, 2, 2]]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (7, 1, 64), (4, 2, 256)])
def test_prompt_then_tree(dev, kind, heads, kv_heads, hd):
    from fellm_amd import ops

    g = torch.Generator().manual_seed(hd)
    dt = DT[kind]
    lens, nodes = [61, 150], [len(p) for p in PARENTS]
    widths = [heads * hd, kv_heads * hd, kv_heads * hd]
    qw, kw = ((1 + 0.2 * torch.randn(hd, generator=g)).to(dev) for _ in range(2))
    inv = ops.rope_inv_freqs(1e6, hd).to(dev)
    n_logical = 12
    table = torch.randperm(2 * n_logical, generator=g).to(torch.int32).to(dev)
    cache = ops.PagedKvCache(arena=torch.full((2 * n_logical * 64 * widths[1],), 255, dtype=torch.uint8, device=dev),
                             block_table=table, n_layers=1, n_logical_blocks=n_logical, block_size=16,
                             block_bytes=64 * widths[1], stride=widths[1], kv_dtype=dt)
    kw_norm = dict(head_dim=hd, pairing=1)
    dims = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    def step(rows, at, rope_at, seqs):
        q, k, v = torch.split(torch.randn(rows, sum(widths), generator=g).to(dt).to(dev), widths, 1)
        k_out = torch.empty(rows, widths[1], dtype=dt, device=dev)
        flag = i32([0])
        q = ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, i32(at), cache, rope_positions=i32(rope_at),
                                      sequences=i32(seqs), k_out=k_out, err_flag=flag, **kw_norm)
        assert int(flag) == 0
        return q, k_out, v

    # the prompts
    seqs = [b for b, n in enumerate(lens) for _ in range(n)]
    at = [i for n in lens for i in range(n)]
    q, k, v = step(sum(lens), at, at, seqs)
    out = ops.prompt_attention(q, k, v, i32([0, lens[0], sum(lens)]), **dims)

    # the trees: node i of a sequence of n tokens stands at slot n + i and position n + depth
    depth, bits, flat = [], [], []
    for p in PARENTS:
        d, b = [], torch.eye(len(p), dtype=torch.bool)
        for i, parent in enumerate(p):
            d.append(0 if parent < 0 else d[parent] + 1)
            if parent >= 0:
                b[i] |= b[parent]
        depth.append(d)
        bits.append(b)
        flat += [sum(1 << j for j in range(len(p)) if b[i, j]) for i in range(len(p))]
    slots = [lens[b] + i for b, n in enumerate(nodes) for i in range(n)]
    places = [lens[b] + d for b, ds in enumerate(depth) for d in ds]
    tq, tk, tv = step(sum(nodes), slots, places, [b for b, n in enumerate(nodes) for _ in range(n)])
    got = ops.paged_tree_attention(tq, i32([0, nodes[0], sum(nodes)]), i32(lens), cache, tree_mask=i32(flat)[:, None],
                                   max_nodes=max(nodes), max_prefix=max(lens), **dims)
    # a new token without siblings: the decode path's own attention
    one = ops.paged_attention(tq[[0, nodes[0]]].contiguous(), i32([n + 1 for n in lens]), cache, max_seq=n_logical * 16,
                              **dims)

    p0 = t0 = 0
    for b, (n, m) in enumerate(zip(lens, nodes)):
        heads_of = lambda x, h: x.cpu().reshape(x.shape[0], h, hd)  # noqa: E731
        pk, pv = heads_of(k[p0:p0 + n], kv_heads), heads_of(v[p0:p0 + n], kv_heads)
        want, tol = attend(heads_of(q[p0:p0 + n], heads), pk, pv, causal_mask(n, 0), p_floor=FLOOR[kind], out_dtype=dt)
        check(heads_of(out[p0:p0 + n], heads), want, tol, f"prompt {b}")
        ak = torch.cat([pk, heads_of(tk[t0:t0 + m], kv_heads)])
        av = torch.cat([pv, heads_of(tv[t0:t0 + m], kv_heads)])
        allow = torch.cat([torch.ones(m, n, dtype=torch.bool), bits[b]], 1)
        want, tol = attend(heads_of(tq[t0:t0 + m], heads), ak, av, allow, p_floor=FLOOR[kind], out_dtype=dt)
        check(heads_of(got[t0:t0 + m], heads), want, tol, f"tree {b}")
        check(heads_of(one[b:b + 1], heads), want[:1], tol[:1], f"decode {b}")
        p0, t0 = p0 + n, t0 + m


def test_chunks_give_the_prompt(dev):
    """A prompt in chunks over the cache and the whole prompt at once, both within
    their tolerance of the formula."""
    from fellm_amd import ops

    heads, kv_heads, hd, n = 8, 2, 128, 300
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h * hd, generator=g).bfloat16().to(dev) for h in (heads, kv_heads, kv_heads))
    stride = kv_heads * hd
    cache = ops.PagedKvCache(arena=torch.zeros(20 * 64 * stride, dtype=torch.uint8, device=dev),
                             block_table=torch.arange(19, -1, -1, dtype=torch.int32, device=dev), n_layers=1,
                             n_logical_blocks=20, block_size=16, block_bytes=64 * stride, stride=stride,
                             kv_dtype=torch.bfloat16)
    dims = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd)
    whole = ops.prompt_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device=dev), **dims)
    blocks = cache.arena.view(torch.bfloat16).view(20, 2, 16, stride)
    parts, at = [], 0
    for m in (100, 1, 150, 49):
        for i in range(at, at + m):
            blocks[19 - i // 16, 0, i % 16] = k[i]
            blocks[19 - i // 16, 1, i % 16] = v[i]
        parts.append(ops.paged_tree_attention(q[at:at + m], torch.tensor([0, m], dtype=torch.int32, device=dev),
                                              torch.tensor([at], dtype=torch.int32, device=dev), cache, max_nodes=m,
                                              max_prefix=at, **dims))
        at += m
    rows = [x.cpu().view(n, -1, hd) for x in (q, k, v)]
    want, tol = attend(*rows, causal_mask(n, 0), out_dtype=torch.bfloat16)
    for got in (whole, torch.cat(parts)):
        check(got.view(n, heads, hd), want, tol)
