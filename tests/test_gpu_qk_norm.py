"""Per-head norm + rotation (+ paged append) against the 64-bit formula.

Tolerance of an output y of a head with a = the larger magnitude of its
pair after the norm (y's own where it is not rotated):
  half a step of the output's type at y
  + a * (D / 2 + 16) * 2^-24: the roundings of the sum of squares (D products
    summed, halved by the square root) and of the few operations after it, and
    the polynomials' 7.3e-8 and the final angle's rounding (below 8 of those steps).
"""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attention_util import U32, check, half_step  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from fellm_amd import ops as _ops

    return _ops


def expected(x, w, eps, inv, pos, hd, rope_dim, pairing, out_dtype):
    """(y, tolerance) f64 [rows, width]."""
    y = x.double().view(x.shape[0], -1, hd)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    mag = y.abs()
    ang = (pos.double()[:, None] * inv.double()[None, :])[:, None, :]
    c, s = torch.cos(ang), torch.sin(ang)
    h = rope_dim // 2
    if pairing == 1:
        a, b = slice(0, h), slice(h, rope_dim)
    else:
        lo = hd - rope_dim if pairing == 2 else 0
        a, b = slice(lo, lo + rope_dim, 2), slice(lo + 1, lo + rope_dim, 2)
    out, m2 = y.clone(), mag.clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., a] * s + y[..., b] * c
    m2[..., a] = m2[..., b] = torch.maximum(mag[..., a], mag[..., b])
    f = torch.finfo(out_dtype)
    tol = half_step(out_dtype) * out.abs() + m2 * (hd / 2 + 16) * U32 + f.smallest_normal * f.eps
    return out.flatten(1), tol.flatten(1)


def inv_freqs(rope_dim, theta=1e6):
    i = torch.arange(max(rope_dim // 2, 1), dtype=torch.float64)
    return (theta ** (-2 * i / max(rope_dim, 1))).float()


def inputs(rows, nq, nk, hd, act, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (2 * torch.randn(rows, n * hd, generator=g) for n in (nq, nk, nk))
    q[:, 3::hd] *= 20
    qw, kw = (1 + 0.3 * torch.randn(hd, generator=g) for _ in range(2))
    pos = torch.randint(0, 200000, (rows,), generator=g, dtype=torch.int32)
    return [x.to(DT[act]) for x in (q, k, v)], qw, kw, pos


def run_check(ops, dev, rows, nq, nk, hd, rope_dim, pairing, act, seed=0, eps=1e-6):
    (q, k, _), qw, kw, pos = inputs(rows, nq, nk, hd, act, seed)
    inv = inv_freqs(rope_dim)
    gq, gk = ops.qk_norm_rope(q.to(dev), k.to(dev), qw.to(dev), kw.to(dev), eps, inv.to(dev), head_dim=hd,
                              rope_dim=rope_dim, pairing=pairing, positions=pos.to(dev))
    for got, x, w in ((gq, q, qw), (gk, k, kw)):
        check(got, *expected(x, w, eps, inv[:rope_dim // 2], pos, hd, rope_dim, pairing, DT[act]))


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairing", [0, 1, 2])
@pytest.mark.parametrize("hd,rope_dim", [(64, 64), (128, 128), (256, 256), (128, 64), (64, 32), (96, 96), (80, 32),
                                         (112, 112), (512, 128), (16, 16)])
def test_head_sizes(ops, dev, act, pairing, hd, rope_dim):
    run_check(ops, dev, 5, 6, 2, hd, rope_dim, pairing, act, hd)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairing", [0, 1, 2])
@pytest.mark.parametrize("hd,rope_dim", [(2, 2), (6, 4), (40, 24), (100, 50), (130, 130), (128, 0), (1024, 1024),
                                         (72, 36), (1536, 64)])
def test_odd_head_sizes(ops, dev, act, pairing, hd, rope_dim):
    run_check(ops, dev, 3, 3, 1, hd, rope_dim, pairing, act, hd)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 255, 257, 2047, 2049, 2051])
@pytest.mark.parametrize("nq,nk,hd", [(32, 4, 128), (7, 1, 64), (1, 1, 256)])
def test_rows(ops, dev, rows, nq, nk, hd):
    run_check(ops, dev, rows, nq, nk, hd, hd, 1, "bf16", rows)


def test_far_positions(ops, dev):
    """Angles of positions up to 2^31 hold the exact product."""
    hd = 128
    pos = torch.tensor([0, 1, 131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1], dtype=torch.int32)
    x = torch.randn(6, 2 * hd, generator=torch.Generator().manual_seed(1))
    one, inv = torch.ones(hd), inv_freqs(hd)
    got, _ = ops.qk_norm_rope(x.to(dev), x.to(dev), one.to(dev), one.to(dev), 1e-5, inv.to(dev), head_dim=hd,
                              pairing=1, positions=pos.to(dev))
    check(got, *expected(x, one, 1e-5, inv, pos, hd, hd, 1, torch.float32))


def test_position0_strides_and_in_place(ops, dev):
    (q, k, v), qw, kw, _ = inputs(37, 8, 2, 128, "f16", 4)
    proj = torch.cat([q, k, v], 1).to(dev)
    inv = inv_freqs(128).to(dev)
    qv, kv, vv = torch.split(proj, [1024, 256, 256], 1)
    args = (qw.to(dev), kw.to(dev), 1e-6, inv)
    want = ops.qk_norm_rope(q.to(dev), k.to(dev), *args, head_dim=128, pairing=1,
                            positions=torch.arange(9, 46, dtype=torch.int32, device=dev))
    got = ops.qk_norm_rope(qv, kv, *args, head_dim=128, pairing=1, position0=9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ops.qk_norm_rope(qv, kv, *args, head_dim=128, pairing=1, position0=9, inplace=True)
    assert torch.equal(qv, want[0]) and torch.equal(kv, want[1]) and torch.equal(vv, v.to(dev))
    # rows that no 16-byte access fits: an odd column offset
    odd = torch.zeros(37, 1536 + 3, dtype=torch.float16, device=dev)
    odd[:, 3:] = torch.cat([q, k, v], 1).to(dev)
    qv, kv, _ = torch.split(odd[:, 3:], [1024, 256, 256], 1)
    ref = [expected(x, w, 1e-6, inv.cpu(), torch.arange(9, 46), 128, 128, 1, torch.float16) for x, w in ((q, qw), (k, kw))]
    got = ops.qk_norm_rope(qv, kv, *args, head_dim=128, pairing=1, position0=9)
    for g, (want, tol) in zip(got, ref):
        check(g, want, tol)
    ops.qk_norm_rope(qv, kv, *args, head_dim=128, pairing=1, position0=9, inplace=True)
    assert torch.equal(qv, got[0]) and torch.equal(kv, got[1])


def make_cache(ops, dev, rows, n_logical, stride, kv, blocks, seed=0, n_layers=1):
    g = torch.Generator().manual_seed(seed)
    arena = torch.randn(blocks, 2, 16, stride, generator=g).to(DT[kv])
    table = torch.randperm(blocks, generator=g)[:rows * n_layers * n_logical].to(torch.int32)
    return ops.PagedKvCache(arena=arena.view(torch.uint8).flatten().to(dev), block_table=table.to(dev), n_layers=n_layers,
                            n_logical_blocks=n_logical, block_size=16, block_bytes=64 * stride, stride=stride,
                            kv_dtype=DT[kv])


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,hd,rope_dim,pairing", [(8, 2, 128, 128, 1), (4, 4, 64, 32, 0), (3, 1, 256, 256, 2),
                                                       (3, 1, 20, 12, 1)])
@pytest.mark.parametrize("shared", [False, True])
def test_append(ops, dev, act, kv, nq, nk, hd, rope_dim, pairing, shared):
    """shared: a prompt's rows on the sequences' table rows; else a decode batch."""
    rows = 21
    (q, k, v), qw, kw, pos = inputs(rows, nq, nk, hd, act, 3)
    seqs = torch.tensor([0] * 12 + [2] * 9, dtype=torch.int32) if shared else torch.arange(rows, dtype=torch.int32)
    at = torch.cat([torch.arange(7, 19), torch.arange(30, 39)]).to(torch.int32) if shared else pos % 48
    cache = make_cache(ops, dev, 3 if shared else rows, 3, nk * hd, kv, 80)
    before = cache.arena.view(DT[kv]).view(-1, 2, 16, nk * hd).clone()
    inv = inv_freqs(rope_dim)
    k_out = torch.zeros(rows, nk * hd, dtype=DT[act], device=dev)
    flag = torch.zeros(1, dtype=torch.int32, device=dev)
    gq = ops.qk_norm_rope_kv_write(q.to(dev), k.to(dev), v.to(dev), qw.to(dev), kw.to(dev), 1e-6, inv.to(dev), at.to(dev),
                                   cache, head_dim=hd, rope_dim=rope_dim, pairing=pairing, rope_positions=pos.to(dev),
                                   sequences=seqs.to(dev) if shared else None, k_out=k_out, err_flag=flag)
    check(gq, *expected(q, qw, 1e-6, inv, pos, hd, rope_dim, pairing, DT[act]))
    check(k_out, *expected(k, kw, 1e-6, inv, pos, hd, rope_dim, pairing, DT[act]))
    after = cache.arena.view(DT[kv]).view(-1, 2, 16, nk * hd)
    phys = cache.block_table.view(-1, 3).cpu()[seqs.long(), at.long() // 16].long()
    check(after[phys, 0, at.long() % 16], *expected(k, kw, 1e-6, inv, pos, hd, rope_dim, pairing, DT[kv]))
    assert torch.equal(after[phys, 1, at.long() % 16].cpu(), v.to(DT[kv]))
    rest = torch.ones(before.shape[:3], dtype=torch.bool)
    rest[phys, :, at.long() % 16] = False
    assert torch.equal(after[rest.to(dev)], before[rest.to(dev)])
    assert int(flag) == 0


def test_slots_outside_the_cache_are_skipped(ops, dev):
    (q, k, v), qw, kw, _ = inputs(4, 4, 2, 64, "f16", 3)
    cache = make_cache(ops, dev, 4, 2, 128, "f16", 8)
    cache.block_table[7] = 1 << 20  # row 3, second block: outside the arena
    before = cache.arena.clone()
    at = torch.tensor([3, 32, 0x7fffffff, 20], dtype=torch.int32, device=dev)
    flag = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.qk_norm_rope_kv_write(q.to(dev), k.to(dev), v.to(dev), qw.to(dev), kw.to(dev), 1e-6, inv_freqs(64).to(dev), at,
                              cache, head_dim=64, err_flag=flag)
    assert int(flag) == 1
    changed = (cache.arena != before).view(8, 2, 16, 256).any(-1).nonzero().cpu().tolist()
    phys = int(cache.block_table[0])
    assert changed == [[phys, 0, 3], [phys, 1, 3]]


def test_graph(ops, dev):
    from fellm_amd import graph

    (q, k, v), qw, kw, pos = inputs(9, 8, 2, 128, "bf16")
    q, k, v, qw, kw, pos = (x.to(dev) for x in (q, k, v, qw, kw, pos % 32))
    cache = make_cache(ops, dev, 9, 2, 256, "bf16", 20)
    inv = inv_freqs(128).to(dev)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), graph.GraphCapture(stream) as cap:
        ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, pos, cache, head_dim=128, pairing=1, q_out=out)
    for i in range(3):
        pos.copy_((pos + i) % 32)
        clean = cache.arena.clone()
        want = ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, pos, cache, head_dim=128, pairing=1)
        arena = cache.arena.clone()
        cache.arena.copy_(clean)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cap.graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache.arena, arena)


def test_empty(ops, dev):
    (q, k, v), qw, kw, pos = inputs(4, 4, 2, 64, "f16")
    q, k, v, qw, kw, pos = (x.to(dev) for x in (q, k, v, qw, kw, pos))
    got = ops.qk_norm_rope(q[:0], k[:0], qw, kw, 1e-6, inv_freqs(64).to(dev), head_dim=64)
    assert got[0].shape == (0, 256) and got[1].shape == (0, 128)
    cache = make_cache(ops, dev, 4, 2, 128, "f16", 8)
    before = cache.arena.clone()
    ops.qk_norm_rope_kv_write(q[:0], k[:0], v[:0], qw, kw, 1e-6, inv_freqs(64).to(dev), pos[:0], cache, head_dim=64)
    assert torch.equal(cache.arena, before)


def test_many_rows_of_any_size(ops, dev):
    """The element-wise kernel and the vector kernel over more workgroups than fit at once."""
    run_check(ops, dev, 5003, 3, 1, 34, 20, 1, "f32")
    run_check(ops, dev, 9001, 3, 1, 64, 64, 0, "f32")


def test_refusals(ops, dev):
    from fellm_amd import FellmRocmError

    (q, k, v), qw, kw, pos = inputs(4, 4, 2, 64, "f16")
    q, k, v, qw, kw, pos = (x.to(dev) for x in (q, k, v, qw, kw, pos))
    inv = inv_freqs(64).to(dev)
    with pytest.raises(FellmRocmError):
        ops.qk_norm_rope(q, k, qw, kw, 1e-6, inv, head_dim=64, pairing=3)
    with pytest.raises(FellmRocmError):
        ops.qk_norm_rope(q, k, qw, kw, 1e-6, inv, head_dim=64, rope_dim=31)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k[:3], qw, kw, 1e-6, inv, head_dim=64)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw[:32], kw, 1e-6, inv, head_dim=64)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, k, qw.half(), kw, 1e-6, inv, head_dim=64)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw, kw, 1e-6, inv[:8], head_dim=64)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw, kw, 1e-6, inv, head_dim=64, positions=pos[:2])
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, qw, kw, 1e-6, inv, head_dim=64, q_out=torch.empty_like(k))
    cache = make_cache(ops, dev, 4, 2, 64, "f16", 8)
    with pytest.raises(FellmRocmError):  # a cache of one head for k of two
        ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, pos, cache, head_dim=64)
    cache = make_cache(ops, dev, 4, 2, 128, "f16", 8)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_kv_write(q, k, v[:, :64], qw, kw, 1e-6, inv, pos, cache, head_dim=64)
    with pytest.raises(TypeError):
        ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, pos, cache, head_dim=64, sequences=pos.long())
    with pytest.raises(ValueError):
        ops.qk_norm_rope_kv_write(q, k, v, qw, kw, 1e-6, inv, pos[:3], cache, head_dim=64)
