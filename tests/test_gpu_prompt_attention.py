"""Prompt attention over packed sequences against the 64-bit formula
(tolerances: attention_util.attend)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from attention_util import attend, causal_mask, check  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
# f16: p is stored times 2^4 or more, its subnormal step is 2^-24
FLOOR = {"f16": 2.0 ** -29, "bf16": 0.0}


@pytest.fixture(scope="module")
def ops():
    from fellm_amd import ops as _ops

    return _ops


def make(lens, heads, kv_heads, hd, kind, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    t = sum(lens) + extra
    q, k, v = (torch.randn(t, n * hd, generator=g).to(DT[kind]) for n in (heads, kv_heads, kv_heads))
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    return q * 1.5, k, v, cu


def reference(q, k, v, lens, heads, kv_heads, hd, kind, mask, scale=None):
    """[(out, tol)] of each sequence; mask(n) -> bool [n, n]."""
    res, at = [], 0
    for n in lens:
        if n:
            part = [x[at:at + n].view(n, h, hd) for x, h in ((q, heads), (k, kv_heads), (v, kv_heads))]
            res.append((at, n, *attend(*part, mask(n), scale, p_floor=FLOOR[kind], out_dtype=DT[kind])))
        at += n
    return res


def run_check(ops, dev, lens, heads, kv_heads, hd, kind, *, causal=True, window=0, scale=0.0, seed=0):
    q, k, v, cu = make(lens, heads, kv_heads, hd, kind, seed)
    got = ops.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), n_heads=heads, n_kv_heads=kv_heads,
                               head_dim=hd, causal=causal, window=window, scale=scale)

    def mask(n):
        if causal:
            return causal_mask(n, 0, window)
        i = torch.arange(n)
        return (i[:, None] - i[None, :]).abs() < (window or n + 1)

    for at, n, want, tol in reference(q, k, v, lens, heads, kv_heads, hd, kind, mask, scale or None):
        check(got[at:at + n].view(n, heads, hd), want, tol, f"sequence at {at}")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 64), (8, 8, 64), (8, 2, 128), (7, 1, 128), (28, 4, 128),
                                               (16, 1, 128), (4, 2, 256), (40, 1, 64), (5, 5, 256)])
def test_heads(ops, dev, heads, kv_heads, hd, kind):
    run_check(ops, dev, [1, 17, 64, 130], heads, kv_heads, hd, kind)


@pytest.mark.parametrize("lens", [[1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [300],
                                  [0, 5, 0, 0, 70, 1, 0], [1] * 130, [700, 3]])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (7, 1, 64)])
def test_lengths(ops, dev, lens, heads, kv_heads, hd):
    run_check(ops, dev, lens, heads, kv_heads, hd, "bf16", seed=len(lens))


@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 1000])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_windows(ops, dev, window, causal, hd):
    run_check(ops, dev, [1, 200, 333], 4, 2, hd, "f16", causal=causal, window=window)


def test_all_keys(ops, dev):
    run_check(ops, dev, [1, 77, 260], 4, 1, 128, "bf16", causal=False)


def test_scale(ops, dev):
    run_check(ops, dev, [150], 4, 1, 128, "f16", scale=0.31)


def test_scores_that_rise_and_fall(ops, dev):
    """Maxima that grow tile by tile, and by less and more than the lazy step."""
    hd, n = 128, 400
    q, k, v, cu = make([n], 2, 1, hd, "bf16", 3)
    k = (k.float() * torch.linspace(0.1, 3.0, n)[:, None]).bfloat16()
    for kk in (k, k.flip(0)):
        got = ops.prompt_attention(q.to(dev), kk.to(dev), v.to(dev), cu.to(dev), n_heads=2, n_kv_heads=1, head_dim=hd)
        (_, _, want, tol), = reference(q, kk, v, [n], 2, 1, hd, "bf16", lambda m: causal_mask(m, 0))
        check(got.view(n, 2, hd), want, tol)


def test_strided_rows_and_untouched_tail(ops, dev):
    lens, heads, kv_heads, hd = [50, 81], 8, 2, 128
    g = torch.Generator().manual_seed(5)
    t = sum(lens)
    widths = [heads * hd, kv_heads * hd, kv_heads * hd]
    proj = torch.randn(t + 9, sum(widths), generator=g).half().to(dev)
    q, k, v = torch.split(proj, widths, 1)
    cu = torch.tensor([0, 50, 131], dtype=torch.int32, device=dev)
    out = torch.full((t + 9, heads * hd), 7.0, dtype=torch.float16, device=dev)
    ops.prompt_attention(q, k, v, cu, n_heads=heads, n_kv_heads=kv_heads, head_dim=hd, out=out)
    assert (out[t:] == 7.0).all()
    dense = ops.prompt_attention(q[:t].contiguous(), k[:t].contiguous(), v[:t].contiguous(), cu, n_heads=heads,
                                 n_kv_heads=kv_heads, head_dim=hd)
    assert torch.equal(out[:t], dense)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), "max"])
def test_masked_values_do_not_count(ops, dev, kind, value):
    """Keys and values that a row does not attend may hold anything."""
    lens, heads, kv_heads, hd = [40, 90], 4, 2, 128
    q, k, v, cu = make(lens, heads, kv_heads, hd, kind, 8, extra=20)
    clean = ops.prompt_attention(*(x.to(dev) for x in (q, k, v, cu)), n_heads=heads, n_kv_heads=kv_heads, head_dim=hd)
    value = torch.finfo(DT[kind]).max if value == "max" else value
    k2, v2 = k.clone(), v.clone()
    for x in (k2, v2):
        x[100:] = value  # the end of sequence 1 and the rows of none
        x[39] = value    # the last token of sequence 0
    got = ops.prompt_attention(*(x.to(dev) for x in (q, k2, v2, cu)), n_heads=heads, n_kv_heads=kv_heads, head_dim=hd)
    # rows that attend none of them, within the tolerance of both
    ref = reference(q, k, v, lens, heads, kv_heads, hd, kind, lambda m: causal_mask(m, 0))
    for (at, n, want, tol), m in zip(ref, (39, 60)):
        check(got[at:at + m].view(m, heads, hd), want[:m], tol[:m])
        check(clean[at:at + m].view(m, heads, hd), want[:m], tol[:m])


def test_attended_infinite_value(ops, dev):
    n, heads, hd = 100, 2, 64
    q, k, v, cu = make([n], heads, 1, hd, "bf16", 2)
    v[30, 5] = float("inf")
    v[60, 9] = float("nan")
    got = ops.prompt_attention(*(x.to(dev) for x in (q, k, v, cu)), n_heads=heads, n_kv_heads=1, head_dim=hd)
    got = got.view(n, heads, hd).float().cpu()
    assert torch.isfinite(got[:30]).all()
    assert (got[30:, :, 5] == float("inf")).all() and torch.isnan(got[60:, :, 9]).all()
    fine = torch.ones(hd, dtype=torch.bool)
    fine[[5, 9]] = False
    assert torch.isfinite(got[..., fine]).all() and torch.isfinite(got[:60, :, 9]).all()
    v2 = v.clone()
    v2[30, 5] = v2[60, 9] = 0
    (_, _, want, tol), = reference(q, k, v2, [n], heads, 1, hd, "bf16", lambda m: causal_mask(m, 0))
    check(got[..., fine], want[..., fine], tol[..., fine])


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_all_are_nan(ops, dev, hd):
    q, k, v, cu = make([300], 4, 2, hd, "bf16", 6)
    v[:] = float("nan")
    v[:, 1] = 2.0
    got = ops.prompt_attention(*(x.to(dev) for x in (q, k, v, cu)), n_heads=4, n_kv_heads=2, head_dim=hd)
    got = got.view(300, 4, hd)
    assert torch.isnan(got[:, 2:]).all() and torch.isnan(got[:, :2, 2:]).all()
    # two: the sums carry n roundings of p and the quotient one of the output
    assert (got[:, :2, 1] - 2.0).abs().max() <= 2 * (2.0 ** -8 + 300 * 2.0 ** -23)


def test_offsets_past_32_bits(ops, dev):
    """Rows 65600 elements apart: the last sequence starts past 4 GiB."""
    stride, t, hd = 65600, 34000, 64
    g = torch.Generator(device=dev).manual_seed(1)
    big = torch.empty(t, stride, dtype=torch.bfloat16, device=dev)
    big[:, :3 * hd] = torch.randn(t, 3 * hd, generator=g, device=dev).bfloat16()
    q, k, v = (big[:, i * hd:(i + 1) * hd] for i in range(3))
    cu = torch.tensor([0, t - 150, t], dtype=torch.int32, device=dev)
    got = ops.prompt_attention(q, k, v, cu, n_heads=1, n_kv_heads=1, head_dim=hd, window=40)
    tail = [x[-150:].cpu().contiguous().view(150, 1, hd) for x in (q, k, v)]
    want, tol = attend(*tail, causal_mask(150, 0, 40), out_dtype=torch.bfloat16)
    check(got[-150:].view(150, 1, hd), want, tol)
    head = [x[:150].cpu().contiguous().view(150, 1, hd) for x in (q, k, v)]
    want, tol = attend(*head, causal_mask(150, 0, 40), out_dtype=torch.bfloat16)
    check(got[:150].view(150, 1, hd), want, tol)


def test_other_stream_and_graph(ops, dev):
    from fellm_amd import graph

    lens, heads, kv_heads, hd = [90, 33], 8, 2, 128
    q, k, v, cu = (x.to(dev) for x in make(lens, heads, kv_heads, hd, "bf16", 4))
    kw = dict(n_heads=heads, n_kv_heads=kv_heads, head_dim=hd)
    want = ops.prompt_attention(q, k, v, cu, **kw)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), graph.GraphCapture(stream) as cap:
        ops.prompt_attention(q, k, v, cu, out=out, **kw)
    for i in range(3):
        q2 = q * (1 + i)
        want = ops.prompt_attention(q2, k, v, cu, **kw)
        keep = q.clone()
        q.copy_(q2)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cap.graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        q.copy_(keep)


def test_lengths_past_the_tokens_stay_inside(ops, dev):
    """Offsets that decrease or pass the rows are cut, not followed."""
    q, k, v, _ = (x.to(dev) for x in make([64], 4, 2, 64, "f16", 1))
    out = torch.zeros(64, 256, dtype=torch.float16, device=dev)
    for cu in ([0, 40, 30, 200], [50, 10, 64], [100, 200]):
        ops.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=dev), n_heads=4, n_kv_heads=2,
                             head_dim=64, out=out)
    assert torch.isfinite(out).all()


def test_empty(ops, dev):
    q, k, v, _ = (x.to(dev) for x in make([4], 4, 2, 64, "f16"))
    out = torch.full_like(q, 3)
    ops.prompt_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=dev), n_heads=4, n_kv_heads=2, head_dim=64,
                         out=out)
    assert (out == 3).all()
    e = q[:0]
    assert ops.prompt_attention(e, k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=dev), n_heads=4, n_kv_heads=2,
                                head_dim=64).shape == (0, 256)


def test_refusals(ops, dev):
    from fellm_amd import FellmRocmError

    q, k, v, cu = (x.to(dev) for x in make([8], 4, 2, 64, "f16"))
    kw = dict(n_heads=4, n_kv_heads=2, head_dim=64)
    with pytest.raises(FellmRocmError):
        ops.prompt_attention(q.float(), k.float(), v.float(), cu, **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k, v[:4], cu, **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k.bfloat16(), v, cu, **kw)
    with pytest.raises(TypeError):
        ops.prompt_attention(q, k, v, cu.long(), **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k[:, :64], v, cu, **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k, v, cu, out=torch.empty(8, 128, dtype=torch.float16, device=dev), **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k, v, cu.cpu(), **kw)
    with pytest.raises(ValueError):  # every second column
        ops.prompt_attention(torch.empty(8, 512, dtype=torch.float16, device=dev)[:, ::2], k, v, cu, **kw)
    with pytest.raises(ValueError):  # one row for all
        ops.prompt_attention(q[:1].expand(8, 256), k, v, cu, **kw)
