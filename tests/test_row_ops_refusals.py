"""What the per-head norm and the row attention entry points refuse, before any
GPU work: these run where no GPU exists.  The pointers are never followed."""
from __future__ import annotations

import ctypes as C

import pytest

from fellm_amd import lib
from fellm_amd._lib import FellmRocmPagedKv

ARITY, SHAPE, DTYPE, OK = -1, -2, -10, 0
F32, F16, BF16, Q4K = 0, 1, 30, 12
P = 1 << 20  # an aligned address


def paged(**kw):
    f = dict(arena=P, arena_len=1 << 20, block_table=P, n_block_table=64, n_logical_blocks=8, n_layers=1, layer=0,
             block_size=16, block_bytes=64 * 256, stride=256, kv_dtype=F16)
    f.update(kw)
    return FellmRocmPagedKv(**f)


def dtypes():
    from fellm_amd.abi import DType

    return int(DType.F32), int(DType.F16), int(DType.BF16), int(DType.Q4K)


def test_codes():
    assert dtypes() == (F32, F16, BF16, Q4K)


def norm(**kw):
    a = dict(q=P, q_stride=1024, q_out=P + 65536, q_out_stride=1024, n_q=8, k=P, k_stride=256, k_out=P, k_out_stride=256,
             n_k=2, act=F16, rows=4, head_dim=128, rope_dim=128, pairing=1, qw=P, kw=P, eps=1e-6, inv=P, pos=None, pos0=0)
    a.update(kw)
    return lib().fellm_rocm_qk_norm_rope(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    ({"q": None}, ARITY), ({"q_out": None}, ARITY), ({"k": None}, ARITY), ({"k_out": None}, ARITY), ({"qw": None}, ARITY),
    ({"kw": None}, ARITY), ({"inv": None}, ARITY), ({"head_dim": 0}, SHAPE), ({"head_dim": 127}, SHAPE),
    ({"rope_dim": 130}, SHAPE), ({"rope_dim": 63}, SHAPE), ({"pairing": 3}, SHAPE), ({"n_q": 0}, SHAPE),
    ({"n_k": 0}, SHAPE), ({"q_stride": 1023}, SHAPE), ({"k_stride": 255}, SHAPE), ({"q_out_stride": 1000}, SHAPE),
    ({"k_out_stride": 128}, SHAPE), ({"q_out": P, "q_out_stride": 2048}, SHAPE), ({"act": Q4K}, DTYPE),
    ({"rows": 0, "q": None, "k": None}, OK)])
def test_norm_rope(kw, rc):
    assert norm(**kw) == rc


def norm_write(kv=None, **kw):
    a = dict(q=P, q_stride=1024, q_out=P + 65536, q_out_stride=1024, n_q=8, k=P, k_stride=256, k_out=None, v=P,
             v_stride=256, n_k=2, act=F16, rows=4, head_dim=128, rope_dim=128, pairing=1, qw=P, kw=P, eps=1e-6, inv=P,
             rope_pos=None, kv_pos=P, seqs=None)
    a.update(kw)
    return lib().fellm_rocm_qk_norm_rope_kv_write(*a.values(), C.byref(kv or paged()), None, None)


@pytest.mark.parametrize("kw,kv,rc", [
    ({"v": None}, {}, ARITY), ({"kv_pos": None}, {}, ARITY), ({"v_stride": 255}, {}, SHAPE), ({}, {"stride": 128}, SHAPE),
    ({}, {"arena": None}, SHAPE), ({}, {"block_bytes": 64 * 256 - 64}, SHAPE), ({}, {"layer": 1}, SHAPE),
    ({}, {"kv_dtype": F32}, DTYPE), ({"act": Q4K}, {}, DTYPE), ({"rows": 0, "v": None}, {}, OK)])
def test_norm_rope_kv_write(kw, kv, rc):
    assert norm_write(paged(**kv), **kw) == rc


def prompt(**kw):
    a = dict(q=P, q_stride=1024, k=P, k_stride=256, v=P, v_stride=256, out=P, dtype=BF16, cu=P, n_seqs=1, tokens=4,
             n_heads=8, n_kv=2, head_dim=128, scale=0.0, causal=1, window=0)
    a.update(kw)
    return lib().fellm_rocm_prompt_attention(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    ({"dtype": F32}, DTYPE), ({"dtype": Q4K}, DTYPE), ({"n_kv": 0}, SHAPE), ({"n_heads": 0}, SHAPE), ({"n_kv": 3}, SHAPE),
    ({"head_dim": 96}, SHAPE), ({"q": None}, ARITY), ({"k": None}, ARITY), ({"v": None}, ARITY), ({"out": None}, ARITY),
    ({"cu": None}, ARITY), ({"q_stride": 1016}, SHAPE), ({"k_stride": 248}, SHAPE), ({"v_stride": 260}, SHAPE),
    ({"k_stride": 1 << 27}, SHAPE), ({"q": P + 8}, SHAPE), ({"v": P + 2}, SHAPE), ({"out": P + 4}, SHAPE),
    ({"tokens": 1 << 31, "n_heads": 2, "q_stride": 1024}, SHAPE), ({"tokens": 0, "q": None}, OK),
    ({"n_seqs": 0, "cu": None}, OK)])
def test_prompt_attention(kw, rc):
    assert prompt(**kw) == rc


def tree(kv=None, **kw):
    a = dict(q=P, q_dtype=F16, out=P, out_dtype=F16, cu=P, prefix=P, n_seqs=2, tokens=6, mask=P, words=1, n_heads=8,
             n_kv=2, head_dim=128, max_nodes=4, max_prefix=100, scale=0.0, window=0)
    tail = [kw.pop("ws", None), kw.pop("ws_bytes", 0)]
    a.update(kw)
    return lib().fellm_rocm_paged_tree_attention(*a.values(), C.byref(kv or paged()), *tail, None)


@pytest.mark.parametrize("kw,kv,rc", [
    ({"head_dim": 80}, {}, SHAPE), ({"n_kv": 0}, {}, SHAPE), ({"n_heads": 9}, {}, SHAPE), ({"q_dtype": Q4K}, {}, DTYPE),
    ({"out_dtype": BF16}, {}, DTYPE), ({"q_dtype": F32}, {}, DTYPE), ({}, {"kv_dtype": F32}, DTYPE), ({"q": None}, {}, ARITY),
    ({"cu": None}, {}, ARITY), ({"prefix": None}, {}, ARITY), ({}, {"arena": None}, ARITY), ({}, {"block_table": None}, ARITY),
    ({"mask": None}, {}, SHAPE), ({"words": 0}, {}, SHAPE), ({"window": 4}, {}, SHAPE), ({}, {"stride": 512}, SHAPE),
    ({}, {"block_size": 32}, SHAPE), ({}, {"block_bytes": 64 * 256 + 8}, SHAPE), ({}, {"layer": 2}, SHAPE),
    ({}, {"n_logical_blocks": 1 << 27}, SHAPE), ({"q": P + 8}, {}, SHAPE), ({}, {"arena": P + 8}, SHAPE),
    ({"ws": P + 4, "ws_bytes": 1 << 20}, {}, SHAPE), ({"tokens": 1 << 30}, {}, SHAPE), ({"tokens": 0, "q": None}, {}, OK),
    ({"n_seqs": 0}, {}, OK)])
def test_tree_attention(kw, kv, rc):
    assert tree(paged(**kv), **kw) == rc


def test_tree_workspace():
    ws = lib().fellm_rocm_paged_tree_attention_workspace
    assert ws(0, 0, 8, 2, 128, 4, 100) == 0
    assert ws(1, 8, 8, 2, 96, 8, 100) == 0 and ws(1, 8, 8, 3, 128, 8, 100) == 0
    assert ws(1, 8, 32, 8, 128, 8, 5) <= ws(1, 8, 32, 8, 128, 8, 100000) < 1 << 30
    # bounds past every real size stay bounded: as many records as workgroups are resident
    assert ws(1000, 100000, 64, 8, 256, 0xffffffff, 0xffffffff) < 1 << 30
