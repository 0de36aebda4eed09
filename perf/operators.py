"""Performance cases of the operators around a prompt and a drafted tree.

Three kinds of call:

  norm    RMSNorm of every query and key head with the rotation in the same
          pass; with a cache, the rotated k and v are appended to it
  prompt  causal attention over packed whole prompts with grouped heads
  tree    attention of several new tokens a sequence over the paged cache: a
          drafted tree given by ancestor bits, or a chunk of a prompt

Each is computed in its plain form (elementary torch operations in 32 bits)
or, with ``own``, by the calls a user of ``fellm_amd.ops`` makes.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 16  # tokens per cache block
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # One decoded token at Qwen3-30B-A3B heads: launch latency.
        {"name": "norm_write_b1", "kind": "norm", "rows": 1, "seqs": 1, "heads": 32, "kv_heads": 4, "head_dim": 128,
         "rope_dim": 128, "pairing": 1, "act": "bf16", "kv": "bf16", "max_pos": 32768, "fused": True},
        # A serving step of 256 sequences with f32 activations and the f16 cache.
        {"name": "norm_write_b256_f32", "kind": "norm", "rows": 256, "seqs": 256, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "rope_dim": 128, "pairing": 1, "act": "f32", "kv": "f16", "max_pos": 32768, "fused": False},
        # Five prompts' chunks, an odd row count, half of a head of 64 rotated, adjacent pairs.
        {"name": "norm_write_t1999_partial", "kind": "norm", "rows": 1999, "seqs": 5, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "rope_dim": 32, "pairing": 0, "act": "f16", "kv": "f16", "max_pos": 4096, "fused": True},
        # Prefill of 16384 tokens at Qwen3-30B-A3B heads, out of one fused projection.
        {"name": "norm_t16384", "kind": "norm", "rows": 16384, "seqs": 1, "heads": 32, "kv_heads": 4, "head_dim": 128,
         "rope_dim": 128, "pairing": 1, "act": "bf16", "kv": "", "max_pos": 16384, "fused": True},
        # One short prompt at Llama-3.2-1B heads: latency.
        {"name": "prompt_1b_t64", "kind": "prompt", "seqs": 1, "max_len": 64, "mix": 0, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "act": "f16", "window": 0, "fused": True},
        # A ragged batch of 17 prompts of up to 2048 tokens at Qwen2-7B heads (seven query heads a K/V head).
        {"name": "prompt_7b_ragged17", "kind": "prompt", "seqs": 17, "max_len": 2048, "mix": 1, "heads": 28,
         "kv_heads": 4, "head_dim": 128, "act": "f16", "window": 0, "fused": True},
        # One prompt of 4096 tokens at Llama-3-8B heads.
        {"name": "prompt_8b_t4096", "kind": "prompt", "seqs": 1, "max_len": 4096, "mix": 0, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "act": "bf16", "window": 0, "fused": True},
        # One long prompt at Qwen3-30B-A3B heads.
        {"name": "prompt_30b_t16384", "kind": "prompt", "seqs": 1, "max_len": 16384, "mix": 0, "heads": 32,
         "kv_heads": 4, "head_dim": 128, "act": "bf16", "window": 0, "fused": False},
        # A tree of eight drafted tokens for one sequence behind 2047 keys: latency.
        {"name": "tree_8b_b1_n8", "kind": "tree", "seqs": 1, "nodes": 8, "prefix": 2047, "mix": 0, "chain": False,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "f16", "kv": "f16", "window": 0},
        # f32 activations over the f16 cache, ragged trees of up to 63 tokens at Qwen2-7B heads.
        {"name": "tree_7b_b8_n63_f32", "kind": "tree", "seqs": 8, "nodes": 63, "prefix": 4000, "mix": 2,
         "chain": False, "heads": 28, "kv_heads": 4, "head_dim": 128, "act": "f32", "kv": "f16", "window": 0},
        # A serving batch of 32 sequences of up to 8192 keys verifying trees of up to 32 tokens, Llama-3-70B heads.
        {"name": "tree_70b_b32_n32", "kind": "tree", "seqs": 32, "nodes": 32, "prefix": 8192, "mix": 3, "chain": False,
         "heads": 64, "kv_heads": 8, "head_dim": 128, "act": "bf16", "kv": "bf16", "window": 0},
        # A chunk of 512 prompt tokens behind a cached prefix of 32256, Llama-3-8B heads.
        {"name": "chunk_8b_n512_s32256", "kind": "tree", "seqs": 1, "nodes": 512, "prefix": 32256, "mix": 0,
         "chain": True, "heads": 32, "kv_heads": 8, "head_dim": 128, "act": "bf16", "kv": "bf16", "window": 0},
    ]


# ------------------------------------------------------------------------------ draws
HEADS = [(32, 8, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (32, 4, 128), (16, 4, 256), (16, 16, 64), (8, 1, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(["norm", "prompt", "tree"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    if kind == "norm":
        rows = _log(rng, 1, 16384)
        kv = rng.choice(["", "f16", "bf16"])
        seqs = rng.choice([1, min(rows, 7), rows]) if kv and rows <= 512 else min(rows, rng.randint(1, 9))
        return {**c, "rows": rows, "seqs": seqs, "rope_dim": head_dim // rng.choice([1, 1, 2]),
                "pairing": rng.choice([0, 1, 1, 2]), "act": rng.choice(["f32", "f16", "bf16"]), "kv": kv,
                "max_pos": rng.choice([16384, 32768, 131072]), "fused": rng.random() < 0.5}
    if kind == "prompt":
        return {**c, "seqs": _log(rng, 1, 32), "max_len": _log(rng, 1, 16384), "mix": rng.randint(1, 10 ** 6),
                "act": rng.choice(["f16", "bf16"]), "window": rng.choice([0, 0, 0, 1024]), "fused": rng.random() < 0.5}
    kv = rng.choice(["f16", "bf16"])
    chain = rng.random() < 0.3
    return {**c, "seqs": _log(rng, 1, 32), "nodes": _log(rng, 1, 512 if chain else 64), "prefix": _log(rng, 1, 32768),
            "mix": rng.randint(1, 10 ** 6), "chain": chain, "act": rng.choice([kv, kv, "f32"]), "kv": kv,
            "window": rng.choice([0, 0, 1024]) if chain else 0}


def draw(rng):
    top = [work(c) for c in listed()]
    most_bytes, most_flops = max(w["bytes"] for w in top), max(w["flops"] for w in top)
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return c


# ------------------------------------------------------------------- lengths and trees
def _lengths(n, longest, mix):
    """n lengths, the first the longest, the others log-uniform; mix 0: all the longest."""
    rng = random.Random(mix)
    return [longest if i == 0 or not mix else _log(rng, max(longest // 16, 1), longest) for i in range(n)]


def _tree_sizes(c):
    return _lengths(c["seqs"], c["nodes"], c["mix"]), _lengths(c["seqs"], c["prefix"], c["mix"] and c["mix"] + 1)


def _tree_bits(c):
    """For each sequence, each node's ancestors and itself as the bits of an int.  Half of the
    nodes continue the node before them, the others branch from any earlier one."""
    rng = random.Random(c["mix"] + 17)
    out = []
    for n in _tree_sizes(c)[0]:
        bits = []
        for i in range(n):
            parent = i - 1 if rng.random() < 0.5 else rng.randint(0, max(i - 1, 0))
            bits.append((bits[parent] if i else 0) | 1 << i)
        out.append(bits)
    return out


def _pairs(n, before, window):
    """Attended (row, key) pairs of n causal rows behind `before` keys."""
    if not window:
        return n * before + n * (n + 1) // 2
    return sum(min(before + i + 1, window) for i in range(n))


def work(case):
    c = case
    hq, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "norm":
        s, t = SIZE[c["act"]], c["rows"] * d
        moved = t * (2 * hq + 2 * hk) * s if not c["kv"] else t * ((2 * hq + 2 * hk) * s + 2 * hk * 2)
        return {"bytes": moved + 8 * d + 4 * c["rows"], "flops": 8 * t * (hq + hk)}
    if c["kind"] == "prompt":
        lens = _lengths(c["seqs"], c["max_len"], c["mix"])
        return {"bytes": sum(lens) * d * (2 * hq + 2 * hk) * SIZE[c["act"]],
                "flops": 4 * d * hq * sum(_pairs(n, 0, c["window"]) for n in lens)}
    nodes, prefix = _tree_sizes(c)
    w = c["window"]
    keys = sum(n + (min(p, max(w - 1, 0)) if w else p) for n, p in zip(nodes, prefix))
    if c["chain"]:
        pairs = sum(_pairs(n, p, w) for n, p in zip(nodes, prefix))
    else:
        pairs = sum(p * len(b) + sum(x.bit_count() for x in b) for p, b in zip(prefix, _tree_bits(c)))
    return {"bytes": keys * hk * d * 2 * 2 + sum(nodes) * hq * d * 2 * SIZE[c["act"]], "flops": 4 * d * hq * pairs}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _projection(g, rows, widths, dtype, fused):
    """q, k and v: column slices of one projection's output, or tensors of their own."""
    if fused:
        return list(torch.split(_randn(g, rows, sum(widths), dtype=dtype), widths, dim=1))
    return [_randn(g, rows, w, dtype=dtype) for w in widths]


def _prepare_norm(c, s, g, seed):
    d, rows = c["head_dim"], c["rows"]
    widths = [c["heads"] * d, c["kv_heads"] * d, c["kv_heads"] * d]
    s["q"], s["k"], s["v"] = _projection(g, rows, widths, DT[c["act"]], c["fused"])
    # a few channels much larger than the rest, as projections have them
    for t in (s["q"], s["k"]):
        t[:, 5::d] *= 8
    s["qw"], s["kw"] = (1.0 + 0.2 * _randn(g, d) for _ in range(2))
    half = c["rope_dim"] // 2
    s["inv"] = torch.tensor([THETA ** (-i / half) for i in range(half)], dtype=torch.float32, device="cuda")
    rng = random.Random(seed)
    share = [rows // c["seqs"] + (i < rows % c["seqs"]) for i in range(c["seqs"])]
    first = [rng.randint(0, c["max_pos"] - n) for n in share]
    seq_of = [b for b, n in enumerate(share) for _ in range(n)]
    pos = [p + i for p, n in zip(first, share) for i in range(n)]
    s["pos"], s["seq"] = _i32(pos), _i32(seq_of)
    if c["kv"]:
        stride, n_logical = widths[1], c["max_pos"] // BLOCK
        # every block that n tokens can touch from any start; other tokens' rows fill the blocks already
        blocks = sum(n // BLOCK + 2 for n in share)
        used = sorted({(b, p // BLOCK) for b, p in zip(seq_of, pos)})
        at = torch.tensor(used, device="cuda")
        s["table"] = torch.zeros(c["seqs"], n_logical, dtype=torch.int32, device="cuda")
        s["table"][at[:, 0], at[:, 1]] = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:len(used)]
        s["arena"] = _randn(g, blocks * 2 * BLOCK * stride, dtype=DT[c["kv"]]).view(torch.uint8)


def _prepare_prompt(c, s, g):
    lens = _lengths(c["seqs"], c["max_len"], c["mix"])
    d, t = c["head_dim"], sum(lens)
    widths = [c["heads"] * d, c["kv_heads"] * d, c["kv_heads"] * d]
    q, k, s["v"] = _projection(g, t, widths, DT[c["act"]], c["fused"])
    # normed and rotated q and k are tensors of their own, v stays a slice of the projection
    s["q"], s["k"] = (q * 1.5).contiguous(), k.contiguous()
    s["lens"], s["cu"] = lens, _i32(_offsets(lens))


def _prepare_tree(c, s, g):
    nodes, prefix = _tree_sizes(c)
    s["nodes"], s["prefix"] = nodes, prefix
    d, stride = c["head_dim"], c["kv_heads"] * c["head_dim"]
    need = [(p + n + BLOCK - 1) // BLOCK for n, p in zip(nodes, prefix)]
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(c["seqs"], max(need), dtype=torch.int32, device="cuda")
    table[torch.arange(max(need), device="cuda")[None, :] < _i32(need)[:, None]] = order
    s["table"], s["blocks"] = table, need
    s["arena"] = _randn(g, sum(need) * 2 * BLOCK * stride, dtype=DT[c["kv"]]).view(torch.uint8)
    s["q"] = _randn(g, sum(nodes), c["heads"] * d, std=1.5, dtype=DT[c["act"]])
    s["cu"], s["plen"] = _i32(_offsets(nodes)), _i32(prefix)
    s["mask"] = None
    if not c["chain"]:
        words = (max(nodes) + 31) // 32
        flat = [[(x >> 32 * w) & 0xffffffff for w in range(words)] for b in _tree_bits(c) for x in b]
        s["mask"] = torch.tensor([[x - (x >> 31 << 32) for x in row] for row in flat], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = dict(case)
    g, s = _gen(seed), {"c": c}
    if c["kind"] == "norm":
        _prepare_norm(c, s, g, seed)
    elif c["kind"] == "prompt":
        _prepare_prompt(c, s, g)
    else:
        _prepare_tree(c, s, g)
    return s


# --------------------------------------------------------------------------------- runs
def run(state):
    c = state["c"]
    return (_OWN if own else _PLAIN)[c["kind"]](c, state)


def _cache(c, s):
    from fellm_amd import ops
    stride = c["kv_heads"] * c["head_dim"]
    return ops.PagedKvCache(arena=s["arena"], block_table=s["table"], n_layers=1, n_logical_blocks=s["table"].shape[1],
                            block_size=BLOCK, block_bytes=2 * BLOCK * stride * 2, stride=stride, kv_dtype=DT[c["kv"]])


def _own_norm(c, s):
    from fellm_amd import ops
    kw = {"head_dim": c["head_dim"], "rope_dim": c["rope_dim"], "pairing": c["pairing"]}
    if not c["kv"]:
        return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], EPS, s["inv"], positions=s["pos"], **kw)
    q = ops.qk_norm_rope_kv_write(s["q"], s["k"], s["v"], s["qw"], s["kw"], EPS, s["inv"], s["pos"], _cache(c, s),
                                  sequences=s["seq"], **kw)
    return [q, s["arena"].view(DT[c["kv"]])]


def _own_prompt(c, s):
    from fellm_amd import ops
    return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], n_heads=c["heads"], n_kv_heads=c["kv_heads"],
                                head_dim=c["head_dim"], window=c["window"])


def _own_tree(c, s):
    from fellm_amd import ops
    return ops.paged_tree_attention(s["q"], s["cu"], s["plen"], _cache(c, s), tree_mask=s["mask"], n_heads=c["heads"],
                                    n_kv_heads=c["kv_heads"], head_dim=c["head_dim"], max_nodes=c["nodes"],
                                    max_prefix=c["prefix"], window=c["window"])


def _rotated(c):
    """The first and the second members of every rotated pair of a head."""
    d, r, h = c["head_dim"], c["rope_dim"], c["rope_dim"] // 2
    if c["pairing"] == 1:
        return slice(0, h), slice(h, r)
    lo = d - r if c["pairing"] == 2 else 0
    return slice(lo, lo + r, 2), slice(lo + 1, lo + r, 2)


def _plain_head_rows(c, x, w, inv, pos):
    d = c["head_dim"]
    h = x.float().view(x.shape[0], -1, d)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w
    angle = pos.double()[:, None] * inv.double()[None, :]
    cos, sin = (f(angle).float()[:, None, :] for f in (torch.cos, torch.sin))
    a, b = _rotated(c)
    out = y.clone()
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., a] * sin + y[..., b] * cos
    return out.view(x.shape[0], -1)


def _plain_norm(c, s):
    q = _plain_head_rows(c, s["q"], s["qw"], s["inv"], s["pos"]).to(DT[c["act"]])
    k = _plain_head_rows(c, s["k"], s["kw"], s["inv"], s["pos"])
    if not c["kv"]:
        return q, k.to(DT[c["act"]])
    kv = s["arena"].view(DT[c["kv"]])
    blocks = kv.view(-1, 2, BLOCK, k.shape[1])
    pos = s["pos"].long()
    at = s["table"][s["seq"].long(), pos // BLOCK].long()
    blocks[at, 0, pos % BLOCK] = k.to(kv.dtype)
    blocks[at, 1, pos % BLOCK] = s["v"].to(kv.dtype)
    return [q, kv]


def _plain_attend(q, k, v, seen, scale):
    """q [R, G, hk, d], k and v [S, hk, d], seen(first row, rows) -> bool [rows, S]: f32 [R, G, hk, d]."""
    rows, g, hk, d = q.shape
    keys = k.shape[0]
    kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    out = torch.empty(rows, g, hk, d, device=q.device)
    step = max(1, min(rows, (1 << 28) // (g * hk * keys)))
    for r in range(0, rows, step):
        part = q[r:r + step]
        n = part.shape[0]
        sc = torch.matmul(part.permute(2, 0, 1, 3).reshape(hk, n * g, d), kt).view(hk, n, g, keys) * scale
        sc.masked_fill_(~seen(r, n)[None, :, None, :], -math.inf)
        sc = torch.exp(sc - sc.amax(-1, keepdim=True))
        sc = sc / sc.sum(-1, keepdim=True)
        out[r:r + n] = torch.matmul(sc.view(hk, n * g, keys), vt).view(hk, n, g, d).permute(1, 2, 0, 3)
    return out


def _causal(before, keys, window):
    """Row i stands at position before + i."""
    at = torch.arange(keys, device="cuda")

    def seen(r, n):
        me = before + r + torch.arange(n, device="cuda")[:, None]
        ok = at[None, :] <= me
        return ok & (at[None, :] > me - window) if window else ok

    return seen


def _heads_of(x, c):
    """[T, heads * d] -> f32 [T, G, hk, d]; query head h reads K/V head h // G."""
    hk, g = c["kv_heads"], c["heads"] // c["kv_heads"]
    return x.float().view(x.shape[0], hk, g, c["head_dim"]).transpose(1, 2)


def _plain_prompt(c, s):
    d = c["head_dim"]
    out = torch.empty_like(s["q"])
    at = 0
    for n in s["lens"]:
        q, k, v = (s[x][at:at + n] for x in "qkv")
        o = _plain_attend(_heads_of(q, c), k.float().view(n, -1, d), v.float().view(n, -1, d),
                          _causal(0, n, c["window"]), 1.0 / math.sqrt(d))
        out[at:at + n] = o.transpose(1, 2).reshape(n, -1).to(out.dtype)
        at += n
    return out


def _tree_keys(c, s, b):
    """K and V [S, hk, d] of sequence b, out of its pages."""
    stride = c["kv_heads"] * c["head_dim"]
    keys = s["prefix"][b] + s["nodes"][b]
    pages = s["arena"].view(DT[c["kv"]]).view(-1, 2, BLOCK, stride)[s["table"][b, :s["blocks"][b]].long()]
    return [pages[:, i].reshape(-1, c["kv_heads"], c["head_dim"])[:keys] for i in range(2)]


def _tree_seen(c, s, b, at):
    p, n = s["prefix"][b], s["nodes"][b]
    if s["mask"] is None:
        return _causal(p, p + n, c["window"])
    word = s["mask"][at:at + n].long()
    j = torch.arange(n, device="cuda")
    ok = (word[:, j // 32] >> (j % 32)[None, :]) & 1 != 0
    ok = torch.cat([torch.ones(n, p, dtype=torch.bool, device="cuda"), ok], 1)
    return lambda r, m: ok[r:r + m]


def _plain_tree(c, s):
    out = torch.empty_like(s["q"])
    at = 0
    for b, n in enumerate(s["nodes"]):
        k, v = (x.float() for x in _tree_keys(c, s, b))
        o = _plain_attend(_heads_of(s["q"][at:at + n], c), k, v, _tree_seen(c, s, b, at), 1.0 / math.sqrt(c["head_dim"]))
        out[at:at + n] = o.transpose(1, 2).reshape(n, -1).to(out.dtype)
        at += n
    return out


_OWN = {"norm": _own_norm, "prompt": _own_prompt, "tree": _own_tree}
_PLAIN = {"norm": _plain_norm, "prompt": _plain_prompt, "tree": _plain_tree}


# -------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["kind"] == "norm":
        return _exact_norm(c, s)
    if work(c)["flops"] > 3e12:
        return None
    d = c["head_dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(s["lens"] if c["kind"] == "prompt" else s["nodes"]):
        if c["kind"] == "prompt":
            before = 0
            k, v = (s[x][at:at + n].reshape(n, -1, d).double() for x in "kv")
        else:
            before = s["prefix"][b]
            k, v = (x.double() for x in _tree_keys(c, s, b))
        q = s["q"][at:at + n].double()
        for h in range(c["heads"]):
            kh, vh = (x[:, h // (c["heads"] // c["kv_heads"])] for x in (k, v))
            for r in range(0, n, 2048):
                m = min(2048, n - r)
                z = q[r:r + m, h * d:(h + 1) * d] @ kh.t() / math.sqrt(d)
                far = (torch.arange(r, r + m, device="cuda") + before)[:, None] - torch.arange(k.shape[0], device="cuda")
                hidden = (far < 0) | (far >= (c["window"] or k.shape[0] + 1))
                if c["kind"] == "tree" and not c["chain"]:
                    rows = _tree_bits(c)[b][r:r + m]
                    own_bits = [[not x >> j & 1 for j in range(n)] for x in rows]
                    hidden = torch.zeros_like(hidden)
                    hidden[:, before:] = torch.tensor(own_bits, device="cuda")
                z[hidden] = -math.inf
                out[at + r:at + r + m, h * d:(h + 1) * d] = torch.softmax(z, -1) @ vh
        at += n
    return out


def _exact_norm(c, s):
    d, r = c["head_dim"], c["rope_dim"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(s["pos"].double(), s["inv"].double()))[:, None]
    lo = d - r if c["pairing"] == 2 else 0

    def heads(x, w):
        y = x.double().reshape(len(x), -1, d)
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / d + EPS) * w.double()
        z = y[..., lo:lo + r]
        z = z.unflatten(-1, (2, r // 2)).transpose(-1, -2) if c["pairing"] == 1 else z.unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        y[..., lo:lo + r] = (z.transpose(-1, -2) if c["pairing"] == 1 else z).flatten(-2)
        return y.flatten(1)

    q, k = heads(s["q"], s["qw"]), heads(s["k"], s["kw"])
    if not c["kv"]:
        return q, k
    full = s["arena"].view(DT[c["kv"]]).double()
    rows = full.view(-1, BLOCK, k.shape[1])
    pos = s["pos"].long()
    page = s["table"].long()[s["seq"].long(), pos // BLOCK]
    rows[2 * page, pos % BLOCK] = k
    rows[2 * page + 1, pos % BLOCK] = s["v"].double()
    return [q, full]
