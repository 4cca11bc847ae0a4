"""Performance cases of two operators of a decode or prefill step, through their public entry points.

  rotary_write    ``rotary_reshape_and_cache`` / ``_flash``: queries and keys rotated by their
                  positions, keys and values appended to the paged cache (quantised if it is fp8)
  shared_prefix   ``paged_attention_shared_prefix``: decode attention of a batch whose sequences begin
                  with the same blocks, which are read once for all of them

``own`` false: the same results from elementary tensor operations, in 32 bits, rounded once.  Lengths
are quantiles of the range that a case names, so that its work follows from the case alone; the seed
decides their order, the block tables and every value.
"""
from __future__ import annotations

import math
import types

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TABLE = 40960  # positions that the rotation table holds


def _heads(heads, kv_heads, head_size, block_size, dtype="bf16", kv="auto"):
    return {"heads": heads, "kv_heads": kv_heads, "head_size": head_size, "block_size": block_size,
            "dtype": dtype, "kv": kv}


def _rotary(layout, runs, run_lo, run_hi, padded=0, rot=None, neox=True, table="fp32", **heads):
    """`runs` sequences with [run_lo, run_hi] new tokens each at consecutive positions, most of them
    starting inside a block, then `padded` rows of a captured batch that have no slot."""
    return {"op": "rotary_write", "layout": layout, "runs": runs, "run_lo": run_lo, "run_hi": run_hi,
            "padded": padded, "rot": rot or heads["head_size"], "neox": neox, "table": table, **heads}


def _shared(seqs, prefix, lo, hi, alibi=False, **heads):
    """`seqs` sequences with the same first `prefix` tokens and [lo, hi] of their own behind them."""
    return {"op": "shared_prefix", "seqs": seqs, "prefix": prefix, "lo": lo, "hi": hi, "alibi": alibi, **heads}


def listed():
    gqa8b = _heads(32, 8, 128, 16)
    gqa70b_fp8 = _heads(64, 8, 128, 16, kv="fp8")
    return [
        # one interactive user, one new token: a launch and the host's call
        {"name": "rotary_decode_1", **_rotary("x", 1, 1, 1, **gqa8b)},
        # a decode step of a busy server, each token in a block of its own, rows padded to the captured size
        {"name": "rotary_decode_250", **_rotary("x", 250, 1, 1, padded=6, table="bf16", **gqa70b_fp8)},
        # a prefill step at an 8 k-token budget
        {"name": "rotary_prefill_8k", **_rotary("x", 4, 1536, 2560, **gqa8b)},
        # prompts of a quantising server, chunks that start anywhere in a block
        {"name": "rotary_prefill_fp8", **_rotary("x", 121, 100, 171, table="bf16", **gqa70b_fp8)},
        # the flash layout, ragged prompts, a quarter of the head rotated, neighbours paired
        {"name": "rotary_flash_ragged", **_rotary("NHD", 13, 30, 900, rot=32, neox=False, table="fp16",
                                                  **_heads(32, 32, 128, 16, "fp16", "fp8_e5m2"))},
        # a few samples of one prompt, just begun: two launches
        {"name": "shared_samples_4", **_shared(4, 1008, 1, 40, **gqa8b)},
        # multi-head, ALiBi, a head size that is no power of two, blocks of 32
        {"name": "shared_alibi_33", **_shared(33, 1600, 20, 700, alibi=True, **_heads(40, 40, 80, 32, "fp16"))},
        # one long document, eight questions
        {"name": "shared_document_8", **_shared(8, 65008, 30, 1500, **gqa8b)},
        # a full decode batch behind a system prompt with tools and examples
        {"name": "shared_prompt_256", **_shared(256, 4096, 60, 1000, **gqa8b)},
        # the same for a 70B-shape layer with an fp8 cache
        {"name": "shared_fp8_128", **_shared(128, 8192, 200, 2000, **gqa70b_fp8)},
        # the largest: short answers for 2000 users of one prompt
        {"name": "shared_serving_2000", **_shared(2000, 2016, 8, 250, **_heads(64, 8, 128, 32, kv="fp8"))},
    ]


# ------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_heads(rng, types_):
    head_size = 128 if rng.random() < 0.5 else rng.choice([32, 64, 80, 96, 112, 120, 192, 256])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (32, 32), (40, 40), (8, 2), (32, 2), (16, 1),
                                  (12, 4), (8, 8), (28, 4)])
    dtype = rng.choice(types_)
    kv = rng.choice(["auto", "auto", "fp8", "fp8", "fp8_e5m2"])
    if head_size == 120:  # not a multiple of the 16 elements that an fp8 cache keeps together
        kv = "auto"
    return _heads(heads, kv_heads, head_size, rng.choice([16, 16, 32]), dtype, kv)


def _range(rng, lo, hi):
    a, b = sorted((_log(rng, lo, hi), _log(rng, lo, hi)))
    return a, b


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    most = {"rotary_write": 0.0, "shared_prefix": 0.0}
    for c in listed():
        most[c["op"]] = max(most[c["op"]], _cost(c))
    while True:
        if rng.random() < 0.45:
            h = _draw_heads(rng, ["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
            runs, lo, hi = _log(rng, 1, 600), 1, 1
            if rng.random() < 0.6:
                lo, hi = _range(rng, 1, 4096)
            D = h["head_size"]
            c = _rotary(rng.choice(["x", "x", "NHD", "HND"]), runs, lo, hi, rng.choice([0, 0, _log(rng, 1, 16)]),
                        rng.choice([D, D, D, D // 2, D // 4]), rng.random() < 0.7, rng.choice([h["dtype"], "fp32"]), **h)
            n = sum(_new(c))
            if n > 20000 or n * h["kv_heads"] * D > 1 << 26:
                continue
        else:
            h = _draw_heads(rng, ["bf16", "bf16", "fp16"])
            B = h["block_size"]
            lo, hi = _range(rng, 1, 3000)
            c = _shared(_log(rng, 2, 2000), max(1, _log(rng, 64, 65536) // B) * B, lo, hi, rng.random() < 0.15, **h)
            keys = c["seqs"] * (c["prefix"] + hi) * c["heads"]
            if c["seqs"] * hi * h["kv_heads"] * h["head_size"] > 6e8 or keys > 4e8:  # (the plain form's tensors)
                continue
        if _cost(c) <= most[c["op"]]:
            return c


# ------------------------------------------------------------------ lengths and work
def _quantiles(n, lo, hi):
    return [int(lo + (hi - lo) * (i + 0.5) / n + 0.5) for i in range(n)]


def _new(case):
    return _quantiles(case["runs"], case["run_lo"], case["run_hi"])


def _sizes(case):
    es = 4 if case["dtype"] == "fp32" else 2
    return es, (es if case["kv"] == "auto" else 1)  # bytes of an input element, of a cache element


def work(case):
    """Bytes: every input read once, every output written once; the prefix counts once."""
    es, ec = _sizes(case)
    D, H, HK = case["head_size"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary_write":
        n = sum(_new(case))
        rows = n + case["padded"]
        rotation = min(rows, TABLE) * case["rot"] * (4 if case["table"] == "fp32" else 2)
        return {"bytes": rows * (2 * H * D * es + 16) + n * 2 * HK * D * (es + ec) + rotation,
                "flops": 3 * case["rot"] * (rows * H + n * HK)}
    N, P = case["seqs"], case["prefix"]
    lens = _quantiles(N, case["lo"], case["hi"])
    blocks = P // case["block_size"] + sum(-(-v // case["block_size"]) for v in lens)
    return {"bytes": (P + sum(lens)) * HK * D * 2 * ec + 2 * N * H * D * es + 4 * blocks + 4 * N,
            "flops": 4 * H * D * (N * P + sum(lens))}


# ------------------------------------------------------------------ inputs
def _fp8_type(kv):
    return (torch.float8_e5m2, 57344.0) if kv == "fp8_e5m2" else (torch.float8_e4m3fn, 448.0)


def _fill_cache(flat, case, scale, gen):
    """N(0, 1) keys and values, as the cache holds them."""
    step = 1 << 28
    for a in range(0, flat.numel(), step):
        part = flat[a:a + step]
        if case["kv"] == "auto":
            part.normal_(generator=gen)
        else:
            t, top = _fp8_type(case["kv"])
            x = torch.empty(part.numel(), dtype=torch.float16, device=DEV).normal_(generator=gen)
            part.copy_(x.mul_(1.0 / scale).clamp_(-top, top).to(t).view(torch.uint8))


def _state(case):
    fp8 = case["kv"] != "auto"
    s = types.SimpleNamespace(case=case, kv=case["kv"], D=case["head_size"], H=case["heads"], HK=case["kv_heads"],
                              B=case["block_size"], dtype=DTYPES[case["dtype"]], fp8=fp8)
    # a per-tensor scale as calibration gives it: the largest magnitude onto the largest code
    s.kv_scale = 5.3 / _fp8_type(case["kv"])[1] if fp8 else 1.0
    s.k_scale = torch.tensor(s.kv_scale, dtype=torch.float32, device=DEV)
    s.v_scale = torch.tensor(s.kv_scale * 0.75 if fp8 else 1.0, dtype=torch.float32, device=DEV)
    s.cache_dtype = torch.uint8 if fp8 else s.dtype
    s.x = 16 // (1 if fp8 else s.dtype.itemsize)
    return s


def _prepare_rotary(case, rng, gen):
    s = _state(case)
    order = rng.permutation(case["runs"])
    new = np.array(_new(case), dtype=np.int64)[order]
    n, rows, B, D, H, HK = int(new.sum()), int(new.sum()) + case["padded"], s.B, s.D, s.H, s.HK
    start = 37 * (order % 11)  # (most runs start inside a block)
    need = -(-(start + new) // B)
    perm = rng.permutation(int(need.sum()) + 9).astype(np.int64)  # a few blocks that nothing is written to
    first = np.concatenate([[0], np.cumsum(need)[:-1]])
    seq = np.repeat(np.arange(len(new)), new)
    pos = np.concatenate([np.arange(a, a + t) for a, t in zip(start, new)])
    slots = perm[first[seq] + pos // B] * B + pos % B
    # prefill chunks and decodes stand anywhere in their contexts; whole blocks further on
    far = rng.integers(0, (TABLE - int((start + new).max())) // B, len(new)) * B
    positions = np.concatenate([pos + far[seq], np.zeros(case["padded"], np.int64)])
    s.positions = torch.from_numpy(positions).to(DEV)
    s.slots = torch.from_numpy(np.concatenate([slots, np.full(case["padded"], -1)])).to(DEV)
    s.n = n
    # what a fused projection gives: q, k and v of a token next to each other
    qkv = torch.empty((rows, (H + 2 * HK) * D), dtype=s.dtype, device=DEV).normal_(generator=gen)
    q, k, v = qkv.split([H * D, HK * D, HK * D], dim=1)
    s.query, s.key, s.value = q.view(rows, H, D), k.view(rows, HK, D), v.view(rows, HK, D)
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = torch.arange(TABLE, dtype=torch.float64, device=DEV)[:, None] * freq
    s.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1).to(DTYPES[case["table"]])
    s.neox = case["neox"]
    nb = len(perm)
    if case["layout"] == "x":
        s.key_cache = torch.zeros((nb, HK, D // s.x, B, s.x), dtype=s.cache_dtype, device=DEV)
        s.value_cache = torch.zeros((nb, HK, D, B), dtype=s.cache_dtype, device=DEV)
    else:
        shape = (nb, B, HK, D) if case["layout"] == "NHD" else (nb, HK, B, D)
        caches = [torch.zeros(shape, dtype=s.cache_dtype, device=DEV) for _ in range(2)]
        s.key_cache, s.value_cache = caches if case["layout"] == "NHD" else [c.transpose(1, 2) for c in caches]
    s.query_out = torch.empty((rows, H, D), dtype=s.dtype, device=DEV)
    return s


def _prepare_shared(case, rng, gen):
    s = _state(case)
    N, P, B, D, H, HK = case["seqs"], case["prefix"], s.B, s.D, s.H, s.HK
    suffix = rng.permutation(np.array(_quantiles(N, case["lo"], case["hi"]), dtype=np.int64))
    need = -(-suffix // B)
    pb = P // B
    nb = pb + int(need.sum()) + 8
    perm = rng.permutation(nb).astype(np.int32)
    table = np.zeros((N, pb + int(need.max())), dtype=np.int32)
    table[:, :pb] = perm[:pb]
    own_rows = np.repeat(np.arange(N), need)
    first = np.concatenate([[0], np.cumsum(need)[:-1]])
    table[own_rows, pb + np.arange(len(own_rows)) - first[own_rows]] = perm[pb:pb + len(own_rows)]
    s.prefix, s.max_len, s.scale = P, P + int(suffix.max()), D ** -0.5
    s.suffix_max = int(suffix.max())
    s.table = torch.from_numpy(table).to(DEV)
    s.lens = torch.from_numpy((P + suffix).astype(np.int32)).to(DEV)
    s.key_cache = torch.empty((nb, HK, D // s.x, B, s.x), dtype=s.cache_dtype, device=DEV)
    s.value_cache = torch.empty((nb, HK, D, B), dtype=s.cache_dtype, device=DEV)
    _fill_cache(s.key_cache.view(-1), case, s.kv_scale, gen)
    _fill_cache(s.value_cache.view(-1), case, s.kv_scale, gen)
    s.query = torch.empty((N, H, D), dtype=s.dtype, device=DEV).normal_(generator=gen)
    slopes = [2.0 ** (-8.0 * (i + 1) / H) for i in range(H)]
    s.alibi = torch.tensor(slopes, dtype=torch.float32, device=DEV) if case["alibi"] else None
    s.out = torch.empty_like(s.query)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    return (_prepare_rotary if case["op"] == "rotary_write" else _prepare_shared)(case, rng, gen)


# ------------------------------------------------------------------ the plain forms
def _to_cache(s, x, scale):
    """fp32 values as the cache stores them."""
    if not s.fp8:
        return x.to(s.dtype)
    t, top = _fp8_type(s.kv)
    return (x / scale).clamp(-top, top).to(t).view(torch.uint8)


def _from_cache(s, x, scale):
    return x.view(_fp8_type(s.kv)[0]).float() * scale if s.fp8 else x.float()


def _rotated(x, cos, sin, rot, neox):
    x = x.float()
    cos, sin = cos.float()[:, None, :], sin.float()[:, None, :]
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if neox else (x[..., :rot:2], x[..., 1:rot:2])
    y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-2 if neox else -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], dim=-1)


def _plain_rotary(s):
    rot, n = s.case["rot"], s.n
    cos, sin = s.cos_sin.index_select(0, s.positions).split(rot // 2, dim=1)
    query = _rotated(s.query, cos, sin, rot, s.neox).to(s.dtype)
    key = _to_cache(s, _rotated(s.key[:n], cos[:n], sin[:n], rot, s.neox), s.k_scale)
    value = _to_cache(s, s.value[:n].float(), s.v_scale)
    slots = s.slots[:n]
    block, at = slots // s.B, slots % s.B
    if s.case["layout"] == "x":
        s.key_cache[block, :, :, at] = key.view(n, s.HK, s.D // s.x, s.x)
        s.value_cache[block, :, :, at] = value
    else:
        s.key_cache[block, at] = key
        s.value_cache[block, at] = value
    return query


def _plain_shared(s):
    N, P, HK, D, L = s.case["seqs"], s.prefix, s.HK, s.D, s.suffix_max
    G = s.H // HK
    q = s.query.float().view(N, HK, G, D) * s.scale
    pb, need = P // s.B, -(-L // s.B)

    def pages(cache, blocks, scale):  # [..., blocks] -> [..., tokens, HK, D]
        c = _from_cache(s, cache[blocks.long()], scale)
        if c.dim() - blocks.dim() == 4:  # K: HK, D / x, B, x
            c = c.movedim(-2, -4).flatten(-2)
        else:
            c = c.movedim(-1, -3)
        return c.flatten(-4, -3)

    kp, vp = (pages(c, s.table[0, :pb], sc) for c, sc in ((s.key_cache, s.k_scale), (s.value_cache, s.v_scale)))
    logits = torch.empty((HK, N, G, P + need * s.B), dtype=torch.float32, device=DEV)
    qh = q.permute(1, 0, 2, 3)  # HK, N, G, D
    logits[..., :P] = torch.matmul(qh.reshape(HK, N * G, D), kp.permute(1, 2, 0)).view(HK, N, G, P)
    ks = pages(s.key_cache, s.table[:, pb:pb + need], s.k_scale)
    logits[..., P:] = torch.matmul(qh, ks.permute(2, 0, 3, 1))
    del ks
    at = torch.arange(P + need * s.B, device=DEV)
    if s.alibi is not None:
        bias = (at - (s.lens[:, None] - 1)).float()  # N, keys
        logits += s.alibi.view(HK, 1, G, 1) * bias[None, :, None, :]
    logits.masked_fill_((at >= s.lens[:, None])[None, :, None, :], -math.inf)
    logits -= logits.amax(dim=-1, keepdim=True)
    p = logits.exp_()
    p /= p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p[..., :P].reshape(HK, N * G, P), vp.permute(1, 0, 2)).view(HK, N, G, D)
    vs = pages(s.value_cache, s.table[:, pb:pb + need], s.v_scale)
    # (blocks behind a sequence's end: whatever they hold counts nothing)
    vs.masked_fill_((at[P:] >= s.lens[:, None])[:, :, None, None], 0)
    out += torch.matmul(p[..., P:], vs.permute(2, 0, 1, 3))
    return out.permute(1, 0, 2, 3).reshape(N, s.H, D).to(s.dtype)


def _values(s, cache):
    return cache.view(_fp8_type(s.kv)[0]) if s.fp8 else cache


def run(s):
    if s.case["op"] == "rotary_write":
        if own:
            from vllm_b200 import _custom_ops as ops
            write = ops.rotary_reshape_and_cache if s.case["layout"] == "x" else ops.rotary_reshape_and_cache_flash
            write(s.query_out, s.positions, s.query, s.key, s.value, s.cos_sin, s.neox, s.key_cache, s.value_cache,
                  s.slots, s.kv, s.k_scale, s.v_scale)
            query = s.query_out
        else:
            query = _plain_rotary(s)
        return {"query": query, "key_cache": _values(s, s.key_cache), "value_cache": _values(s, s.value_cache)}
    if own:
        from vllm_b200 import _custom_ops as ops
        ops.paged_attention_shared_prefix(s.out, s.query, s.key_cache, s.value_cache, s.HK, s.scale, s.table, s.lens,
                                          s.prefix, s.B, s.max_len, s.alibi, s.kv, s.k_scale, s.v_scale)
        return s.out
    return _plain_shared(s)


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_rotary(case, s):
    half, n = case["rot"] // 2, s.n
    table = s.cos_sin.double()[s.positions]
    turn = torch.complex(table[:, :half], table[:, half:])[:, None, :]  # a + ib times e^(i angle)

    def turned(x):
        y = x.double().clone()
        i = torch.arange(half, device=DEV)
        first, second = (i, i + half) if case["neox"] else (2 * i, 2 * i + 1)
        z = torch.complex(y[..., first], y[..., second]) * turn[:x.shape[0]]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def stored(x, scale):
        top = _fp8_type(case["kv"])[1]
        return (x / scale.double()).clamp(-top, top) if s.fp8 else x

    caches = []
    slots = s.slots[:n]
    for x, scale, cache, is_key in ((turned(s.key[:n]), s.k_scale, s.key_cache, True),
                                    (s.value[:n].double(), s.v_scale, s.value_cache, False)):
        nb, flat = cache.shape[0], torch.zeros((cache.shape[0] * s.B, s.HK, s.D), dtype=torch.float64, device=DEV)
        flat[slots] = stored(x, scale)
        flat = flat.view(nb, s.B, s.HK, s.D)
        if case["layout"] == "x":
            flat = flat.permute(0, 2, 3, 1)  # nb, HK, D, B
            if is_key:
                flat = flat.unflatten(2, (s.D // s.x, s.x)).transpose(3, 4)
        elif case["layout"] == "HND":
            flat = flat.transpose(1, 2).contiguous().transpose(1, 2)
        # (two mantissa bits: their rounding alone is 5 % of the values, which says nothing about an error)
        caches.append(None if case["kv"] == "fp8_e5m2" else flat)
    return {"query": turned(s.query), "key_cache": caches[0], "value_cache": caches[1]}


def _exact_shared(case, s):
    N, HK, D, G = case["seqs"], s.HK, s.D, s.H // s.HK
    pb = s.prefix // s.B
    out = torch.empty((N, s.H, D), dtype=torch.float64, device=DEV)
    lens = s.lens.long()
    # a few sequences at a time, every one with its whole context: prefix and suffix make no difference here
    step = max(1, int(2e8) // (s.max_len * D))
    pos = torch.arange(s.table.shape[1] * s.B, device=DEV)
    kt, vt = (_values(s, c) for c in (s.key_cache, s.value_cache))
    ks, vs = (float(t) if s.fp8 else 1.0 for t in (s.k_scale, s.v_scale))
    for h in range(HK):
        k_all = kt[:, h].double().mul_(ks).transpose(2, 3).flatten(1, 2)  # blocks, D, B
        v_all = vt[:, h].double().mul_(vs)
        for a in range(0, N, step):
            b = min(N, a + step)
            t = s.table[a:b].long()
            k = k_all[t].transpose(1, 2).flatten(2)  # sequences, D, keys
            v = v_all[t].transpose(1, 2).flatten(2)
            q = s.query[a:b, h * G:(h + 1) * G].double()
            z = (q @ k).mul_(s.scale)
            gone = (pos >= lens[a:b, None])[:, None, :]
            if s.alibi is not None:
                z += s.alibi[h * G:(h + 1) * G].double()[None, :, None] * (pos + 1 - lens[a:b, None])[:, None, :]
            z.masked_fill_(gone, -math.inf)
            p = torch.softmax(z, dim=-1)
            out[a:b, h * G:(h + 1) * G] = p @ v.masked_fill_(gone, 0).transpose(1, 2)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotary(case, s) if case["op"] == "rotary_write" else _exact_shared(case, s)
