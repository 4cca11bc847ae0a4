"""paged_attention_shared_prefix: decode attention of a batch that begins with the same blocks, against the
definition in 64 bits.

Tolerance, of an output row with weights p and values v: P is rounded to 16 bits before the second product
(half a step of the operands' type each: u = eps / 2, f16 for fp8 caches) while its sum is not, the rest is
fp32 (2^-20 covers its few hundred additions and the exponentials), and the result is rounded once more.  So
|error| <= u_p sum(p |v|) + 2^-20 sum(p |v|) + u_out |out|, with the logits' own fp32 error of a few 2^-22 of
sum |q k| in the exponent: sum |q k| <= 40 here, 40 * 2^-22 = 2^-16.7 of sum(p |v|), in all below
(u_p + 2^-16) sum(p |v|) + u_out |out|.  A further 2^-22 for the subnormal results of fp16."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from vllm_b200 import _custom_ops as ops
from vllm_b200 import capi

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = {"fp8": torch.float8_e4m3fn, "fp8_e5m2": torch.float8_e5m2}


class Case:
    def __init__(self, own=(1, 20, 33, 7), prefix=256, H=8, HK=2, D=128, B=16, dtype="bf16", kv="auto", alibi=False,
                 seed=0, q_size=1.0, stale=True):
        g = torch.Generator().manual_seed(seed)
        N = len(own)
        self.N, self.prefix, self.H, self.HK, self.D, self.B, self.kv = N, prefix, H, HK, D, B, kv
        self.dtype = DT[dtype]
        pb = prefix // B
        lens = [max(0, prefix + n) for n in own]
        need = [max(0, -(-n // B)) for n in own]
        nb = pb + sum(need) + 3
        perm = torch.randperm(nb, generator=g).to(torch.int32)
        self.bt = torch.full((N, pb + max(max(need), 1)), nb - 1, dtype=torch.int32)
        self.bt[:, :pb] = perm[:pb]
        at = pb
        for i, n in enumerate(need):
            self.bt[i, pb:pb + n] = perm[at:at + n]
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.max_len = max(max(lens), 1)
        fp8 = kv != "auto"
        x = 16 // (1 if fp8 else self.dtype.itemsize)
        kc, vc = torch.randn(nb, HK, D // x, B, x, generator=g), torch.randn(nb, HK, D, B, generator=g)
        self.ks, self.vs = torch.tensor(0.37 if fp8 else 1.0), torch.tensor(0.21 if fp8 else 1.0)
        kc, vc = ((t * 2).to(F8[kv]).view(torch.uint8) if fp8 else t.to(self.dtype) for t in (kc, vc))
        if stale:  # what lies behind the end of a sequence must not matter
            bad = 0x7F if fp8 else float("nan")
            for i, n in enumerate(own):
                if n > 0 and n % B:
                    b = self.bt[i, pb + n // B]
                    kc[b, :, :, n % B:] = bad
                    vc[b, :, :, n % B:] = bad
        q = torch.randn(N, H, D, generator=g) * q_size
        self.q, self.kc, self.vc = q.to(self.dtype).to(DEV), kc.to(DEV), vc.to(DEV)
        self.bt, self.lens, self.ks, self.vs = (t.to(DEV) for t in (self.bt, self.lens, self.ks, self.vs))
        self.scale = D ** -0.5
        self.alibi = torch.tensor([2.0 ** (-8.0 * (i + 1) / H) for i in range(H)], device=DEV) if alibi else None

    def call(self, out=None, **kw):
        out = torch.full((self.N, self.H, self.D), 9.0, dtype=self.dtype, device=DEV) if out is None else out
        a = dict(out=out, query=self.q, key_cache=self.kc, value_cache=self.vc, num_kv_heads=self.HK, scale=self.scale,
                 block_tables=self.bt, seq_lens=self.lens, prefix_len=self.prefix, block_size=self.B,
                 max_seq_len=self.max_len, alibi_slopes=self.alibi, kv_cache_dtype=self.kv, k_scale=self.ks,
                 v_scale=self.vs)
        a.update(kw)
        ops.paged_attention_shared_prefix(**a)
        return out

    def want(self):
        """(out, sum of p |v|, lse) in 64 bits."""
        N, H, HK, D, B = self.N, self.H, self.HK, self.D, self.B
        val = (lambda t, s: t.view(F8[self.kv]).double() * s.double()) if self.kv != "auto" else (lambda t, s: t.double())
        out, mag = torch.zeros(2, N, H, D, dtype=torch.float64, device=DEV)
        lse = torch.full((H, N), -float("inf"), dtype=torch.float64, device=DEV)
        table = self.bt
        for i in range(N):
            n = int(self.lens[i])
            if n <= 0:
                continue
            blocks = table[i, :-(-n // B)].long()
            k = val(self.kc[blocks].permute(0, 3, 1, 2, 4).reshape(-1, HK, D)[:n], self.ks)
            v = val(self.vc[blocks].permute(0, 3, 1, 2).reshape(-1, HK, D)[:n], self.vs)
            q = self.q[i].double().view(HK, H // HK, D)
            z = torch.einsum("hgd,nhd->hgn", q, k) * self.scale
            if self.alibi is not None:
                z = z + self.alibi.double().view(HK, -1, 1) * torch.arange(1 - n, 1, device=DEV)
            p = torch.softmax(z, -1)
            out[i] = torch.einsum("hgn,nhd->hgd", p, v).reshape(H, D)
            mag[i] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(H, D)
            lse[:, i] = torch.logsumexp(z, -1).flatten()
        return out, mag, lse

    def check(self, got, lse=None):
        out, mag, want_lse = self.want()
        u_out = torch.finfo(self.dtype).eps / 2
        u_p = torch.finfo(torch.float16 if self.kv != "auto" else self.dtype).eps / 2
        tol = mag * (u_p + 2.0 ** -16) + out.abs() * u_out + 2.0 ** -22
        bad = (got.double() - out).abs() > tol
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], out[bad][:4])
        if lse is not None:
            assert torch.equal(lse.isinf(), want_lse.isinf())
            fine = ~lse.isinf()
            # (a sum of n fp32 exponentials, its logarithm and the maximum: a few 2^-20)
            assert ((lse.double() - want_lse).abs()[fine] <= 1e-5 * (1 + want_lse.abs()[fine])).all()


def _run(**kw):
    c = Case(**kw)
    lse = torch.full((c.H, c.N), 5.0, device=DEV)
    c.check(c.call(lse=lse), lse)
    assert capi.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["auto", "fp8", "fp8_e5m2"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("H,HK", [(8, 2), (4, 4), (16, 1), (32, 1), (12, 4), (14, 2)])
def test_types_and_heads(kv, dtype, H, HK):
    _run(H=H, HK=HK, kv=kv, dtype=dtype, own=(1, 20, 33, 7, 300))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 80, 96, 112, 120, 192, 256])
@pytest.mark.parametrize("kv,B", [("auto", 16), ("auto", 32), ("fp8", 16), ("fp8_e5m2", 32)])
@pytest.mark.parametrize("N", [3, 70])
def test_head_and_block_sizes(D, kv, B, N):
    if D == 120 and kv != "auto":
        pytest.skip("an fp8 cache keeps 16 head dimensions together")
    _run(D=D, kv=kv, B=B, own=tuple(1 + 13 * i % 90 for i in range(N)), prefix=21 * B)


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [16, 112, 128, 144, 1024, 4112, 20000])
@pytest.mark.parametrize("N", [2, 32, 33, 65, 150])
def test_prefixes_and_row_tiles(prefix, N):
    """Pages that end inside a tile; one row tile of 32 sequences, two, an odd number of them."""
    _run(prefix=prefix, own=tuple(1 + 17 * i % 40 for i in range(N)), H=8, HK=2)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_long_and_uneven_own_parts(kv):
    _run(prefix=512, own=(3000, 1, 16, 500, 17, 2048, 1, 1), kv=kv)
    _run(prefix=512, own=(4000, 3), kv=kv, H=4, HK=1)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_one_long_sequence_among_short_ones(kv):
    """Its own part is cut over nearly all warps, into as many pieces as there may be."""
    _run(prefix=1024, own=(30000,) + tuple(1 + 7 * i % 100 for i in range(60)), kv=kv, H=8, HK=1)
    _run(prefix=2048, own=(3, 9000, 12, 9000) + (20,) * 60, kv=kv, H=16, HK=2, D=64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kv", [("bf16", "auto"), ("fp16", "fp8")])
@pytest.mark.parametrize("N", [4, 40])
def test_alibi(dtype, kv, N):
    _run(alibi=True, dtype=dtype, kv=kv, own=tuple(1 + 29 * i % 200 for i in range(N)), prefix=800, H=8, HK=8)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 80])
def test_sequences_without_own_tokens_and_shorter_ones(N):
    """Rows that see a part of the prefix only, or nothing at all: zeros and an lse of -inf."""
    _run(own=tuple((0, -3, 5, -250, -256, -300, -130, 1)[i % 8] for i in range(N)), prefix=256)
    _run(own=tuple((0, -3, 5, -250, -256, -300, -130, 1)[i % 8] for i in range(N)), prefix=256, alibi=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,behind", [("auto", 6), ("fp8_e5m2", 6), ("auto", 300), ("fp8_e5m2", 300)])
def test_prefix_values_that_a_shorter_sequence_does_not_see(kv, behind):
    """An infinite value of the prefix reaches the sequences that have it, and no other one."""
    c = Case(own=(-100, behind, -255, -1, behind, -256) * 15, prefix=256, kv=kv)
    c.vc[c.bt[0, 15], :, 5, 15] = 0x7C if kv != "auto" else float("inf")  # the prefix's last token
    lse = torch.full((c.H, c.N), 5.0, device=DEV)
    got = c.call(lse=lse)
    full = c.lens >= c.prefix
    assert (got[full][:, :, 5] == float("inf")).all()
    out, mag, want_lse = c.want()
    u = torch.finfo(torch.float16 if kv != "auto" else c.dtype).eps / 2
    tol = mag * (u + 2.0 ** -16) + out.abs() * 2.0 ** -8 + 2.0 ** -22
    short = (~full).nonzero().flatten()
    assert ((got[short].double() - out[short]).abs() <= tol[short]).all()
    assert ((lse.double() - want_lse).abs()[:, c.lens > 0] <= 1e-5 * (1 + want_lse.abs()[:, c.lens > 0])).all()


@pytest.mark.gpu
def test_all_rows_empty_or_no_sequences():
    c = Case(own=(-256, -256, -300), prefix=256)
    assert (c.call() == 0).all()
    c.call(out=torch.empty(0, 8, 128, dtype=torch.bfloat16, device=DEV), query=c.q[:0])


@pytest.mark.gpu
def test_peaked_logits():
    """The maximum jumps late and early, in the prefix and behind it: the largest logits are over 100."""
    for seed in range(3):
        c = Case(own=(30, 500, 1), prefix=1024, q_size=0.05, seed=seed)
        for i, (blk, off) in enumerate(((0, 3), (63, 15), (30, 8))):
            c.kc[c.bt[0, blk], :, :, off] = (c.q[i, 0].view(-1, 8) * 400).to(c.dtype)
        got = c.call()
        out, mag, _ = c.want()
        # (logits of 200 in fp32: 200 * 2^-22 more of sum(p |v|))
        assert ((got.double() - out).abs() <= mag * (2.0 ** -8 + 2.0 ** -13) + out.abs() * 2.0 ** -8).all()


@pytest.mark.gpu
def test_infinite_and_nan_keys_stay_with_their_rows():
    c = Case(own=(20, 30, 40) * 20, prefix=4096)
    c.lens[3:] = 0
    assert _route(num_seqs=60, max_seq_len=c.max_len, prefix=4096) != 0
    kc = c.kc.clone()
    c.q[1] = 0.0
    c.q[1, :, 0] = 1.0
    c.kc[c.bt[1, 256], :, 0, 2, 0] = -float("inf")   # one own key of sequence 1: weight 0
    got = c.call()
    c.kc = kc
    keep = torch.ones(c.N, dtype=torch.bool)
    out, mag, _ = c.want()
    assert got[1].isfinite().all()
    ok = (got.double() - out).abs() <= mag * 2.0 ** -7 + out.abs() * 2.0 ** -7
    assert ok[keep.nonzero().flatten()[[0, 2]]].all()
    c.q[2, 3] = float("nan")
    got = c.call()
    assert got[2, 3].isnan().all() and not got[[0, 1]].isnan().any() and not got[2, :3].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["auto", "fp8_e5m2"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("blocks", [range(256, 257), range(256, 258), range(257, 258), range(256, 264), range(0, 8),
                                    range(8, 16), range(0, 256)], ids=lambda r: f"{r.start}-{r.stop}")
def test_logits_of_minus_infinity(blocks, D, kv):
    """Whole tiles, the whole prefix, and all own tokens (blocks from 256 on) with logits of -inf: weights of 0."""
    c = Case(own=(20, 50, 100, 128, 7) * 12, prefix=4096, D=D, kv=kv)
    if "B200PA_TUNE_BEHIND" not in os.environ:
        assert _route(prefix=c.prefix, num_seqs=60, head_size=D, q_stride=8 * D, kv_block_stride=32 * D, kv_head_stride=16 * D,
                      max_seq_len=c.max_len) != 0
    c.q[:, :, 0] = c.q[:, :, 0].abs() + 0.25
    for b in blocks:
        for i in range(c.N):
            if b * c.B < int(c.lens[i]):
                c.kc[c.bt[i, b], :, 0, :, 0] = 0xFC if kv != "auto" else -float("inf")
    lse = torch.full((c.H, c.N), 5.0, device=DEV)
    c.check(c.call(lse=lse), lse)


@pytest.mark.gpu
@pytest.mark.parametrize("H,HK", [(28, 4), (12, 4), (40, 8)])
@pytest.mark.parametrize("dtype,kv", [("bf16", "auto"), ("fp16", "fp8"), ("bf16", "fp8_e5m2")])
def test_rows_of_a_tile_without_a_sequence_change_nothing(H, HK, dtype, kv):
    """Head groups that do not divide 128 leave rows of a tile unused: what the launch before has left in shared memory
    there decides nothing, not even when the others are scaled again (the results are the same to the last bit)."""
    c = Case(own=tuple(7 + 11 * i % 110 for i in range(200)), prefix=1504, H=H, HK=HK, dtype=dtype, kv=kv)
    before = Case(own=(1,) * 64, prefix=8192, H=64, HK=8, dtype=dtype, kv=kv)  # (8 heads: every row in use, every SM)
    q, got = before.q.clone(), []
    for size in (0.0, 30.0):
        before.q.copy_(q * size)
        before.call()
        got.append(c.call())
    assert torch.equal(*got)
    c.check(got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("own", [(1,) * 40, (60, 300) * 20, (5, 900) * 60])
def test_scales_that_change_right_before_the_call(own):
    """v_scale comes from the launch just before: powers of two scale the result exactly."""
    c = Case(own=own, prefix=4096, kv="fp8")
    want = c.call().float()
    for i in range(100):
        f = 2.0 ** (i % 5 - 2)
        c.vs.fill_(0.21 * f)
        assert torch.equal(c.call().float(), want * f)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(dtype="fp32"), dict(B=8), dict(own=(40,))])
def test_shapes_without_a_kernel_run_as_ordinary_decodes(kw):
    c = Case(prefix=64, **kw)
    got = c.call()
    out, mag, _ = c.want()
    assert ((got.double() - out).abs() <= (mag + out.abs()) * 2.0 ** -7).all()


@pytest.mark.gpu
def test_strided_query_and_caches():
    c = Case(own=(5, 9, 30, 1), prefix=144)
    want = c.call()
    wide = torch.randn(4, 12, 128, device=DEV).to(c.dtype)
    wide[:, 2:10] = c.q
    assert torch.equal(c.call(query=wide[:, 2:10]), want)
    both = torch.empty(2, *c.vc.shape, dtype=c.dtype, device=DEV).transpose(0, 1)  # K's and V's blocks in turns
    both = torch.empty(c.vc.shape[0], 2, *c.vc.shape[1:], dtype=c.dtype, device=DEV)
    both[:, 0], both[:, 1] = c.kc.reshape(c.vc.shape), c.vc
    kc = both[:, 0].view(c.kc.shape)
    assert torch.equal(c.call(key_cache=kc, value_cache=both[:, 1]), want)
    odd = torch.empty(4 * 8 * 128 + 1, dtype=c.dtype, device=DEV)[1:].view(4, 8, 128)  # unaligned: ordinary decodes
    odd.copy_(c.q)
    c.check(c.call(query=odd))


@pytest.mark.gpu
def test_no_prefix():
    c = Case(own=(5, 9, 30), prefix=0)
    c.check(c.call())


@pytest.mark.gpu
def test_it_is_the_same_every_time_and_against_v1():
    c = Case(own=tuple(1 + 7 * i % 60 for i in range(90)), prefix=2000, H=16, HK=4)
    a = c.call()
    for _ in range(3):
        assert torch.equal(c.call(), a)
    b = torch.empty_like(a)
    ops.paged_attention_v1(b, c.q, c.kc, c.vc, c.HK, c.scale, c.bt, c.lens, c.B, c.max_len, None, c.kv, c.ks, c.vs)
    assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm()


@pytest.mark.gpu
def test_two_streams_and_two_graphs_at_once():
    cs = [Case(own=tuple(1 + 7 * i % 300 for i in range(50 + s)), prefix=3008, seed=s) for s in range(2)]
    want = [c.call() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [torch.empty_like(w) for w in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, o in zip(cs, streams, outs):
            with torch.cuda.stream(s):
                c.call(out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for c, o in zip(cs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.call(out=o)
        graphs.append(g)
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    # other lengths and queries under the same graph
    c, d = cs[0], Case(own=tuple(3 + 5 * i % 290 for i in range(50)), prefix=3008, seed=9)
    c.q.copy_(d.q)
    c.lens.copy_(torch.minimum(d.lens, c.lens))
    graphs[0].replay()
    torch.cuda.synchronize()
    c.check(outs[0])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes, with the blocks in use at its end."""
    c = Case(own=(20, 3, 40), prefix=256, H=8, HK=8)
    nb, per = c.kc.shape[0], c.kc[0].numel()
    n = (1 << 32) // (per * 2) + nb + 1
    kc = torch.zeros((n, *c.kc.shape[1:]), dtype=c.dtype, device=DEV)
    vc = torch.zeros((n, *c.vc.shape[1:]), dtype=c.dtype, device=DEV)
    kc[-nb:], vc[-nb:] = c.kc, c.vc
    want = c.call()
    assert torch.equal(c.call(key_cache=kc, value_cache=vc, block_tables=c.bt + (n - nb)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("what,kw,msg", [
    ("prefix inside a block", lambda c: dict(prefix_len=100), "multiple of the block size"),
    ("prefix below zero", lambda c: dict(prefix_len=-16), "prefix_len"),
    ("prefix beyond the tables", lambda c: dict(prefix_len=16 * 100), "does not fit"),
    ("lse shape", lambda c: dict(lse=torch.empty(4, 8, device=DEV)), "lse"),
    ("too few lengths", lambda c: dict(seq_lens=c.lens[:3]), "row for every sequence"),
    ("too few tables", lambda c: dict(block_tables=c.bt[:3]), "row for every sequence"),
    ("block size", lambda c: dict(block_size=32), "block size"),
    ("heads", lambda c: dict(num_kv_heads=4), "heads"),
    ("slopes", lambda c: dict(alibi_slopes=torch.ones(3, device=DEV)), "alibi_slopes"),
    ("kv name", lambda c: dict(kv_cache_dtype="int4"), "Unsupported data type"),
    ("types", lambda c: dict(out=torch.empty(4, 8, 128, device=DEV)), "dtypes differ"),
])
def test_refusals(what, kw, msg):
    c = Case()
    out = torch.full((c.N, c.H, c.D), 9.0, dtype=c.dtype, device=DEV)
    with pytest.raises((RuntimeError, NotImplementedError), match=msg):
        c.call(**(dict(out=out) | kw(c)))
    torch.cuda.synchronize()
    assert (out == 9.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["V's blocks elsewhere", "fewer V blocks", "K in pieces", "V in pieces", "slopes"])
def test_layouts_that_are_refused(which):
    """V is read by K's strides."""
    c = Case(own=(5, 9, 30, 1), prefix=144, alibi=True)
    kw = {}
    if which == "V's blocks elsewhere":
        kw["value_cache"] = torch.stack([c.vc, c.vc], 1)[:, 0]
    elif which == "fewer V blocks":
        kw["value_cache"] = c.vc[:-1]
    elif which == "K in pieces":
        kw["key_cache"] = torch.stack([c.kc, c.kc], 4)[:, :, :, :, 0]
        kw["value_cache"] = torch.stack([c.vc, c.vc], 1)[:, 0].as_strided(c.vc.shape, (*kw["key_cache"].stride()[:2], 16, 1))
    elif which == "V in pieces":
        kw["value_cache"] = c.vc.transpose(2, 3).contiguous().transpose(2, 3)
    else:
        kw["alibi_slopes"] = torch.stack([c.alibi, c.alibi], 1)[:, 0]
    out = torch.full((c.N, c.H, c.D), 9.0, dtype=c.dtype, device=DEV)
    with pytest.raises(RuntimeError, match="strides|alibi_slopes"):
        c.call(out=out, **kw)
    torch.cuda.synchronize()
    assert (out == 9.0).all()


@pytest.mark.gpu
def test_the_c_interface_asks_for_scratch():
    c = Case(own=(5, 9, 30) * 20, prefix=4096)
    out = torch.full((c.N, c.H, c.D), 9.0, dtype=c.dtype, device=DEV)
    a = _c_args(num_seqs=c.N, num_heads=c.H, num_kv_heads=c.HK, max_seq_len=c.max_len, scale=c.scale,
                max_num_blocks_per_seq=c.bt.shape[1], q_stride=c.H * c.D, kv_block_stride=c.kc.stride(0),
                kv_head_stride=c.kc.stride(1), out=out.data_ptr(), query=c.q.data_ptr(), key_cache=c.kc.data_ptr(),
                value_cache=c.vc.data_ptr(), block_tables=c.bt.data_ptr(), seq_lens=c.lens.data_ptr())[0]
    n = capi.shared_prefix_scratch_bytes(a, c.prefix)
    assert n > 0 and capi.shared_prefix_route(a, c.prefix) > 0
    scratch = torch.empty(n, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    for ptr, size in ((0, n), (scratch.data_ptr(), n - 1), (scratch.data_ptr() + 8, n)):
        with pytest.raises(RuntimeError, match="bytes of scratch"):
            capi.paged_attention_shared_prefix(a, c.prefix, ptr, size, stream)
    capi.paged_attention_shared_prefix(a, c.prefix, scratch.data_ptr(), n, stream)
    c.check(out)


def _c_args(**kw):
    buf = C.create_string_buffer(1024)
    mem = C.addressof(buf) + 255 & ~255  # (any aligned address: nothing is launched)
    a = capi.AttnArgs()
    a.num_seqs, a.num_heads, a.num_kv_heads, a.head_size = 4, 8, 2, 128
    a.block_size, a.max_seq_len, a.max_num_blocks_per_seq = 16, 300, 20
    a.q_dtype, a.kv_dtype, a.scale = capi.BF16, capi.KV_AUTO, 0.088
    a.q_stride, a.kv_block_stride, a.kv_head_stride = 1024, 4096, 2048
    for k in ("out", "query", "key_cache", "value_cache", "block_tables", "seq_lens"):
        setattr(a, k, mem)
    for k, v in kw.items():
        setattr(a, k, v)
    return a, buf


@pytest.mark.parametrize("kw,prefix,msg", [
    (dict(head_size=48), 64, "Unsupported head size"), (dict(block_size=64), 64, "Unsupported block size"),
    (dict(), 100, "multiple of the block size"), (dict(), -16, "multiple of the block size"),
    (dict(), 336, "does not fit"), (dict(query=None), 64, "null tensor"), (dict(num_heads=7), 64, "not a multiple"),
    (dict(blocksparse_vert_stride=2, blocksparse_block_size=64), 64, "block-sparse"),
    (dict(kv_dtype=capi.KV_FP8_E4M3), 64, "k_scale"),
])
def test_the_c_interface_refuses(kw, prefix, msg):
    a, _ = _c_args(**kw)
    capi.launch_count(reset=True)
    with pytest.raises(RuntimeError, match=msg):
        capi.paged_attention_shared_prefix(a, prefix, 0, 0)
    with pytest.raises(RuntimeError, match=msg):
        capi.shared_prefix_scratch_bytes(a, prefix)
    assert capi.launch_count() == 0


def _route(prefix=256, **kw):
    a, _ = _c_args(**(dict(max_num_blocks_per_seq=10000) | kw))
    return capi.shared_prefix_route(a, prefix)


@pytest.mark.skipif("B200PA_TUNE_BEHIND" in os.environ, reason="forced")
def test_which_way_a_call_goes():
    """Little to share: the ordinary kernels.  Few sequences with short own parts, many with short ones, long ones."""
    assert _route(num_seqs=1) == 0 and _route(prefix=0) == 0 and _route(num_seqs=4, prefix=64) == 0
    assert capi.shared_prefix_scratch_bytes(_c_args(num_seqs=4)[0], 64) == 0
    assert _route(num_seqs=64, prefix=4096, max_seq_len=4096 + 60) == 1
    assert _route(num_seqs=2000, num_heads=64, num_kv_heads=8, prefix=4096, max_seq_len=4096 + 100) == 2
    assert _route(num_seqs=256, num_heads=32, num_kv_heads=8, prefix=4096, max_seq_len=4096 + 1000) == 3
    assert _route(num_seqs=256, num_heads=32, num_kv_heads=8, head_size=120, q_stride=3840, kv_block_stride=1920 * 8,
                  kv_head_stride=1920, prefix=4096, max_seq_len=4096 + 1000) in (1, 2)  # (no persistent kernel)


@pytest.mark.gpu
@pytest.mark.skipif("B200PA_TUNE_BEHIND" in os.environ, reason="forced")
@pytest.mark.parametrize("behind", ["1", "2", "3"])
def test_every_way_at_every_size(behind):
    """B200PA_TUNE_BEHIND forces one way for every call that has a kernel for the prefix (read once per process)."""
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", __file__],
                       env=dict(os.environ, B200PA_TUNE_BEHIND=behind), cwd=str(root), capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stdout[-3000:]


def test_what_needs_scratch():
    """The plan is arithmetic on the sizes: a slot to every item and one more to every CTA."""
    def need(prefix=256, **kw):
        a, _ = _c_args(**(dict(max_num_blocks_per_seq=64) | kw))
        return capi.shared_prefix_scratch_bytes(a, prefix)
    assert need(num_seqs=0) == 0 and need(num_seqs=1) == 0 and need(prefix=0) == 0
    assert need(q_dtype=capi.F32, head_size=64) == 0 and need(block_size=8) == 0 and need(q_stride=1025) == 0
    many = dict(num_seqs=200, prefix=4096, max_num_blocks_per_seq=300)
    assert need(**many, kv_head_stride=0) == 0 and need(**many, num_kv_heads=1, kv_head_stride=0) > 0
    part = 128 * (128 * 4 + 8)
    assert need(num_seqs=64, prefix=4096, max_num_blocks_per_seq=300) >= 2 * part


@pytest.mark.skipif("B200PA_TUNE_BEHIND" in os.environ, reason="forced")
@pytest.mark.parametrize("H,HK", [(40, 40), (16, 8), (24, 8), (40, 8), (32, 4), (64, 4)])
def test_partials_have_room_for_the_heads_that_there_are(H, HK):
    """Where the persistent kernel is behind the prefix: a partial of an item's heads to every item, and one more to every
    range (12 to 16 warps of 148 SMs at most), beside the prefix's parts."""
    N, D, prefix = 300, 128, 4096
    kw = dict(num_seqs=N, num_heads=H, num_kv_heads=HK, q_stride=H * D, kv_block_stride=HK * D * 16, kv_head_stride=D * 16,
              max_num_blocks_per_seq=400, max_seq_len=prefix + 1000)
    assert _route(prefix=prefix, **(kw)) == 3
    a, _ = _c_args(**kw)
    group = H // HK
    heads = min(group, 8 if group <= 8 else 16)
    items = N * HK * -(-group // heads)
    tiles = 2 * HK * -(--(-N // (128 // group)) // 2)
    prefix_parts = (tiles + 2 * 148) * 128 * (D * 4 + 8)
    own = (items + 16 * 148) * (heads * D * 4 + -(-heads * 8 // 16) * 16)
    assert capi.shared_prefix_scratch_bytes(a, prefix) <= prefix_parts + own + items * 8 + 4096
