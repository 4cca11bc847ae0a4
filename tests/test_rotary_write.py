"""rotary_reshape_and_cache[_flash]: queries and keys rotated on the way into the cache, against the
definition in 64 bits.

Tolerances.  One rotated value is a c - b s in fp32: the product b s is off by at most 2^-24 |b s|, the
fused product and sum by 2^-24 of the result, |c|, |s| <= 1 + 2^-8 (a rounded table); together less than
2^-22 (|a| + |b|).  Rounding to the output's type adds half a step: eps / 2 of the value; below the smallest
normal number steps are tiny = smallest_normal * eps wide whatever the value (fp16: 2^-14 * 2^-10 = 2^-24; a
rotated value of 2.5e-6 comes back up to 2^-25 = 3.0e-8 off, where eps / 2 of it would be 1.2e-9), so half of
that is added.  What is not rotated is exact, and equal to what
reshape_and_cache writes."""
import ctypes as C

import pytest
import torch

from vllm_b200 import _custom_ops as ops
from vllm_b200 import capi

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = {"fp8": (torch.float8_e4m3fn, 448.0), "fp8_e5m2": (torch.float8_e5m2, 57344.0)}


class Case:
    """Inputs of a call: runs of consecutive positions at random places, every token with a slot of its own."""

    def __init__(self, layout="x", runs=((0, 5),), H=4, HK=2, D=128, B=16, dtype="bf16", kv="auto", rot=None,
                 neox=True, table="fp32", scale=(0.013, 0.021), padded=0, packed=True, shift=0, seed=0, max_pos=3000):
        g = torch.Generator().manual_seed(seed)
        self.layout, self.H, self.HK, self.D, self.B, self.kv, self.neox = layout, H, HK, D, B, kv, neox
        self.rot, self.dtype = rot or D, DT[dtype]
        starts = torch.tensor([a for a, _ in runs])
        pos = torch.cat([torch.arange(a, a + n) for a, n in runs])
        seq = torch.cat([torch.full((n,), i) for i, (_, n) in enumerate(runs)])
        per = int((starts + torch.tensor([n for _, n in runs])).max() - 1) // B + 1
        self.nb = len(runs) * per + 3
        perm = torch.randperm(self.nb, generator=g)
        slots = perm[seq * per + pos // B] * B + pos % B
        self.n = len(pos)
        rows = self.n + padded
        shifts = torch.randint(0, max_pos - int(pos.max()), (len(runs),), generator=g)
        self.positions = torch.cat([pos + shifts[seq], torch.zeros(padded, dtype=torch.int64)]).to(DEV)
        self.slots = torch.cat([slots, torch.full((padded,), -1)]).to(DEV)
        w = (H + 2 * HK) * D if packed else max(H, HK) * D
        if packed:
            buf = torch.randn(rows * w + shift, generator=g).to(self.dtype).to(DEV)[shift:].view(rows, w)
            q, k, v = buf.split([H * D, HK * D, HK * D], dim=1)
        else:
            q, k, v = (torch.randn(rows * h * D + shift, generator=g).to(self.dtype).to(DEV)[shift:].view(rows, h * D)
                       for h in (H, HK, HK))
        self.q, self.k, self.v = q.view(rows, H, D), k.view(rows, HK, D), v.view(rows, HK, D)
        half = self.rot // 2
        ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half) / max(half, 1))
        self.table = torch.cat([ang.cos(), ang.sin()], 1).to(DT[table]).to(DEV)
        self.ks, self.vs = (torch.tensor(s, device=DEV) for s in scale)
        cd = torch.uint8 if kv != "auto" else self.dtype
        self.x = 16 // cd.itemsize
        fill = 7
        if layout == "x":
            self.kc = torch.full((self.nb, HK, D // self.x, B, self.x), fill, dtype=cd, device=DEV)
            self.vc = torch.full((self.nb, HK, D, B), fill, dtype=cd, device=DEV)
        else:
            shape = (self.nb, B, HK, D) if layout == "NHD" else (self.nb, HK, B, D)
            kc, vc = (torch.full(shape, fill, dtype=cd, device=DEV) for _ in range(2))
            self.kc, self.vc = (kc, vc) if layout == "NHD" else (kc.transpose(1, 2), vc.transpose(1, 2))
        self.out = torch.full((rows + 2, H, D), 3.0, dtype=self.dtype, device=DEV)

    def call(self, out=None, **kw):
        f = ops.rotary_reshape_and_cache if self.layout == "x" else ops.rotary_reshape_and_cache_flash
        a = dict(query_out=self.out if out is None else out, positions=self.positions, query=self.q, key=self.k,
                 value=self.v, cos_sin_cache=self.table, is_neox=self.neox, key_cache=self.kc, value_cache=self.vc,
                 slot_mapping=self.slots, kv_cache_dtype=self.kv, k_scale=self.ks, v_scale=self.vs)
        a.update(kw)
        f(**a)

    def rotated(self, x):
        """(values, |a| + |b|) in 64 bits; NaN where the position is outside the table."""
        x = x.double()
        known = (self.positions >= 0) & (self.positions < self.table.shape[0])
        t = self.table.double()[torch.where(known, self.positions, 0)]
        t[~known] = float("nan")
        half = self.rot // 2
        c, s = t[:, None, :half], t[:, None, half:]
        i = torch.arange(half, device=DEV)
        ia, ib = (i, i + half) if self.neox else (2 * i, 2 * i + 1)
        a, b = x[..., ia], x[..., ib]
        y, size = x.clone(), torch.zeros_like(x)
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = a.abs() + b.abs()
        return y, size

    def rows_of(self, cache):
        """[tokens, HK, D] of the tokens with a slot."""
        blk, off = self.slots[:self.n] // self.B, self.slots[:self.n] % self.B
        if self.layout != "x":
            return cache[blk, off]
        if cache.dim() == 5:
            return cache[blk, :, :, off].flatten(2)
        return cache[blk, :, :, off]

    def check(self, out=None):
        rows = self.slots.numel()
        out = self.out if out is None else out
        want, size = self.rotated(self.q)
        got = out[:rows].double()
        self._near(got, want, size, self.dtype)
        if out is self.out:
            assert (out[rows:] == 3.0).all()  # rows behind the last token
        # copies are exact
        assert torch.equal(out[:rows, :, self.rot:].view(torch.uint8), self.q[:, :, self.rot:].contiguous().view(torch.uint8))
        k, size = self.rotated(self.k)
        k, size = k[:self.n], size[:self.n]
        got = self.rows_of(self.kc)
        if self.kv == "auto":
            self._near(got.double(), k, size, self.dtype)
        else:
            t, top = F8[self.kv]
            s = float(self.ks)
            self._near(got.view(t).double(), (k / s).clamp(-top, top), size / s, t)
        # V, the copied part of K and every other byte of the caches: as reshape_and_cache writes them
        kc, vc = (torch.full_like(c, 7) for c in (self.kc, self.vc))
        write = ops.reshape_and_cache if self.layout == "x" else ops.reshape_and_cache_flash
        write(self.k[:rows], self.v[:rows], kc, vc, self.slots, self.kv, self.ks, self.vs)
        assert torch.equal(vc.view(torch.uint8), self.vc.view(torch.uint8))
        assert torch.equal(self.rows_of(kc)[..., self.rot:], got[..., self.rot:])
        kc2 = self.kc.clone()
        blk, off = self.slots[:self.n] // self.B, self.slots[:self.n] % self.B
        if self.layout == "x":
            kc2[blk, :, :, off] = 7
        else:
            kc2[blk, off] = 7
        assert (kc2 == 7).all()

    @staticmethod
    def _near(got, want, size, t):
        half_step = torch.finfo(t).eps / 2
        sub = torch.finfo(t).smallest_normal * half_step
        assert torch.equal(got.isnan(), want.isnan())
        bad = (got - want).abs() > want.abs() * half_step + size * 2.0 ** -22 * (1 + half_step) + sub
        assert not bad.any(), (bad.sum().item(), (got - want)[bad][:4], want[bad][:4])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["x", "NHD", "HND"])
@pytest.mark.parametrize("kv", ["auto", "fp8", "fp8_e5m2"])
@pytest.mark.parametrize("dtype,neox,rot", [("bf16", True, 128), ("fp16", False, 128), ("bf16", True, 32),
                                            ("bf16", False, 64), ("fp32", True, 128), ("fp16", True, 50)])
def test_types_layouts_and_pairs(layout, kv, dtype, neox, rot):
    for table in {dtype, "fp32"}:
        c = Case(layout, ((0, 40), (5, 1), (11, 33), (15, 2)), kv=kv, dtype=dtype, neox=neox, rot=rot, table=table,
                 padded=3)
        c.call()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 80, 96, 112, 120, 192, 256])
@pytest.mark.parametrize("kv,B", [("auto", 16), ("auto", 8), ("auto", 32), ("fp8", 16), ("fp8_e5m2", 32)])
def test_head_and_block_sizes(D, kv, B):
    if D == 120 and kv != "auto":
        pytest.skip("an fp8 cache keeps 16 head dimensions together")
    for layout in ("x", "NHD"):
        for neox in (True, False):
            c = Case(layout, ((3, 21), (0, 16), (31, 1)), H=6, HK=3, D=D, kv=kv, B=B, neox=neox, seed=D)
            c.call()
            c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("runs", [((0, 1),), ((7, 2),), ((0, 16),), ((0, 4096),), ((9, 4100),),
                                  tuple((17 * i, 1) for i in range(257)),
                                  tuple((i % 31, 1 + 7 * i % 90) for i in range(150))],
                         ids=["1", "2", "tile", "4096", "inside", "decode", "mixed"])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_lengths(runs, kv):
    for H, HK, layout in ((8, 2, "x"), (3, 1, "x"), (5, 5, "HND")):
        c = Case(layout, runs, H=H, HK=HK, kv=kv, padded=len(runs) % 3, max_pos=9000, table="bf16")
        c.call()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("shift,packed", [(1, True), (4, False), (8, True)])
@pytest.mark.parametrize("kv", ["auto", "fp8"])
def test_unaligned_tensors(shift, packed, kv):
    c = Case("x", ((2, 30), (0, 4)), kv=kv, shift=shift, packed=packed)
    c.call()
    c.check()
    c = Case("NHD", ((2, 30), (0, 4)), kv=kv, H=2, HK=1, D=80, shift=shift, packed=packed)
    c.call()
    c.check()


@pytest.mark.gpu
def test_strided_flash_caches():
    """K and V of a layer next to each other in one block, as some engines allocate them."""
    for kv in ("auto", "fp8"):
        c = Case("NHD", ((2, 30), (0, 4)), kv=kv)
        both = torch.full((c.nb, 2, c.B, c.HK, c.D), 7, dtype=c.kc.dtype, device=DEV)
        c.kc, c.vc = both[:, 0], both[:, 1]
        c.call()
        got = c.kc, c.vc
        c.kc, c.vc = (t.contiguous() for t in got)
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("neox", [True, False])
def test_in_place(neox):
    """The rotated query over the query itself, in the projection's own buffer."""
    for rot in (128, 64):
        c = Case("x", ((0, 70), (5, 1)), neox=neox, rot=rot)
        q0 = c.q.clone()
        c.call(out=c.q)
        got = c.q.clone()
        c.q = q0
        c.check(out=got)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (80, 50)])
def test_positions_outside_the_table(D, rot):
    """They read nothing and turn what they would have rotated into NaN; other tokens are not touched."""
    c = Case("x", ((0, 20),), D=D, rot=rot, max_pos=100)
    c.positions[3], c.positions[7], c.positions[19] = 100, -1, 1 << 62
    c.call()
    assert c.out[3, :, :rot].isnan().all() and c.out[7, :, :rot].isnan().all() and not c.out[4].isnan().any()
    c.check()


@pytest.mark.gpu
def test_values_that_overflow_and_nan():
    c = Case("x", ((0, 32),), kv="fp8", scale=(1e-6, 1e30))
    c.q[3, 1, 5], c.k[4, 0, 6], c.k[5, 1, 7] = float("inf"), float("nan"), 3e38
    c.call()
    k = c.rows_of(c.kc).view(torch.float8_e4m3fn).float()
    assert k[4, 0, 6].isnan() and k[4, 0, 70].isnan() and not k[3].isnan().any()
    big = c.rotated(c.k)[0][:32] / 1e-6
    ok = (big.abs() > 500) & big.isfinite()
    assert (k[ok].abs() == 448).all() and (k[ok].sign() == big[ok].sign()).all()
    assert c.out[3, 1, [5, 69]].isfinite().sum() == 0 and c.out[2].isfinite().all()
    v = c.rows_of(c.vc)
    assert ((v & 0x7F) == 0).all()


@pytest.mark.gpu
def test_no_tokens_and_few_heads():
    c = Case("x", ((0, 5),), H=1, HK=1)
    c.call(slot_mapping=c.slots[:0])
    assert (c.out == 3.0).all() and (c.kc == 7).all()
    c.call()
    c.check()


@pytest.mark.gpu
def test_other_stream_and_captured_replays():
    c = Case("x", ((0, 60), (3, 1)), kv="fp8", padded=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.call()
    s.synchronize()
    c.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.call()
    for seed in (3, 4):
        d = Case("x", ((0, 60), (3, 1)), kv="fp8", padded=2, seed=seed)
        for name in ("positions", "slots", "q", "k", "v", "kc", "vc", "out"):
            getattr(c, name).copy_(getattr(d, name))
        g.replay()
        torch.cuda.synchronize()
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("what,kw,msg", [
    ("table", lambda c: dict(cos_sin_cache=c.table[:, :127].contiguous()), "rot_dim"),
    ("table type", lambda c: dict(cos_sin_cache=c.table.half()), "cos_sin_cache"),
    ("table strides", lambda c: dict(cos_sin_cache=c.table[:, :64]), "cos_sin_cache"),
    ("positions type", lambda c: dict(positions=c.positions.int()), "positions"),
    ("positions count", lambda c: dict(positions=c.positions[:-1]), "positions"),
    ("query type", lambda c: dict(query=c.q.half()), "query"),
    ("query heads", lambda c: dict(query=c.q[:, :3]), "query"),
    ("query rows", lambda c: dict(query=c.q[:-1]), "query"),
    ("out rows", lambda c: dict(query_out=c.out[:1].expand(20, -1, -1)), "overlap"),
    ("key rows", lambda c: dict(key=c.k[:-1]), "key"),
    ("value heads", lambda c: dict(value=c.v[:, :1]), "value"),
    ("cache heads", lambda c: dict(key_cache=c.kc[:, :1].contiguous(), value_cache=c.vc[:, :1].contiguous()), "heads"),
    ("cache type", lambda c: dict(kv_cache_dtype="fp8"), "1-byte"),
    ("kv name", lambda c: dict(kv_cache_dtype="int4"), "Unsupported data type"),
    ("host tensor", lambda c: dict(positions=c.positions.cpu()), "positions"),
])
def test_refusals(what, kw, msg):
    c = Case("x", ((0, 20),))
    with pytest.raises((RuntimeError, NotImplementedError), match=msg):
        c.call(**kw(c))
    torch.cuda.synchronize()
    assert (c.out == 3.0).all() and (c.kc == 7).all() and (c.vc == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout,spoil", [
    ("x", lambda v: v.view(-1, 2, 64, 32)), ("x", lambda v: v.view(-1, 2, 256, 8)), ("x", lambda v: v.view(-1, 1, 128, 32)),
    ("x", lambda v: v[:-1]),
    ("NHD", lambda v: v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)),  # as HND in memory
    ("HND", lambda v: v.contiguous()), ("NHD", lambda v: v.view(-1, 32, 1, 128)), ("NHD", lambda v: v.view(-1, 8, 4, 128)),
    ("NHD", lambda v: v[:-1]),
])
def test_caches_of_two_layouts_are_refused(layout, spoil):
    """As many elements, and blocks as far apart, but V's in other places than K's."""
    c = Case(layout, ((0, 20),))
    vc = spoil(c.vc)
    with pytest.raises(RuntimeError, match="same|stride"):
        c.call(value_cache=vc)
    torch.cuda.synchronize()
    assert (c.out == 3.0).all() and (c.kc == 7).all() and (vc == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_strides_of_dimensions_of_size_one_mean_nothing(layout):
    """One kv head: NHD and HND caches are the same bytes, whatever strides they name."""
    c = Case(layout, ((0, 20),), HK=1)
    other = torch.full((c.nb, 1, c.B, c.D), 7, dtype=c.vc.dtype, device=DEV).transpose(1, 2)
    c.vc = other if layout == "NHD" else other.contiguous().view(c.nb, c.B, 1, c.D)
    c.call()
    c.check()


def _c_args(**kw):
    buf = C.create_string_buffer(1024)
    mem = C.addressof(buf) + 255 & ~255  # (any aligned address: nothing is launched)
    r = capi.RotaryArgs(query_out=mem, query=mem, positions=mem, cos_sin=mem, query_out_stride=512, query_stride=512,
                        max_position=100, num_heads=4, rot_dim=128, neighbours=0, table_dtype=capi.F32)
    a = capi.CacheArgs(key=mem, value=mem, key_cache=mem, value_cache=mem, slot_mapping=mem, key_stride=256,
                       value_stride=256, num_tokens=3, num_heads=2, head_size=128, block_size=16, x=8,
                       in_dtype=capi.BF16, kv_dtype=0)
    for k, v in kw.items():
        setattr(r if hasattr(r, k) and k != "num_heads" else a, k, v)
    return r, a, buf


@pytest.mark.parametrize("kw,msg", [
    (dict(rot_dim=130), "rot_dim"), (dict(rot_dim=7), "rot_dim"), (dict(rot_dim=0), "rot_dim"),
    (dict(max_position=0), "table is empty"), (dict(table_dtype=capi.F16), "rotation table"),
    (dict(num_tokens=-1), "bad sizes"), (dict(x=7), "multiple of x"), (dict(in_dtype=9), "Unsupported input type"),
    (dict(kv_dtype=9), "Unsupported data type"), (dict(query_out=None), "null tensor"), (dict(key=None), "null tensor"),
    (dict(positions=None), "null tensor"), (dict(kv_dtype=capi.KV_FP8_E4M3), "k_scale"),
])
def test_the_c_interface_refuses(kw, msg):
    r, a, _ = _c_args(**kw)
    capi.launch_count(reset=True)
    with pytest.raises(RuntimeError, match=msg):
        capi.rotary_reshape_and_cache(r, a)
    assert capi.launch_count() == 0


@pytest.mark.parametrize("out,stride", [(8, 512), (-8, 512), (512, 512), (-512, 512), (0, 520), (511, 2048),
                                        (4096, 512), (4097 - 512, 512), (4096 + 255, 512), (8192, 512), (8192 - 1024, 1024)])
def test_the_c_interface_refuses_a_query_out_over_its_inputs(out, stride):
    """Element offsets of query_out: over query (rows of 512 from 0 on, 2048 apart), key (256 from 4096) and value (from
    8192), 3 rows each.  (Nothing runs: the addresses are the test's own.)"""
    r, a, buf = _c_args()
    base = r.query
    a.key, a.value = base + 2 * 4096 * 2, base + 2 * 8192 * 2
    r.query_stride = 2048 if stride == 2048 else 512
    r.query_out, r.query_out_stride = base + 2 * out, stride
    if out >= 4096 - 512:
        a.key, a.value = base + 2 * 4096, base + 2 * 8192
    capi.launch_count(reset=True)
    with pytest.raises(RuntimeError, match="must not overlap"):
        capi.rotary_reshape_and_cache(r, a)
    assert capi.launch_count() == 0


@pytest.mark.parametrize("stride", [0, 511, -512])
def test_the_c_interface_refuses_rows_of_query_out_over_each_other(stride):
    r, a, _ = _c_args(query_out_stride=stride, query_stride=stride)
    a.key = a.value = r.query + 65536
    with pytest.raises(RuntimeError, match="must not overlap"):
        capi.rotary_reshape_and_cache(r, a)
    a.num_tokens, a.key_cache = 1, None  # (one row: the stride means nothing; refused for the cache, not launched)
    with pytest.raises(RuntimeError, match="null tensor"):
        capi.rotary_reshape_and_cache(r, a)


@pytest.mark.gpu
def test_outputs_beside_the_inputs():
    """query_out in the same buffer as the projection's output, in columns of its own: no overlap."""
    for H, HK in ((4, 2), (8, 1)):
        c = Case("x", ((0, 70), (5, 1)), H=H, HK=HK)
        n, w = c.slots.numel(), (H + 2 * HK) * c.D
        buf = torch.randn(n, w + H * c.D, device=DEV).to(c.dtype)
        buf[:, :w] = torch.cat([c.q, c.k, c.v], 1).view(n, w)
        parts = buf.split([H * c.D, HK * c.D, HK * c.D, H * c.D], 1)
        c.q, c.k, c.v, out = (t.view(n, -1, c.D) for t in parts)
        c.call(out=out)
        c.check(out=out)
        with pytest.raises(RuntimeError, match="must not overlap"):
            c.call(out=buf[:, c.D:].split(H * c.D, 1)[0].view(n, H, c.D))


def test_the_c_interface_takes_nothing_to_do():
    r, a, _ = _c_args(num_tokens=0, query=None, key=None)
    capi.rotary_reshape_and_cache(r, a)
    capi.rotary_reshape_and_cache_flash(r, a)
    assert capi.lib().b200pa_rotary_reshape_and_cache(None, None, None) == -1
