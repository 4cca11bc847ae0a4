"""Engine steps as a model layer makes them of the operators together: queries and keys rotated and written to the
cache in one launch, then attention over a prefix that all requests share.  The reference attends, in 64 bits, to what
the cache holds (the writes have their own tests), so the tolerance is that of attention alone: P rounded to 16 bits,
half a step u of the operands' type (f16 for fp8 caches), its parts in fp32, the result rounded once, and, where a step's
rows go to the ordinary kernels, partials rounded to 16 bits in between: 2 u sum(p |v|) + 2 u_out |out| + 2^-16 sum(p |v|)."""
import types

import pytest
import torch

from vllm_b200 import _custom_ops as ops
from vllm_b200.backend import (B200PagedAttentionBackend, B200PagedAttentionImpl,
                               B200PagedAttentionMetadataBuilder)
from vllm_b200.paged_attn import PagedAttention

DEV = "cuda"


class Session:
    def __init__(self, N, prefix, own, H=8, HK=2, D=128, B=16, kv="auto", dtype=torch.bfloat16, neox=True, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.N, self.H, self.HK, self.D, self.B, self.kv, self.dtype, self.prefix = N, H, HK, D, B, kv, dtype, prefix
        self.g, self.neox = g, neox
        pb, per = prefix // B, -(-(max(own) + 700) // B)
        self.nb = pb + N * per
        perm = torch.randperm(self.nb, generator=g).to(torch.int32)
        table = torch.empty((N, pb + per), dtype=torch.int32)
        table[:, :pb] = perm[:pb]
        table[:, pb:] = perm[pb:].view(N, per)
        self.table = table.to(DEV)
        self.lens = torch.tensor([prefix + n for n in own])
        shape = B200PagedAttentionBackend.get_kv_cache_shape(self.nb, B, HK, D, kv)
        fill = torch.randn(shape, generator=g)
        self.cache = (fill * 2).to(torch.float8_e4m3fn).view(torch.uint8).to(DEV) if kv != "auto" else fill.to(dtype).to(DEV)
        one = torch.tensor(0.4 if kv != "auto" else 1.0, device=DEV)
        self.layer = types.SimpleNamespace(_k_scale=one, _v_scale=one)
        ang = torch.arange(prefix + 5000, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2) / (D // 2))
        self.rope = torch.cat([ang.cos(), ang.sin()], 1).float().to(DEV)
        self.impl = B200PagedAttentionImpl(H, D, D ** -0.5, HK, kv_cache_dtype=kv)
        self.builder = B200PagedAttentionMetadataBuilder(types.SimpleNamespace(block_size=B), ["l"], None, DEV)

    def step(self, new):
        """`new[r]` tokens of request r; returns (output, what it should be, sum of p |v|)."""
        N, H, HK, D, B = self.N, self.H, self.HK, self.D, self.B
        new = torch.tensor(new)
        n = int(new.sum())
        seq = torch.repeat_interleave(torch.arange(N), new)
        pos = torch.cat([torch.arange(int(a), int(a + t)) for a, t in zip(self.lens, new)])
        self.lens = self.lens + new
        slots = self.table.cpu()[seq, pos // B].long() * B + pos % B
        qkv = torch.randn(n, (H + 2 * HK) * D, generator=self.g).to(self.dtype).to(DEV)
        q, k, v = (t.view(n, -1, D) for t in qkv.split([H * D, HK * D, HK * D], 1))
        qsl = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).int()
        lens = self.lens.int().to(DEV)
        common = types.SimpleNamespace(
            query_start_loc=qsl.to(DEV), query_start_loc_cpu=qsl, seq_lens=lens, num_reqs=N, num_actual_tokens=n,
            max_query_len=int(new.max()), max_seq_len=int(self.lens.max()), block_table_tensor=self.table,
            slot_mapping=slots.to(DEV))
        shares = self.builder.use_cascade_attention(self.prefix, new.numpy(), H, HK, False, False, False, 148)
        md = self.builder.build(self.prefix if shares else 0, common)
        assert md.use_cascade == shares
        out = torch.full((n, H * D), 7.0, dtype=self.dtype, device=DEV)
        assert self.impl.fused_rope_kvcache_supported()
        self.impl.do_rope_and_kv_cache_update(self.layer, q, k, v, pos.to(DEV), self.rope, self.neox, self.cache,
                                              md.slot_mapping)
        assert self.impl.forward(self.layer, q, None, None, self.cache, md, output=out) is out
        kc, vc = PagedAttention.split_kv_cache(self.cache, HK, D)
        s = self.layer._k_scale.double()
        val = (lambda t: t.view(torch.float8_e4m3fn).double() * s) if self.kv != "auto" else (lambda t: t.double())
        want, mag = torch.zeros(2, n, H, D, dtype=torch.float64, device=DEV)
        for r in range(N):
            L, rows = int(self.lens[r]), slice(int(qsl[r]), int(qsl[r + 1]))
            b = self.table[r, :-(-L // B)].long()
            keys = val(kc[b].permute(0, 3, 1, 2, 4).reshape(-1, HK, D)[:L])
            vals = val(vc[b].permute(0, 3, 1, 2).reshape(-1, HK, D)[:L])
            z = torch.einsum("thgd,nhd->htgn", q[rows].double().view(-1, HK, H // HK, D), keys) * D ** -0.5
            t = z.shape[1]
            last = torch.arange(L - t, L, device=DEV)
            z = z.masked_fill(torch.arange(L, device=DEV)[None, None, None] > last[None, :, None, None], -torch.inf)
            p = torch.softmax(z, -1)
            want[rows] = torch.einsum("htgn,nhd->thgd", p, vals).reshape(t, H, D)
            mag[rows] = torch.einsum("htgn,nhd->thgd", p, vals.abs()).reshape(t, H, D)
        got = out.view(n, H, D)
        u_out = torch.finfo(self.dtype).eps / 2
        u_p = torch.finfo(torch.float16 if self.kv != "auto" else self.dtype).eps / 2
        # (16-bit partials of the ordinary kernels are of the query's type)
        tol = mag * (u_p + u_out + 2.0 ** -16) + want.abs() * 2 * u_out + 2.0 ** -22
        bad = (got.double() - want).abs() > tol
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())
        return md


@pytest.mark.gpu
@pytest.mark.parametrize("kv,dtype,neox", [("auto", torch.bfloat16, True), ("fp8", torch.float16, False)])
def test_decode_steps_behind_a_prompt(kv, dtype, neox):
    s = Session(40, 2048, [5 + 3 * i for i in range(40)], kv=kv, dtype=dtype, neox=neox)
    for _ in range(3):
        assert s.step([1] * 40).use_cascade


@pytest.mark.gpu
def test_steps_with_chunks_beside_the_decodes():
    s = Session(20, 1024, [3 + 11 * i for i in range(20)])
    assert s.step([1] * 17 + [40, 300, 1]).num_decodes == 17
    assert not s.step([30] * 20).use_cascade  # no decodes: an ordinary step
    assert not s.step([1] + [5] * 19).use_cascade
    s.step([1] * 20)


@pytest.mark.gpu
def test_shapes_of_the_ordinary_kernels():
    """Block size 8 and one request: the ordinary kernels, through the same calls."""
    s = Session(6, 64, [4, 9, 1, 30, 2, 8], B=8)
    s.step([1] * 6)
    s.step([1] * 4 + [7, 9])
    Session(1, 64, [4]).step([1])


@pytest.mark.gpu
def test_rows_behind_the_batch_stay():
    s = Session(12, 1024, list(range(12)))
    q = torch.randn(14, 8, 128, device=DEV).bfloat16()
    md = s.builder.build(1024, types.SimpleNamespace(
        query_start_loc=torch.arange(13, dtype=torch.int32, device=DEV), query_start_loc_cpu=torch.arange(13, dtype=torch.int32),
        seq_lens=(s.lens + 1).int().to(DEV), num_reqs=12, num_actual_tokens=12, max_query_len=1, max_seq_len=1036,
        block_table_tensor=s.table, slot_mapping=torch.zeros(12, dtype=torch.int64, device=DEV)))
    out = torch.full((14, 1024), 7.0, dtype=torch.bfloat16, device=DEV)
    s.impl.forward(s.layer, q, None, None, s.cache, md, output=out)
    assert (out[12:] == 7.0).all() and not (out[:12] == 7.0).all(dim=1).any()


def test_when_a_step_is_a_cascade():
    use = B200PagedAttentionBackend.use_cascade_attention
    args = dict(num_query_heads=8, num_kv_heads=2, use_alibi=False, use_sliding_window=False, use_local_attention=False,
                num_sms=148)
    assert use(256, [1, 1, 5], **args) and use(16, [1] * 300, **args, dcp_world_size=1)
    assert not use(0, [1, 1], **args) and not use(256, [1, 5], **args) and not use(256, [1], **args)
    assert not use(256, [1, 1], **(args | dict(use_sliding_window=True)))
    assert not use(256, [1, 1], **(args | dict(use_local_attention=True)))
    assert not use(256, [1, 1], **args, dcp_world_size=2)


def test_prefixes_that_are_refused():
    b = B200PagedAttentionMetadataBuilder(16)
    common = types.SimpleNamespace(
        query_start_loc=torch.tensor([0, 1, 2]), seq_lens=torch.tensor([70, 90]), num_reqs=2, num_actual_tokens=2,
        max_query_len=1, max_seq_len=90, block_table_tensor=torch.zeros(2, 6), slot_mapping=torch.zeros(2))
    assert b.build(64, common).common_prefix_len == 64
    for n in (60, 96):
        with pytest.raises(NotImplementedError, match="whole blocks"):
            b.build(n, common)


def test_key_and_value_go_together():
    impl = B200PagedAttentionImpl(8, 128, 0.1, 2)
    md = types.SimpleNamespace(num_actual_tokens=1)
    q = torch.zeros(1, 8, 128)
    with pytest.raises(AssertionError, match="go together"):
        impl.forward(None, q, q, None, None, md, output=torch.zeros(1, 1024))


@pytest.mark.gpu
def test_keys_behind_the_rotation_are_refused():
    """forward would write the unrotated keys over the rotated ones; the step after it may bring its own again."""
    s = Session(3, 64, [4, 9, 1])
    s.step([1] * 3)
    n = 3
    q, k, v = (torch.randn(n, h, s.D, generator=s.g).to(s.dtype).to(DEV) for h in (s.H, s.HK, s.HK))
    slots = (s.table[:, -1].long() * s.B).to(DEV)
    md = s.builder.build(0, types.SimpleNamespace(
        query_start_loc=torch.arange(4, dtype=torch.int32, device=DEV), seq_lens=s.lens.int().to(DEV), num_reqs=n,
        num_actual_tokens=n, max_query_len=1, max_seq_len=int(s.lens.max()), block_table_tensor=s.table, slot_mapping=slots))
    out = torch.full((n, s.H * s.D), 7.0, dtype=s.dtype, device=DEV)
    s.impl.do_rope_and_kv_cache_update(s.layer, q, k, v, s.lens.to(DEV), s.rope, True, s.cache, slots)
    cache = s.cache.clone()
    with pytest.raises(ValueError, match="key and value None"):
        s.impl.forward(s.layer, q, k, v, s.cache, md, output=out)
    torch.cuda.synchronize()
    assert torch.equal(s.cache, cache) and (out == 7.0).all()
    s.impl.do_rope_and_kv_cache_update(s.layer, q, k, v, s.lens.to(DEV), s.rope, True, s.cache, slots)
    s.impl.forward(s.layer, q, None, None, s.cache, md, output=out)
    s.impl.forward(s.layer, q, k, v, s.cache, md, output=out)


def test_keys_behind_the_rotation_are_refused_on_the_host(monkeypatch):
    impl = B200PagedAttentionImpl(8, 128, 0.1, 2)
    monkeypatch.setattr(PagedAttention, "rotate_and_write_to_paged_cache", lambda *a, **k: None)
    monkeypatch.setattr(ops, "attention_step", lambda *a: True)
    q, kv = torch.zeros(1, 8, 128), torch.zeros(1, 2, 128)
    md = types.SimpleNamespace(num_actual_tokens=1, num_decodes=1, max_query_len=1, max_seq_len=4, use_cascade=False,
                               block_table=None, seq_lens=None, slot_mapping=None, query_start_loc=None, common_prefix_len=0)
    layer = types.SimpleNamespace(_k_scale=None, _v_scale=None)
    cache, out = torch.zeros(2, 1, 16 * 2 * 128), torch.zeros(1, 1024)
    rotate = lambda: impl.do_rope_and_kv_cache_update(layer, q, kv, kv, None, None, True, cache, torch.zeros(1))  # noqa: E731
    rotate()
    with pytest.raises(ValueError, match="key and value None"):
        impl.forward(layer, q, kv, kv, cache, md, output=out)
    rotate()
    assert impl.forward(layer, q, None, None, cache, md, output=out) is out
    assert impl.forward(layer, q, kv, kv, cache, md, output=out) is out  # the next step, without the rotation


def _taken(monkeypatch):
    """What ops.attention_step answers, and the launches of it."""
    from vllm_b200 import capi
    step, taken = ops.attention_step, []

    def record(*args):
        capi.launch_count(reset=True)
        done = step(*args)
        taken.append((done, capi.launch_count()))
        return done
    monkeypatch.setattr(ops, "attention_step", record)
    return taken


@pytest.mark.gpu
@pytest.mark.parametrize("N,prefix", [(2, 16), (2, 256), (64, 16), (256, 16), (12, 64)])
@pytest.mark.parametrize("chunks", [0, 2])
def test_too_little_to_share_is_an_ordinary_step(monkeypatch, N, prefix, chunks):
    """A cascade step whose sizes leave nothing to share: the same native call, the same launches, the same bits."""
    taken = _taken(monkeypatch)
    s = Session(N + chunks, prefix, [1 + 3 * i % 50 for i in range(N + chunks)])
    md = s.step([1] * N + [9] * chunks)
    assert md.use_cascade
    out = [torch.empty((md.num_actual_tokens, s.H * s.D), dtype=s.dtype, device=DEV) for _ in range(2)]
    q = torch.randn((md.num_actual_tokens, s.H, s.D), generator=s.g).to(s.dtype).to(DEV)
    for o, shares in zip(out, (True, False)):
        md.use_cascade = shares
        s.impl.forward(s.layer, q, None, None, s.cache, md, output=o)
    assert taken[0] == taken[1] == taken[2] and taken[0][0]
    assert torch.equal(*out)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1] * 40, [1] * 40 + [30, 200]], ids=["decodes", "chunks"])
@pytest.mark.parametrize("write", [True, False])
def test_a_cascade_is_one_native_call(monkeypatch, new, write):
    """The write, the shared prefix and the chunks go with the step's call: as the operators one by one, to the last bit."""
    s = Session(len(new), 2048, [5 + 3 * i for i in range(len(new))])
    md = s.step(new)
    n = md.num_actual_tokens
    q, k, v = (torch.randn((n, h, s.D), generator=s.g).to(s.dtype).to(DEV) for h in (s.H, s.HK, s.HK))
    cache, taken = s.cache.clone(), _taken(monkeypatch)
    out = [torch.full((n + 3, s.H * s.D), 7.0, dtype=s.dtype, device=DEV) for _ in range(2)]
    kv = (k, v) if write else (None, None)
    s.impl.forward(s.layer, q, *kv, s.cache, md, output=out[0])
    done, launches = taken[0]
    assert done and launches > 1 + write + (len(new) > 40)
    monkeypatch.setattr(ops, "attention_step", lambda *args: False)
    s.impl.forward(s.layer, q, *kv, cache, md, output=out[1])
    assert torch.equal(*out) and torch.equal(s.cache, cache)
    assert (out[0][n:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1] * 40, [1] * 40 + [30, 200]], ids=["decodes", "chunks"])
def test_without_memory_for_the_scratch_a_cascade_is_an_ordinary_step(new):
    """An engine may have given all device memory to its cache: the step then shares nothing and raises nothing."""
    s = Session(len(new), 2048, [5 + 3 * i for i in range(len(new))])
    md = s.step(new)
    n = md.num_actual_tokens
    q = torch.randn((n, s.H, s.D), generator=s.g).to(s.dtype).to(DEV)
    out = [torch.empty((n, s.H * s.D), dtype=s.dtype, device=DEV) for _ in range(2)]
    md.use_cascade = False
    s.impl.forward(s.layer, q, None, None, s.cache, md, output=out[0])
    md.use_cascade = True
    torch.cuda.empty_cache()
    hold = []  # what is free inside the allocator's segments, down to less than any scratch
    torch.cuda.set_per_process_memory_fraction(1e-6)
    for size in (1 << 26, 1 << 23, 1 << 21, (1 << 20) + 1):
        try:
            while True:
                hold.append(torch.empty(size, dtype=torch.uint8, device=DEV))
        except torch.OutOfMemoryError:
            pass
    try:
        s.impl.forward(s.layer, q, None, None, s.cache, md, output=out[1])
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    torch.cuda.synchronize()
    assert torch.equal(*out)


@pytest.mark.gpu
def test_a_captured_step_holds_for_batches_without_the_prefix():
    """What is replayed may be any batch of as many decodes: a common prefix at capture says nothing about it."""
    s = Session(40, 2048, [5 + 3 * i for i in range(40)])
    md = s.step([1] * 40)
    assert md.use_cascade
    q = torch.randn((40, s.H, s.D), generator=s.g).to(s.dtype).to(DEV)
    out, want = (torch.empty((40, s.H * s.D), dtype=s.dtype, device=DEV) for _ in range(2))
    s.impl.forward(s.layer, q, None, None, s.cache, md, output=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.impl.forward(s.layer, q, None, None, s.cache, md, output=out)
    md.block_table.copy_(torch.randint(0, s.nb, md.block_table.shape, generator=s.g).int())
    md.use_cascade = False
    s.impl.forward(s.layer, q, None, None, s.cache, md, output=want)
    g.replay()
    torch.cuda.synchronize()
    assert (out.float() - want.float()).norm() <= 2e-2 * want.float().norm()


def test_the_step_is_told_the_prefix(monkeypatch):
    seen = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "attention_step", lambda *a: seen.append(a[-1]) or True)
    impl = B200PagedAttentionImpl(8, 128, 0.1, 2)
    q, out = torch.zeros(3, 8, 128), torch.zeros(3, 1024)
    layer = types.SimpleNamespace(_k_scale=None, _v_scale=None)
    b = B200PagedAttentionMetadataBuilder(16)
    common = types.SimpleNamespace(
        query_start_loc=torch.arange(4), seq_lens=torch.tensor([70, 90, 80]), num_reqs=3, num_actual_tokens=3,
        max_query_len=1, max_seq_len=90, block_table_tensor=torch.zeros(3, 6), slot_mapping=torch.zeros(3))
    for prefix in (64, 0):
        impl.forward(layer, q, None, None, torch.zeros(2, 6, 4096), b.build(prefix, common), output=out)
    assert seen == [64, 0]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    impl.forward(layer, q, None, None, torch.zeros(2, 6, 4096), b.build(64, common), output=out)
    assert seen == [64, 0, 0]
