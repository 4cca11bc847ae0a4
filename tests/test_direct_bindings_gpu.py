"""The direct bindings of _custom_ops: whatever has to see an operator - tracers, dispatch modes, the
profiler, function transforms, the operators' own checks - sees it as through torch.ops."""
import pytest
import torch

from vllm_b200 import _custom_ops as ops
import workloads as W

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _write_args():
    gen = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.randn(5, 2, 64, generator=gen, device=DEV).bfloat16() for _ in range(2))
    kc = torch.zeros(4, 2, 8, 16, 8, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros(4, 2, 64, 16, dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor([3, 17, 40, 41, 63], device=DEV)
    one = torch.tensor(1.0, device=DEV)
    return k, v, kc, vc, slots, one


def _write(k, v, kc, vc, slots, one):
    ops.reshape_and_cache(k, v, kc, vc, slots, "auto", one, one)
    return kc


def test_a_dispatch_mode_sees_the_operators():
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    args = _write_args()
    with Record():
        _write(*args)
    assert seen == ["_C_b200_cache_ops.reshape_and_cache.default"]
    assert args[2].any()


def test_the_profiler_sees_the_operators():
    from torch.profiler import ProfilerActivity, profile
    w = W.small(DEV, num_seqs=2, max_len=100, num_blocks=64)
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        W.run_attention(w, version="v1")
        _write(*_write_args())
    names = {e.key for e in prof.key_averages()}
    assert {"_C_b200::paged_attention_v1", "_C_b200_cache_ops::reshape_and_cache"} <= names


def test_tracing_does_not_lose_an_operator():
    """torch.jit.trace refuses these schemas (anonymous alias sets); it must not record a graph without
    the write instead."""
    k, v, kc, vc, slots, one = _write_args()

    def through(write):
        def f(k, v, kc, vc):
            write(k, v, kc, vc, slots, "auto", one, one)
            return kc
        return f
    for write in (torch.ops._C_b200_cache_ops.reshape_and_cache, ops.reshape_and_cache):
        try:
            traced = torch.jit.trace(through(write), (k, v, kc, vc), check_trace=False)
        except RuntimeError:
            continue
        assert "reshape_and_cache" in str(traced.graph)


def test_a_compiled_function_keeps_its_operators():
    eager, compiled = _write_args(), _write_args()
    _write(*eager)
    torch.compile(_write, fullgraph=True, backend="eager")(*compiled)
    assert torch.equal(eager[2], compiled[2]) and torch.equal(eager[3], compiled[3]) and eager[2].any()


def test_function_transforms_are_refused_as_by_the_operators():
    k, v, kc, vc, slots, one = _write_args()
    batch = [t.unsqueeze(0).repeat(2, *[1] * t.dim()) for t in (k, v, kc, vc)]

    def through(write):
        def f(k, v, kc, vc):
            write(k, v, kc, vc, slots, "auto", one, one)
            return kc
        return f
    for write in (torch.ops._C_b200_cache_ops.reshape_and_cache, ops.reshape_and_cache):
        with pytest.raises(RuntimeError):
            torch.vmap(through(write))(*batch)
    assert not batch[2].any()


@pytest.mark.parametrize("spoil", ["slots dtype", "cpu cache", "kv type", "cache dtype", "strided heads"])
def test_wrong_arguments_raise_what_the_operators_raise(spoil):
    k, v, kc, vc, slots, one = _write_args()
    kv = "auto"
    if spoil == "slots dtype":
        slots = slots.int()
    elif spoil == "cpu cache":
        kc = kc.cpu()
    elif spoil == "kv type":
        kv = "int3"
    elif spoil == "cache dtype":
        kc = kc.half()
    else:
        k = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=DEV)[:, ::2]
    errors = []
    for write in (torch.ops._C_b200_cache_ops.reshape_and_cache, ops.reshape_and_cache):
        with pytest.raises((RuntimeError, NotImplementedError)) as e:
            write(k, v, kc, vc, slots, kv, one, one)
        errors.append((type(e.value), str(e.value).splitlines()[0]))
    assert errors[0] == errors[1]
    assert not vc.any()


# ------------------------------------------------------------------ the rotation with the KV write, the shared prefix
def _rotary_args():
    gen = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(5, 4, 64, generator=gen, device=DEV).bfloat16()
    pos = torch.tensor([3, 17, 8, 9, 31], device=DEV)
    table = torch.randn(40, 64, generator=gen, device=DEV)
    k, v, kc, vc, slots, one = _write_args()
    return dict(query_out=torch.zeros_like(q), positions=pos, query=q, key=k, value=v, cos_sin_cache=table, is_neox=True,
                key_cache=kc, value_cache=vc, slot_mapping=slots, kv_cache_dtype="auto", k_scale=one, v_scale=one)


def _flash_args():
    a = _rotary_args()
    return a | {n: torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=DEV) for n in ("key_cache", "value_cache")}


def _shared_args():
    gen = torch.Generator(device=DEV).manual_seed(2)
    N, H, HK, D, B, pb = 40, 8, 2, 128, 16, 256
    nb = pb + N
    bt = torch.cat([torch.arange(pb).expand(N, -1), pb + torch.arange(N)[:, None]], 1).int().to(DEV)
    kc, vc = (torch.randn(s, generator=gen, device=DEV).bfloat16() for s in ((nb, HK, D // 8, B, 8), (nb, HK, D, B)))
    q = torch.randn(N, H, D, generator=gen, device=DEV).bfloat16()
    one = torch.tensor(1.0, device=DEV)
    lens = (pb * B + 1 + torch.arange(N, device=DEV) % 16).int()
    return dict(out=torch.zeros_like(q), query=q, key_cache=kc, value_cache=vc, num_kv_heads=HK, scale=0.1, block_tables=bt,
                seq_lens=lens, prefix_len=pb * B, block_size=B, max_seq_len=pb * B + 16, alibi_slopes=None,
                kv_cache_dtype="auto", k_scale=one, v_scale=one, lse=torch.zeros(H, N, device=DEV))


NEW = [("_C_b200_cache_ops", "rotary_reshape_and_cache", _rotary_args, ("query_out", "key_cache", "value_cache")),
       ("_C_b200_cache_ops", "rotary_reshape_and_cache_flash", _flash_args, ("query_out", "key_cache", "value_cache")),
       ("_C_b200", "paged_attention_shared_prefix", _shared_args, ("out", "lse"))]
new_ops = pytest.mark.parametrize("space,name,make,outs", NEW, ids=[n[1] for n in NEW])


def _both(space, name):
    return getattr(getattr(torch.ops, space), name), getattr(ops, name)


@new_ops
def test_the_registered_operators_do_the_same(space, name, make, outs):
    a, b = make(), make()
    registered, wrapper = _both(space, name)
    registered(*a.values())
    wrapper(*b.values())
    assert all(torch.equal(a[n], b[n]) and a[n].any() for n in outs)


@new_ops
def test_modes_and_the_profiler_see_the_new_operators(space, name, make, outs):
    from torch.profiler import ProfilerActivity, profile
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    a = make()
    with Record():
        getattr(ops, name)(**a)
    assert seen == [f"{space}.{name}.default"] and all(a[n].any() for n in outs)
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        getattr(ops, name)(**a)
    assert f"{space}::{name}" in {e.key for e in prof.key_averages()}


@new_ops
def test_a_compiled_function_keeps_the_new_operators(space, name, make, outs):
    eager, compiled = make(), make()

    def f(a):
        getattr(ops, name)(**a)
        return a[outs[0]]
    f(eager)
    torch.compile(f, fullgraph=True, backend="eager")(compiled)
    assert all(torch.equal(eager[n], compiled[n]) and eager[n].any() for n in outs)


@new_ops
def test_function_transforms_refuse_the_new_operators(space, name, make, outs):
    for call in _both(space, name):
        a = make()
        batch = {n: t.unsqueeze(0).repeat(2, *[1] * t.dim()) for n, t in a.items() if n in (*outs, "query")}

        def f(*t):
            call(*(a | dict(zip(batch, t))).values())
            return t[0]
        with pytest.raises(RuntimeError):
            torch.vmap(f)(*batch.values())
        assert not any(batch[n].any() for n in outs)


@new_ops
@pytest.mark.parametrize("spoil", ["cpu cache", "kv type", "cache type", "query type", "whole dtype"])
def test_wrong_arguments_raise_what_the_new_operators_raise(space, name, make, outs, spoil):
    errors = []
    for call in _both(space, name):
        a = make()
        if spoil == "cpu cache":
            a["key_cache"] = a["key_cache"].cpu()
        elif spoil == "kv type":
            a["kv_cache_dtype"] = "int3"
        elif spoil == "cache type":
            a["value_cache"] = a["value_cache"].half()
        elif spoil == "query type":
            a["query"] = a["query"].double()
        else:
            whole = "block_tables" if "block_tables" in a else "slot_mapping"
            a[whole] = a[whole].short()
        with pytest.raises((RuntimeError, NotImplementedError)) as e:
            call(*a.values())
        errors.append((type(e.value), str(e.value).splitlines()[0]))
        assert not any(a[n].any() for n in outs if n in ("query_out", "out", "lse"))
    assert errors[0] == errors[1]
