"""torch.library.opcheck on the registered ops, as the reference's kernel tests do
(tests/kernels/utils.py:1062-1080 with the checks of :33-38)."""
import pytest
import torch

from vllm_b200 import _custom_ops
import workloads as W

pytestmark = pytest.mark.gpu
_custom_ops.claim_reference_names()  # the checks below address the ops by the reference's names
CHECKS = ("test_schema", "test_autograd_registration", "test_faketensor")


def _opcheck(op, args):
    torch.library.opcheck(op, args, test_utils=CHECKS, raise_exception=True)


def test_opcheck_attention_ops():
    w = W.small("cuda", seed=40, num_seqs=3, num_heads=8, num_kv_heads=2, max_len=700, num_blocks=128)
    out = torch.empty_like(w.query)
    tail = (w.query, w.key_cache, w.value_cache, w.num_kv_heads, w.scale, w.block_tables, w.seq_lens,
            w.block_size, w.max_seq_len, None, "auto", w.k_scale, w.v_scale, 0, 0, 0, 64, 0)
    _opcheck(torch.ops._C.paged_attention_v1, (out,) + tail)
    e, m, t = w.scratch()
    _opcheck(torch.ops._C.paged_attention_v2, (out, e, m, t) + tail)


def test_opcheck_cache_ops():
    T, H, D, B, NB = 20, 4, 64, 16, 8
    key = torch.randn(T, H, D, device="cuda", dtype=torch.bfloat16)
    val = torch.randn_like(key)
    slots = torch.randperm(NB * B, device="cuda")[:T]
    one = torch.tensor(1.0, device="cuda")
    kc = torch.zeros(NB, H, D // 8, B, 8, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros(NB, H, D, B, device="cuda", dtype=torch.bfloat16)
    _opcheck(torch.ops._C_cache_ops.reshape_and_cache, (key, val, kc, vc, slots, "auto", one, one))
    kf = torch.zeros(NB, B, H, D, device="cuda", dtype=torch.bfloat16)
    vf = torch.zeros_like(kf)
    _opcheck(torch.ops._C_cache_ops.reshape_and_cache_flash, (key, val, kf, vf, slots, "auto", one, one))
    q8 = torch.empty(T, H, D, device="cuda", dtype=torch.uint8)
    _opcheck(torch.ops._C_cache_ops.convert_fp8, (q8, key, 1.0, "fp8"))


def _rotary_args():
    gen = torch.Generator(device="cuda").manual_seed(3)
    T, H, HK, D, B, NB = 20, 4, 2, 64, 16, 8
    q, k, v = (torch.randn(T, h, D, generator=gen, device="cuda").bfloat16() for h in (H, HK, HK))
    slots = torch.randperm(NB * B, generator=gen, device="cuda")[:T]
    pos = torch.randint(0, 100, (T,), generator=gen, device="cuda")
    table = torch.randn(100, D, generator=gen, device="cuda")
    one = torch.tensor(1.0, device="cuda")
    return torch.empty_like(q), pos, q, k, v, table, True, slots, one, (NB, HK, D, B)


def test_opcheck_rotary_writes():
    out, pos, q, k, v, table, neox, slots, one, (NB, HK, D, B) = _rotary_args()
    kc = torch.zeros(NB, HK, D // 8, B, 8, device="cuda", dtype=torch.bfloat16)
    vc = torch.zeros(NB, HK, D, B, device="cuda", dtype=torch.bfloat16)
    ops = torch.ops._C_b200_cache_ops
    _opcheck(ops.rotary_reshape_and_cache, (out, pos, q, k, v, table, neox, kc, vc, slots, "auto", one, one))
    kf, vf = (torch.zeros(NB, B, HK, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    _opcheck(ops.rotary_reshape_and_cache_flash, (out, pos, q, k, v, table, neox, kf, vf, slots, "auto", one, one))


def test_opcheck_shared_prefix():
    w = W.small("cuda", seed=40, num_seqs=3, num_heads=8, num_kv_heads=2, max_len=700, num_blocks=128)
    w.block_tables[:, :4] = w.block_tables[0, :4].clone()
    out = torch.empty_like(w.query)
    lse = torch.empty(8, 3, device="cuda")
    for extra in ((), (lse,)):
        _opcheck(torch.ops._C_b200.paged_attention_shared_prefix,
                 (out, w.query, w.key_cache, w.value_cache, w.num_kv_heads, w.scale, w.block_tables, w.seq_lens,
                  4 * w.block_size, w.block_size, w.max_seq_len, None, "auto", w.k_scale, w.v_scale, *(extra or (None,))))
