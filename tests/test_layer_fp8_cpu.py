"""Host logic of rotary positions, the e4m3 store and attention over the e4m3 cache: what is refused, the
frequencies of scaled rotations, and the formulas the GPU tests compare with. No GPU work."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import layer_reference as ref
from kvoff import _lib, ops

P = ctypes.c_void_p(256)


def rotary(**change):
    a = dict(q=P, qs=512, qo=P, qos=512, hq=4, k=P, ks=512, ko=P, kos=512, hk=2, dim=64, rot=64, dtype=_lib.BF16,
             pos=P, pb=8, table=P, rows=10, n=3, flags=0, bad=None, stream=None) | change
    return _lib.lib().kvoff_rotary(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(n=-1), "sizes"), (dict(hq=0, hk=0), "sizes"), (dict(hk=-1), "sizes"), (dict(dim=0), "sizes"),
    (dict(qs=-2), "sizes"), (dict(rows=-1), "sizes"), (dict(rot=63), "even"), (dict(rot=66), "at most"),
    (dict(rot=0), "even"), (dict(dtype=7), "dtype"), (dict(pb=2), "int64"), (dict(flags=8), "flags"),
    (dict(q=None), "null"), (dict(ko=None), "null"), (dict(pos=None), "null"), (dict(table=None), "null"),
    (dict(q=ctypes.c_void_p(257)), "aligned"), (dict(flags=1, dim=65), "even number"),
    (dict(flags=1, qs=514), "aligned"), (dict(n=2 ** 31), "exceed"), (dict(hq=65000, dim=65000), "exceed"),
    (dict(qos=256), "overlap"), (dict(kos=128), "overlap"), (dict(qs=1024), "in place"), (dict(kos=1024), "in place"),
])
def test_rotary_refuses(change, message):
    assert rotary(**change) == _lib.KVOFF_EINVAL
    assert message in _lib.last_error()


def store(**change):
    a = dict(key=P, ks=1024, value=P, vs=1024, kc=P, vc=P, kscale=P, vscale=P, heads=2, dim=64, dtype=_lib.BF16,
             block=16, slots=P, n=3, num_slots=64, bad=None, stream=None) | change
    return _lib.lib().kvoff_store_kvcache_fp8(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(n=-1), "sizes"), (dict(heads=0), "sizes"), (dict(num_slots=-16), "sizes"), (dict(ks=-16), "sizes"),
    (dict(dim=60), "multiple of 8"), (dict(dim=264), "multiple of 8"), (dict(dim=0), "multiple of 8"),
    (dict(dtype=_lib.FP32), "bf16 or fp16"), (dict(block=24), "power of two"), (dict(block=0), "power of two"),
    (dict(block=8192, num_slots=8192), "power of two"), (dict(num_slots=72), "divides"),
    (dict(num_slots=2 ** 31), "int32"), (dict(n=65537), "exceed"), (dict(key=None), "null"),
    (dict(vscale=None), "null"), (dict(slots=None), "null"), (dict(key=ctypes.c_void_p(264)), "aligned"),
    (dict(vs=1032), "aligned"), (dict(kc=ctypes.c_void_p(260)), "aligned"),
])
def test_store_refuses(change, message):
    assert store(**change) == _lib.KVOFF_EINVAL
    assert message in _lib.last_error()


def attention(**change):
    a = dict(q=P, qs=1024, out=P, os=1024, lse=None, kc=P, vc=P, ks=P, vs=P, pages=4, page=32, block=16, tables=P,
             stride=4, width=4, contexts=P, starts=None, seqs=2, n=2, most=1, hq=4, hk=2, dim=64, dtype=_lib.BF16,
             scale=0.125, ws=None, wsb=0, stream=None) | change
    return _lib.lib().kvoff_attention_fp8(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(pages=-1), "sizes"), (dict(width=-1), "sizes"), (dict(n=-1), "sizes"), (dict(seqs=-1), "sizes"),
    (dict(qs=-16), "sizes"), (dict(stride=-4), "sizes"), (dict(page=0), "sizes"), (dict(hk=0), "sizes"),
    (dict(dim=96), "64 or 128"), (dict(hq=5), "divide"), (dict(page=24), "multiple of 16"),
    (dict(width=2 ** 27), "sizes"), (dict(block=8), "scale block"), (dict(block=48, page=48), "scale block"),
    (dict(block=64), "scale block"), (dict(dtype=_lib.FP32), "bf16 or fp16"), (dict(n=3), "one token"),
    (dict(most=2), "one token"), (dict(q=None), "null"), (dict(contexts=None), "null"), (dict(tables=None), "null"),
    (dict(vs=None), "null"), (dict(q=ctypes.c_void_p(264)), "aligned"), (dict(vc=ctypes.c_void_p(264)), "aligned"),
    (dict(out=ctypes.c_void_p(258)), "aligned"), (dict(qs=1032), "aligned"),
    (dict(starts=P, most=0), "max_seqlen_q"), (dict(scale=0.0), "softmax_scale"), (dict(scale=-1.0), "softmax_scale"),
    (dict(scale=math.nan), "softmax_scale"), (dict(scale=math.inf), "softmax_scale"),
    (dict(starts=P, most=2 ** 30), "32 bits"), (dict(starts=P, n=2 ** 30), "32 bits"), (dict(os=256), "overlap"),
])
def test_attention_refuses(change, message):
    assert attention(**change) == _lib.KVOFF_EINVAL
    assert message in _lib.last_error()


def test_the_stride_of_one_row_means_nothing():
    x = torch.zeros(4, 64, 1, dtype=torch.bfloat16).permute(2, 0, 1)
    assert x.stride(0) == 1 and ops._rows(x, "x") == 4 * 64 * 2
    assert ops._rows(torch.zeros(3, 6, 64)[:, :4], "x", 4) == 6 * 64 * 4


def test_empty_calls_are_accepted_without_a_device():
    assert rotary(n=0, q=None, k=None) == _lib.KVOFF_OK
    assert store(n=0, key=None) == _lib.KVOFF_OK
    assert attention(seqs=0, n=0, q=None) == _lib.KVOFF_OK


@pytest.mark.parametrize("name,args", [("rotary", 21), ("store_kvcache_fp8", 17), ("attention_fp8", 28)])
def test_packed_forms_reach_the_same_checks(name, args):
    packed = getattr(_lib.lib(), f"kvoff_{name}_packed")
    assert packed(None) == _lib.KVOFF_EINVAL and "null" in _lib.last_error()
    values = (ctypes.c_int64 * args)(*([-1] * args))
    assert packed(ctypes.cast(values, ctypes.c_char_p)) == _lib.KVOFF_EINVAL
    assert f"kvoff_{name}: bad sizes" in _lib.last_error()
    _lib.debug_fail_next(name)
    assert packed(ctypes.cast(values, ctypes.c_char_p)) == _lib.KVOFF_EINJECTED


@pytest.mark.parametrize("op,fn", [("rotary", rotary), ("store_kvcache_fp8", store), ("attention_fp8", attention)])
def test_injected_failures(op, fn):
    _lib.debug_fail_next(op)
    assert fn(n=0) == _lib.KVOFF_EINJECTED
    assert "injected" in _lib.last_error()


def tensors():
    x = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(2, 32, 4, 64).to(torch.float8_e4m3fn)
    scale = torch.zeros(2, 2, 4)
    return x, cache, scale


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def test_ops_refuse_tensors_of_other_kinds():
    x, cache, scale = tensors()
    table, positions = ops.rotary_table(8, 64), torch.arange(3)
    wrong = [
        (dict(k=x[:2]), "same tokens"), (dict(k=x.half()), "dtype"), (dict(positions=positions[:2]), "positions"),
        (dict(positions=positions.float()), "positions"), (dict(table=table.double()), "table"),
        (dict(table=table.T), "table"), (dict(out=(x[:2], x)), "shapes"), (dict(), "CUDA"),
    ]
    for change, message in wrong:
        a = dict(q=x, k=x, positions=positions, table=table) | change
        with pytest.raises(ValueError, match=message):
            ops.rotary(**a)
    slots = int32([0, 1, 2])
    wrong = [
        (dict(value=x[:2]), "shapes"), (dict(key=x.float(), value=x.float()), "bf16 or fp16"),
        (dict(v_cache=cache[:1]), "alike"), (dict(k_cache=cache.view(torch.uint8)), "float8"),
        (dict(v_scale=scale[:, :1]), "scales"), (dict(k_scale=scale.double()), "fp32"),
        (dict(k_cache=cache.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
        (dict(slot_mapping=slots.long()), "slot_mapping"), (dict(slot_mapping=slots[:2]), "slot_mapping"),
        (dict(key=x[:, :2], value=x[:, :2]), "rows"), (dict(), "CUDA"),
    ]
    for change, message in wrong:
        a = dict(key=x, value=x, k_cache=cache, v_cache=cache, k_scale=scale, v_scale=scale, slot_mapping=slots)
        with pytest.raises(ValueError, match=message):
            ops.store_kvcache_fp8(**(a | change))
    tables, contexts = int32([[0, 1]] * 3), int32([1, 2, 3])
    wrong = [
        (dict(q=x.float()), "bf16 or fp16"), (dict(q=x[..., :32]), "head_dim"),
        (dict(block_tables=tables.long()), "block_tables"), (dict(block_tables=tables[0]), "block_tables"),
        (dict(context_lens=contexts[:2]), "context_lens"), (dict(context_lens=contexts.long()), "context_lens"),
        (dict(), "CUDA"),
    ]
    for change, message in wrong:
        a = dict(q=x, k_cache=cache, v_cache=cache, k_scale=scale, v_scale=scale, block_tables=tables,
                 context_lens=contexts)
        with pytest.raises(ValueError, match=message):
            ops.attention_fp8(**(a | change))
    for bad in (x.transpose(0, 1), x[:, ::2], x[..., ::2]):
        with pytest.raises(ValueError, match="dense"):
            ops._rows(bad, "q")


def test_rotary_tables():
    table = ops.rotary_table(5000, 8, base=100.0)
    assert table.shape == (5000, 8) and table.dtype == torch.float32
    for p in (0, 1, 4999):
        for j in range(4):
            angle = p * 100.0 ** (-2 * j / 8)
            assert abs(table[p, j].item() - math.cos(angle)) <= 2.0 ** -24
            assert abs(table[p, 4 + j].item() - math.sin(angle)) <= 2.0 ** -24
    linear = ops.rotary_table(100, 8, base=100.0, scaling={"type": "linear", "factor": 4.0})
    assert torch.allclose(linear[::4], table[:25], atol=2.0 ** -23)
    # NTK: the slowest pair turns as if stretched by the factor, the fastest as before.
    ntk = ops.rotary_table(3, 8, base=100.0, scaling={"rope_type": "ntk", "factor": 4.0})
    assert abs(math.acos(ntk[1, 3].item()) - 100.0 ** -0.75 / 4) <= 1e-5
    assert abs(ntk[1, 0].item() - math.cos(1.0)) <= 2.0 ** -24


def test_rotary_tables_for_long_contexts():
    plain = ops.rotary_table(2, 128, base=1e4).double()
    angle = torch.atan2(plain[1, 64:], plain[1, :64])
    turns = 4096 * angle / (2 * math.pi)
    yarn = ops.rotary_table(2, 128, base=1e4, scaling={"type": "yarn", "factor": 8.0,
                                                       "original_max_position_embeddings": 4096}).double()
    stretch = 0.1 * math.log(8.0) + 1
    assert torch.allclose(yarn[1, :64] ** 2 + yarn[1, 64:] ** 2, torch.full((64,), stretch ** 2, dtype=torch.float64))
    got = torch.atan2(yarn[1, 64:], yarn[1, :64])
    # The ramp ends at whole pairs next to 32 turns and 1 turn.
    pair = lambda t: 64 * math.log(4096 / (t * 2 * math.pi)) / math.log(1e4)  # noqa: E731
    fast, slow = torch.arange(64) <= math.floor(pair(32)), torch.arange(64) >= math.ceil(pair(1))
    assert torch.allclose(got[fast], angle[fast], rtol=1e-6) and (turns[fast] >= 32).all()
    assert torch.allclose(got[slow], angle[slow] / 8, rtol=1e-4) and (turns[slow] <= 1).all()
    between = got[~fast & ~slow] / angle[~fast & ~slow]
    assert (between.diff() < 0).all() and between.max() < 1 and between.min() > 1 / 8
    scaling = {"type": "llama3", "factor": 8.0, "original_max_position_embeddings": 4096, "low_freq_factor": 1.0,
               "high_freq_factor": 4.0}
    llama = ops.rotary_table(2, 128, base=1e4, scaling=scaling).double()
    got = torch.atan2(llama[1, 64:], llama[1, :64])
    assert torch.allclose(got[turns > 4], angle[turns > 4], rtol=1e-6)
    assert torch.allclose(got[turns < 1], angle[turns < 1] / 8, rtol=1e-4)
    mid = (turns <= 4) & (turns >= 1)
    blend = (turns[mid] - 1) / 3
    assert torch.allclose(got[mid], angle[mid] * ((1 - blend) / 8 + blend), rtol=1e-5)


@pytest.mark.parametrize("arguments", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(positions=-1), dict(scaling={"type": "other"}),
    dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "linear", "factor": 2.0, "beta_fast": 1}), dict(scaling={"type": "yarn", "factor": 2.0}),
    dict(scaling={"type": "llama3", "factor": 2.0, "original_max_position_embeddings": 8, "low_freq_factor": 4.0}),
])
def test_rotary_table_refuses(arguments):
    with pytest.raises(ValueError):
        ops.rotary_table(**(dict(positions=4, rotary_dim=8) | arguments))


def test_reference_rounds_to_e4m3_as_torch_does():
    x = torch.cat([torch.randn(4000, dtype=torch.float64) * 10.0 ** torch.randint(-4, 3, (4000,)),
                   torch.arange(-448, 449, dtype=torch.float64) / 7, torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10])])
    x = x.clamp(-448, 448).float()
    assert torch.equal(ref.e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    assert ref.e4m3(torch.tensor([math.inf, math.nan], dtype=torch.float64)).isnan().all()
    assert [ref.power_of_two(a) for a in (448.0, 449.0, 0.0, 1.75, 1.76)] == [1.0, 2.0, 2.0 ** -100, 2.0 ** -8, 2.0 ** -7]


def test_reference_store_and_attention_on_a_small_case():
    cache, scale = torch.zeros(2, 4, 1, 8).to(torch.float8_e4m3fn), torch.zeros(2, 2, 1)
    rows = torch.full((3, 1, 8), 448.0)
    rows[1] *= 2
    rows[2] = 1.0
    payload, scales = ref.store(rows, cache, scale, int32([2, 3, 4]))
    assert scales.flatten().tolist() == [0.0, 2.0, 2.0 ** -8, 0.0]
    assert payload[0, 2, 0, 0] == 224 and payload[0, 3, 0, 0] == 448 and payload[1, 0, 0, 0] == 256
    q = torch.zeros(1, 1, 8)
    out, lse, _, _ = ref.attention(q, cache, payload.to(torch.float8_e4m3fn), scale, scales.float(), int32([[0, 1]]), [5])
    assert torch.allclose(out, torch.full_like(out, (448 + 896 + 1) / 5)) and math.isclose(lse.item(), math.log(5))


def test_attention_reads_no_device_for_refusals_in_python():
    with pytest.raises(_lib.KvoffError) as error:
        _lib.call("kvoff_attention_fp8_workspace", 1, 1, 4, 16, 4, 2, 96, ctypes.byref(ctypes.c_int64()))
    assert error.value.status == _lib.KVOFF_EINVAL
