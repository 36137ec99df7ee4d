"""GPU tests of the prompt kernel's bounded waits: one that runs out ends the call with a flag, and nothing else."""

from __future__ import annotations

import pytest
import torch

import kvoff
from kvoff import _lib, ops

pytestmark = pytest.mark.gpu

WAIT_RAN_OUT = 2  # kvoff_device_error's bit of kvoff_attention_fp8


@pytest.mark.parametrize("byte", [0x00, 0x7F, 0xFF])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", [
    ([(300, 2500)], 4, 2, 128, 256, 64), ([(40, 1200), (500, 3000), (90, 90)], 8, 2, 64, 48, 16),
    ([(33, 4000)], 8, 2, 128, 16, 16), ([(200, 400), (0, 0), (90, 700)], 4, 1, 128, 128, 32),
])
def test_a_wait_that_runs_out_ends_the_call(cuda, byte, lengths, q_heads, kv_heads, dim, page, block):
    """The workspace holds anything before the call: the join must not take it for the kernel's records."""
    g = torch.Generator(device="cuda")
    g.manual_seed(byte)
    need = [-(-c // page) for _, c in lengths]
    tables = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device=cuda)
    for i, n in enumerate(need):
        tables[i, :n] = torch.arange(n, device=cuda) + sum(need[:i])
    shape = (sum(need), page, kv_heads, dim)
    cache = [torch.randn(shape, generator=g, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(shape[0], page // block, kv_heads, device=cuda) for _ in range(2)]
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    longest = max(n for n, _ in lengths)
    q = torch.randn(starts[-1], q_heads, dim, generator=g, device="cuda").bfloat16()
    options = dict(cu_seqlens_q=torch.tensor(starts, dtype=torch.int32, device=cuda), max_seqlen_q=longest)
    args = (q, *cache, *scales, tables, torch.tensor([c for _, c in lengths], dtype=torch.int32, device=cuda))
    want = ops.attention_fp8(*args, **options)
    assert kvoff.device_error(0) == 0

    size = ops.attention_fp8_workspace(len(lengths), longest, tables.shape[1], page, q_heads, kv_heads, dim)
    space = torch.full((size + 4096,), byte, dtype=torch.uint8, device=cuda)
    rows = torch.full((starts[-1] + 16, q_heads, dim), 3.0, dtype=torch.bfloat16, device=cuda)
    kept = [x.view(torch.uint8).clone() for x in (*cache, q)]
    _lib.debug_fail_next("attention_wait")
    ops.attention_fp8(*args, **options, out=rows[:starts[-1]], workspace=space[:size] if size else None)
    torch.cuda.synchronize()
    assert kvoff.device_error(0) == WAIT_RAN_OUT
    assert (space[size:] == byte).all() and (rows[starts[-1]:] == 3.0).all()
    for x, y in zip((*cache, q), kept):
        assert torch.equal(x.view(torch.uint8), y)

    again = ops.attention_fp8(*args, **options, workspace=space[:size] if size else None)
    assert kvoff.device_error(0) == 0
    assert torch.equal(again, want)
