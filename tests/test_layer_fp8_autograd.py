"""Calls of the layer over the e4m3 cache that autograd would not see are refused in grad mode. No GPU work."""

from __future__ import annotations

import pytest
import torch

from kvoff import ops

ROWS = (3, 4, 64)


def rows(grad=False):
    return torch.zeros(ROWS, dtype=torch.bfloat16, requires_grad=grad)


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def cache(grad=False):
    payload = torch.zeros(2, 32, 4, 64).to(torch.float8_e4m3fn)
    return [payload, payload, torch.zeros(2, 2, 4, requires_grad=grad), torch.zeros(2, 2, 4, requires_grad=grad)]


def rotary(q=None, k=None, table=None, out=None):
    table = ops.rotary_table(8, 64) if table is None else table
    ops.rotary(rows() if q is None else q, rows() if k is None else k, torch.arange(3), table, out=out)


def store(key=None, value=None, scales=False):
    ops.store_kvcache_fp8(rows() if key is None else key, rows() if value is None else value, *cache(scales),
                          int32([0, 1, 2]))


def attention(q=None, scales=False, out=None):
    ops.attention_fp8(rows() if q is None else q, *cache(scales), int32([[0, 1]] * 3), int32([1, 2, 3]), out=out)


CALLS = [
    lambda: rotary(q=rows(True)), lambda: rotary(k=rows(True)), lambda: rotary(q=rows(True), out=(rows(), rows())),
    lambda: rotary(q=rows(True) * 2, k=rows(True) * 2),  # not leaves
    lambda: rotary(out=(rows(True), rows())), lambda: rotary(table=ops.rotary_table(8, 64).requires_grad_()),
    lambda: store(key=rows(True)), lambda: store(value=rows(True) * 2), lambda: store(scales=True),
    lambda: attention(q=rows(True)), lambda: attention(scales=True), lambda: attention(out=rows(True)),
]


@pytest.mark.parametrize("call", CALLS)
def test_inputs_that_require_a_gradient_are_refused(call):
    with pytest.raises(ValueError, match="autograd"):
        call()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("call", CALLS)
def test_they_are_taken_where_no_graph_is_made(call, mode):
    with mode(), pytest.raises(ValueError, match="CUDA"):  # the next thing that is wrong with them
        call()


class Turn(torch.autograd.Function):
    """rotary in a graph: its gradient is the inverse turn of the gradients."""

    @staticmethod
    def forward(ctx, q, k, positions, table):
        ctx.save_for_backward(positions, table)
        return ops.rotary(q, k, positions, table, out=(torch.empty_like(q), torch.empty_like(k)))

    @staticmethod
    def backward(ctx, dq, dk):
        positions, table = ctx.saved_tensors
        dq, dk = ops.rotary(dq, dk, positions, table, inverse=True,
                            out=(torch.empty_like(dq), torch.empty_like(dk)))
        return dq, dk, None, None


@pytest.mark.gpu
def test_a_function_gives_rotary_its_gradient(cuda):
    """Against the formula's gradient in 64 bits: <w, y> with y1 = x1 c - x2 s, y2 = x2 c + x1 s."""
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    table, positions = ops.rotary_table(50, 32, device=cuda), torch.arange(5, device=cuda) * 9
    q, k, wq, wk = (torch.randn(5, h, 64, generator=g, device="cuda") for h in (4, 2, 4, 2))
    q.requires_grad_()
    k.requires_grad_()
    y, z = Turn.apply(q, k, positions, table)
    ((y * wq).sum() + (z * wk).sum()).backward()
    for x, w in ((q, wq), (k, wk)):
        want = w.double().clone()
        cos, sin = (table[positions][:, None, i * 16:(i + 1) * 16].double() for i in (0, 1))
        a, b = w[..., :16].double(), w[..., 16:32].double()
        want[..., :16], want[..., 16:32] = a * cos + b * sin, b * cos - a * sin
        # Two products and a sum in fp32.
        bound = 3 * 2.0 ** -24 * (w[..., :32].double().abs().amax() * 2) + 2.0 ** -24 * want.abs()
        assert ((x.grad.double() - want).abs() <= bound).all()
