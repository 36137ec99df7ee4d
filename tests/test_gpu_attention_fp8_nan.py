"""GPU tests of the log-sum-exp of rows whose scores are NaN: NaN, not that of a row without keys."""

from __future__ import annotations

import math

import pytest
import torch

import kvoff
from kvoff import ops

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# The decode kernel whole and split (contexts above 1024 keys), and the prompt kernel whole and split.
@pytest.mark.parametrize("n,context,dim", [(1, 90, 128), (1, 9, 64), (4, 3000, 128), (1, 5000, 64), (70, 300, 128),
                                           (200, 2000, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lse_of_nan_scores_is_nan(cuda, n, context, dim, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(n + context)
    page, heads, q_heads = 16, 2, 4
    pages = 2 * -(-context // page)
    cache = [torch.randn(pages, page, heads, dim, generator=g, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(pages, 1, heads, device="cuda") for _ in range(2)]
    tables = torch.randperm(pages, generator=g, device="cuda").int().view(2, -1)
    contexts, starts = [context, n // 2], [0, n, 2 * n]  # in the second sequence some rows see no key
    q = torch.randn(2 * n, q_heads, dim, generator=g, device="cuda").to(dtype)
    q[n - 1, 1, 5] = math.nan  # every score of the row
    q[0, 2, :] = math.nan
    # A key of NaN that the first sequence's last token alone sees, in the other KV head.
    t = context - 1
    cache[0].view(torch.uint8)[tables[0, t // page].long(), t % page, 1] = 0x7F
    lse = torch.empty(2 * n, q_heads, device="cuda")
    out = ops.attention_fp8(q, *cache, *scales, tables, int32(contexts), cu_seqlens_q=int32(starts), max_seqlen_q=n,
                            lse=lse)
    assert kvoff.device_error(0) == 0
    nan = torch.zeros(2 * n, q_heads, dtype=torch.bool, device="cuda")
    nan[n - 1, 1] = nan[0, 2] = True
    nan[n - 1, 2:] = True
    assert torch.equal(out.isnan().all(-1), nan) and torch.equal(out.isnan().any(-1), nan)
    assert torch.equal(lse.isnan(), nan)
    empty = torch.zeros_like(nan)
    empty[n:2 * n - n // 2] = True
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
