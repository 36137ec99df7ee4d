"""The operators of a layer over an e4m3 paged cache in 64 bits, for the tests.

Written from the formulas, one token or block at a time; runs on any device.
"""

from __future__ import annotations

import math

import torch

FP8_MAX = 448.0
MIN_EXPONENT = -100


def half_step(dtype: torch.dtype) -> float:
    """Relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def rotary(x, positions, table, interleaved=False, inverse=False):
    """(result, |x1| + |x2| of each value's pair) in float64."""
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    half = table.shape[1] // 2
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        cos = table[positions.long(), j].double()[:, None]
        sin = table[positions.long(), half + j].double()[:, None]
        if inverse:
            sin = -sin
        x1, x2 = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = x1 * cos - x2 * sin, x2 * cos + x1 * sin
        size[..., a] = size[..., b] = x1.abs() * cos.abs() + x2.abs() * sin.abs() \
            + x2.abs() * cos.abs() + x1.abs() * sin.abs()
    return y, size


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to even, NaN where not finite) of float64 x, |x| <= 448."""
    _, e = torch.frexp(torch.where(x.isfinite(), x, 0.0))
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    y = torch.round(x / step) * step
    return torch.where(x.isfinite(), y, math.nan)


def power_of_two(amax: float) -> float:
    """The smallest 2^e with amax <= 448 * 2^e, e >= MIN_EXPONENT."""
    e = MIN_EXPONENT
    while amax > FP8_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def store(rows, cache, scale, slots):
    """(payload values, scales) after a store, in float64; the arguments are left as they are."""
    pages, page, heads, dim = cache.shape
    block = page // scale.shape[1]
    payload = cache.float().double().cpu().clone().view(-1, block, heads, dim)
    scales = scale.double().cpu().clone().view(-1, heads)
    rows = rows.double().cpu()
    last = {}
    for i, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * page:
            last[slot] = i  # a later row of the same slot takes its place
    blocks = {}
    for slot, i in last.items():
        blocks.setdefault(slot // block, {})[slot % block] = i
    for at, members in blocks.items():
        offsets = list(members)
        x = rows[list(members.values())]
        for h in range(heads):
            finite = x[:, h][x[:, h].isfinite()]
            new = power_of_two(float(finite.abs().max()) if finite.numel() else 0.0)
            if 0 not in members:
                old = float(scales[at, h])
                old = old if math.isfinite(old) and old > 0 else 0.0
                new = max(new, old)
                if new != old:
                    # The kernel's product is in 32 bits, exact for powers of two.
                    kept = payload[at, :, h].float() * torch.tensor(old).div(new).float()
                    payload[at, :, h] = e4m3(kept.double())
            scales[at, h] = new
            payload[at, offsets, h] = e4m3(x[:, h] / new)
    return payload.view(cache.shape), scales.view(scale.shape)


def attention(q, k_cache, v_cache, k_scale, v_scale, tables, contexts, starts=None, softmax_scale=None):
    """Float64 (out, lse, weight, size): weight = sum p |v| / sum p (the scale of an error of the
    probabilities), size = the largest sum |q k| of a row's visible scores (of an error of a score)."""
    n, q_heads, dim = q.shape
    pages, page, kv_heads, _ = k_cache.shape
    block, group = page // k_scale.shape[1], q_heads // kv_heads
    c = dim ** -0.5 if softmax_scale is None else softmax_scale
    dev = q.device
    out = torch.zeros(n, q_heads, dim, dtype=torch.float64, device=dev)
    weight, size = torch.zeros_like(out), torch.zeros(n, q_heads, 1, dtype=torch.float64, device=dev)
    lse = torch.full((n, q_heads), -math.inf, dtype=torch.float64, device=dev)
    if starts is None:
        starts = list(range(len(contexts) + 1))
    for s, context in enumerate(contexts):
        a, b = starts[s], starts[s + 1]
        keys = torch.arange(min(context, tables.shape[1] * page), device=dev)
        at = tables[s].long()[keys // page] if len(keys) else keys
        present = (at >= 0) & (at < pages)
        at = torch.where(present, at, 0)
        for h in range(kv_heads):
            k = k_cache[at, keys % page, h].float().double() * k_scale[at, keys % page // block, h].double()[:, None]
            v = v_cache[at, keys % page, h].float().double() * v_scale[at, keys % page // block, h].double()[:, None]
            for token in range(a, b):
                seen = present & (keys < context - (b - a) + (token - a) + 1)
                if not bool(seen.any()):
                    continue
                x = q[token, h * group:(h + 1) * group].double() @ k[seen].T * c
                heads = slice(h * group, (h + 1) * group)
                lse[token, heads] = torch.logsumexp(x, dim=-1)
                p = torch.softmax(x, dim=-1)
                out[token, heads] = p @ v[seen]
                weight[token, heads] = p @ v[seen].abs()
                size[token, heads, 0] = (q[token, heads].double().abs() @ k[seen].abs().T * c).amax(-1)
    return out, lse, weight, size


def attention_bound(want, weight, size, dtype, keys, v_most, dim):
    """How far a kernel's out may be from `want`, elementwise.

    A probability is off by its rounding to fp16 (half a step, 2^-11), by the error of its score (a
    sum of `dim` exact products in fp32, each addition off by at most 2^-23 of the sum of magnitudes
    since tensor cores truncate, on both sides of the quotient) and by the exponential's 2^-21; the
    running sums are of `keys` terms in fp32. A weight under fp16's smallest normal number is off by
    at most 2^-25 of a scale that is at least 2^-8 of the largest V, and the sum of p is at least 1.
    The result is rounded once.
    """
    share = half_step(torch.float16) + 2 * (dim + 2) * 2.0 ** -23 * size + 2.0 ** -20 \
        + 2 * (keys + 512) * 2.0 ** -24
    return want.abs() * half_step(dtype) * (1 + 2.0 ** -6) + weight * share + keys * 2.0 ** -33 * v_most \
        + torch.finfo(dtype).smallest_normal * half_step(dtype)
