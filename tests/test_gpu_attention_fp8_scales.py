"""GPU tests of attention over the e4m3 cache where the scales of V lie far apart: a key that a row does not
see, or sees with next to no weight, takes no precision from the keys that make up the row's result."""

from __future__ import annotations

import math

import pytest
import torch

import kvoff
import layer_reference as ref
from kvoff import ops

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_wait_ran_out(cuda):
    yield
    assert kvoff.device_error(0) == 0


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def largest_terms(q, cache, scales, tables, contexts, starts, c):
    """The largest p_t * scale_t and p_t of each row's visible keys, p the softmax, two [N, Hq] in float64."""
    (kc, vc), (ks, vs) = cache, scales
    page, heads = kc.shape[1], kc.shape[2]
    block, group = page // ks.shape[1], q.shape[1] // heads
    most, weight = (torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device) for _ in range(2))
    for s, context in enumerate(contexts):
        keys = torch.arange(context, device=q.device)
        at = tables[s].long()[keys // page]
        for h in range(heads):
            k = kc[at, keys % page, h].float().double() * ks[at, keys % page // block, h].double()[:, None]
            v = vs[at, keys % page // block, h].double()
            v = torch.where((vc[at, keys % page, h].float() != 0).any(-1), v, 0)  # keys of zeros add nothing
            for token in range(starts[s], starts[s + 1]):
                seen = context - (starts[s + 1] - starts[s]) + token - starts[s] + 1
                if seen > 0:
                    rows = slice(h * group, (h + 1) * group)
                    p = torch.softmax(q[token, rows].double() @ k[:seen].T * c, dim=-1)
                    most[token, rows] = (p * v[:seen]).amax(-1)
                    weight[token, rows] = p.amax(-1)
    return most, weight


class Batch:
    """Sequences of (new, context) tokens in a cache that the store filled."""

    def __init__(self, seed, lengths, q_heads, kv_heads, dim, page, block, dtype):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.lengths, self.starts = lengths, [0]
        for n, _ in lengths:
            self.starts.append(self.starts[-1] + n)
        need = [-(-c // page) for _, c in lengths]
        self.tables = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
        order, at = torch.randperm(sum(need), generator=self.g, device="cuda").int(), 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.shape, self.block, self.dtype = (sum(need), page, kv_heads, dim), block, dtype
        self.q = self.randn(self.starts[-1], q_heads, dim).to(dtype)
        self.rows = [(self.randn(c, kv_heads, dim).to(BF16), self.randn(c, kv_heads, dim).to(BF16)) for _, c in lengths]

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def check(self, softmax_scale=None, exact_scores=False, v_factor=1.0):
        pages, page, heads, dim = self.shape
        c = dim ** -0.5 if softmax_scale is None else softmax_scale
        cache = [torch.zeros(self.shape, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
        scales = [torch.zeros(pages, page // self.block, heads, device="cuda") for _ in range(2)]
        for s, (k, v) in enumerate(self.rows):
            t = torch.arange(len(k), device="cuda")
            slots = (self.tables[s].long()[t // page] * page + t % page).int()
            ops.store_kvcache_fp8(k, v, *cache, *scales, slots)
        scales[1] *= v_factor  # scales need not be powers of two
        contexts = [n for _, n in self.lengths]
        args = (*cache, *scales, self.tables)
        lse = torch.empty(self.q.shape[:2], device="cuda")
        got = ops.attention_fp8(self.q, *args, int32(contexts), cu_seqlens_q=int32(self.starts), lse=lse,
                                max_seqlen_q=max(n for n, _ in self.lengths), softmax_scale=softmax_scale)
        want, want_lse, weight, size_of = ref.attention(self.q, *args, contexts, self.starts, c)
        size = size_of
        keys, score = max(contexts), size_of
        most, heaviest = largest_terms(self.q, cache, scales, self.tables, contexts, self.starts, c)
        if exact_scores:
            # Sums of one product have no error. The exponent's error stays, but where one key has all the
            # weight: what a weight is off by stands in the sum of weights too, and the quotient is 1.
            size = torch.zeros_like(size)
            score = torch.where(heaviest[..., None] == 1, 0.0, score)
        # As in attention_bound, with two differences. A weight under f16's smallest normal number is off by at
        # most 2^-25 of a unit that is 2^-8 of the row's own largest p * scale, whatever the other scales are.
        # And the exponent of a weight is a sum of scores and of logarithms of scales: six fp32 roundings of at
        # most 2^-24 of numbers up to 256 + 3 * size (log2 units).
        share = ref.half_step(FP16) + 2 * (dim + 2) * 2.0 ** -23 * size + 2.0 ** -20 + 2 * (keys + 512) * 2.0 ** -24 \
            + 6 * math.log(2) * 2.0 ** -24 * (256 + 3 * score)
        bound = want.abs() * ref.half_step(self.dtype) * (1 + 2.0 ** -6) + weight * share \
            + keys * 2.0 ** -33 * 448 * most[..., None] + torch.finfo(self.dtype).smallest_normal * ref.half_step(self.dtype)
        off = (got.double() - want).abs()
        assert not got.isnan().any()
        assert not (off > bound).any(), f"off by {(off / bound).max():.2f} of the bound"
        error = (dim + 2) * 2.0 ** -23 * size_of[..., 0] + 2.0 ** -20 + (keys + 512) * 2.0 ** -24 + 2.0 ** -20 * want_lse.abs()
        fine = want_lse.isfinite()
        assert torch.equal(fine, lse.isfinite()) and ((lse.double() - want_lse).abs()[fine] <= error[fine]).all()


# Up to 32 rows a KV head go to the decode kernel; contexts above 1024 keys are split over CTAs.
FEW = [([(20, 40)], 1, 1, 128, 16, 16), ([(20, 40)], 2, 2, 64, 48, 16), ([(8, 1500)], 4, 1, 128, 16, 16),
       ([(16, 300), (3, 2100), (16, 16)], 2, 1, 64, 32, 16)]
MANY = [([(200, 300)], 1, 1, 128, 16, 16), ([(300, 1500)], 1, 1, 128, 1024, 1024), ([(130, 1900)], 4, 1, 128, 48, 16),
        ([(300, 400), (90, 1500)], 2, 2, 64, 32, 16)]


def later_keys(batch, value, inside):
    """V of keys that the first new tokens do not see becomes `value`: the last 16 key places of the context, or
    (inside) one key that stands among keys that they do see, whose payload then is zero."""
    for (n, c), (_, v) in zip(batch.lengths, batch.rows):
        if inside:
            v[c - n + n // 2 + 1 if n > 2 else c - 1] = value
        else:
            v[max(c - n + 1, (c - 1) // 16 * 16):] = value


@pytest.mark.parametrize("value,inside", [(1e4, False), (1e9, False), (1e20, False), (1e34, False), (1e9, True),
                                          (1e20, True)])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", FEW)
def test_decode_kernel_later_keys_of_large_values(cuda, value, inside, lengths, q_heads, kv_heads, dim, page, block):
    batch = Batch(1, lengths, q_heads, kv_heads, dim, page, block, BF16)
    later_keys(batch, value, inside)
    batch.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("first,low", [(False, None), (True, None), (False, 4), (False, 1), (True, 4)])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", FEW + [([(1, 130), (1, 3000)], 8, 1, 128, 64, 32)])
def test_decode_kernel_large_values_of_little_weight(cuda, dtype, first, low, lengths, q_heads, kv_heads, dim, page, block):
    check_little_weight(2, dtype, first, low, lengths, q_heads, kv_heads, dim, page, block)


def check_little_weight(seed, dtype, first, low, lengths, q_heads, kv_heads, dim, page, block):
    """The first `low` keys (None: a scale block) have large V and scores so low that they count for less than the
    rest does; with `first` their scores are not as low and they decide the result. The other keys of their block,
    whose payload is zero, have weight."""
    low = low or block
    batch = Batch(seed, lengths, q_heads, kv_heads, dim, page, block, dtype)
    batch.q[..., 0] = 4.0
    for (n, c), (k, v) in zip(batch.lengths, batch.rows):
        k[..., 0] = 0.0
        k[:low, :, 0] = -8.0 if first else -64.0  # 4 * 64 / sqrt(dim) is 22 or 32 below the others' scores
        v[:low] *= 2.0 ** ((60 if first else 30 if dim == 128 else 44) if dtype == BF16 else 12)
        if c > 600:  # another CTA's part
            k[416:416 + low, :, 0] = -48.0
            v[416:416 + low] *= 2.0 ** 20 if dtype == BF16 else 1.0
    batch.check()


def test_decode_kernel_blocks_of_zeros_beside_large_values(cuda):
    """A block of V that is all zero has the smallest scale, and its keys still count in the sum of weights."""
    batch = Batch(3, [(4, 70), (1, 1600)], 4, 1, 128, 16, 16, BF16)
    check_zero_blocks(batch)


def check_zero_blocks(batch):
    for (n, c), (_, v) in zip(batch.lengths, batch.rows):
        v[:16] = 0
        v[32:48] = 0
        v[16:32] *= 2.0 ** 40
        v[c // 2 // 16 * 16:] *= 2.0 ** -30
    batch.check()
    for _, v in batch.rows:
        v.zero_()
    batch.check()


@pytest.mark.parametrize("value,inside", [(1e4, False), (1e9, False), (1e20, False), (1e34, False), (1e9, True),
                                          (1e20, True)])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", MANY)
def test_prompt_kernel_later_keys_of_large_values(cuda, value, inside, lengths, q_heads, kv_heads, dim, page, block):
    batch = Batch(4, lengths, q_heads, kv_heads, dim, page, block, BF16)
    later_keys(batch, value, inside)
    batch.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("first,low", [(False, None), (True, None), (False, 4), (False, 1), (True, 4)])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", MANY)
def test_prompt_kernel_large_values_of_little_weight(cuda, dtype, first, low, lengths, q_heads, kv_heads, dim, page, block):
    check_little_weight(5, dtype, first, low, lengths, q_heads, kv_heads, dim, page, block)


def test_prompt_kernel_blocks_of_zeros_beside_large_values(cuda):
    check_zero_blocks(Batch(6, [(140, 170), (100, 1600)], 4, 1, 128, 16, 16, BF16))


@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", FEW + MANY)
def test_a_large_value_far_below_the_largest_weight(cuda, lengths, q_heads, kv_heads, dim, page, block):
    """V is zero but for one key of 2^60 times 2^-115 of the weight: the units of weights and of terms are 2^120 apart."""
    batch = Batch(7, lengths, q_heads, kv_heads, dim, page, block, BF16)
    batch.q[..., 0] = 4.0
    for (n, c), (k, v) in zip(batch.lengths, batch.rows):
        k[..., 0] = 0.0
        k[c // 2, :, 0] = -20.0 * dim ** 0.5  # 80 below the others' scores
        large = v[c // 2] * 2.0 ** 60
        v.zero_()
        v[c // 2] = large
    batch.check()


@pytest.mark.parametrize("q_log2,k_log2", [(3, 3), (8, 8), (12, 13), (14, 14)])
@pytest.mark.parametrize("v_log2", [-40, 0, 30])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", FEW + MANY)
def test_large_scores(cuda, q_log2, k_log2, v_log2, lengths, q_heads, kv_heads, dim, page, block):
    """Scores up to 2^25 (log2 units) that are exact: one key takes all the weight of the rows that see it, and the
    others give all keys the same. Neither m nor the scale of V may lose the other's bits."""
    batch = Batch(8, lengths, q_heads, kv_heads, dim, page, block, BF16)
    batch.q.zero_()
    batch.q[..., 1] = 2.0 ** q_log2
    for (n, c), (k, v) in zip(batch.lengths, batch.rows):
        k.zero_()
        k[..., 1] = -2.0 ** k_log2
        k[c - n // 2 - 1, :, 1] = 2.0 ** k_log2
        v *= 2.0 ** v_log2
    batch.check(exact_scores=True, v_factor=1.37)
