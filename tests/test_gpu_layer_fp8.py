"""GPU tests of rotary positions, the e4m3 slot store and attention over the e4m3 paged cache,
against the same formulas in 64 bits (tests/layer_reference.py)."""

from __future__ import annotations

import math

import pytest
import torch

import kvoff
import layer_reference as ref
from kvoff import attention as layer
from kvoff import ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NAN_BYTE = 0x7F


@pytest.fixture(autouse=True)
def _no_wait_ran_out(cuda):
    """Each bounded wait inside a kernel ended because what it waited for came."""
    yield
    assert kvoff.device_error(0) == 0


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ---------------------------------------------------------------------------------------------------
# rotary


def check_rotary(x, got, positions, table, interleaved, inverse):
    want, size = ref.rotary(x, positions, table, interleaved, inverse)
    # Two products and a sum in fp32 of inputs that are exact, then one rounding to x's type.
    bound = want.abs() * ref.half_step(x.dtype) + size * 3 * 2.0 ** -24 \
        + torch.finfo(x.dtype).smallest_normal * ref.half_step(x.dtype)
    assert ((got.double() - want).abs() <= bound * (1 + 2.0 ** -6)).all()
    assert torch.equal(got[..., table.shape[1]:], x[..., table.shape[1]:])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary_dim", [
    (1, 32, 8, 128, 128), (4, 7, 1, 64, 64), (129, 5, 5, 128, 64), (33, 3, 2, 80, 40), (17, 2, 1, 24, 6),
    (5, 1, 1, 2, 2), (301, 16, 4, 256, 128),
])
def test_rotary_matches_the_formula(cuda, dtype, interleaved, tokens, q_heads, kv_heads, dim, rotary_dim):
    g = generator(1)
    width = [h * dim for h in (q_heads, kv_heads, 3)]
    q, k, _ = randn(g, tokens, sum(width)).to(dtype).split(width, dim=1)  # strided views, as a model has
    q, k = q.view(tokens, q_heads, dim), k.view(tokens, kv_heads, dim)
    if interleaved and (q.stride(0) * q.element_size()) % (2 * q.element_size()):
        pytest.skip("pairs must be aligned")
    table = ops.rotary_table(70000, rotary_dim, base=1e6, device=cuda,
                             scaling={"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 16384})
    positions = torch.randint(0, 70000, (tokens,), generator=g, device="cuda")
    out = (torch.empty_like(q), torch.full((tokens, kv_heads, dim), 9.0, dtype=dtype, device=cuda))
    before = q.clone(), k.clone()
    for inverse in (False, True):
        got = layer.rotary(q, k, positions, table, interleaved=interleaved, inverse=inverse, out=out)
        assert got[0] is out[0] and got[1] is out[1]
        for x, y in zip((q, k), got):
            check_rotary(x, y, positions, table, interleaved, inverse)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    ops.rotary(q, k, positions.int(), table, interleaved=interleaved)  # in place, int32 positions
    check_rotary(before[0], q, positions, table, interleaved, False)
    check_rotary(before[1], k, positions, table, interleaved, False)


def test_rotary_takes_unaligned_rows(cuda):
    g = generator(2)
    flat = randn(g, 9 * (6 * 64 + 3) + 8).to(BF16)
    q = flat[1:].as_strided((9, 4, 64), (6 * 64 + 3, 64, 1))
    k = flat[1 + 4 * 64:].as_strided((9, 2, 64), (6 * 64 + 3, 64, 1))
    table = ops.rotary_table(100, 64, device=cuda)
    positions = torch.arange(9, device=cuda) * 11
    out = torch.empty(9, 4, 64, dtype=BF16, device=cuda), torch.empty(9, 2, 64, dtype=BF16, device=cuda)
    ops.rotary(q, k, positions, table, out=out)
    check_rotary(q, out[0], positions, table, False, False)
    check_rotary(k, out[1], positions, table, False, False)


def test_rotary_skips_positions_outside_the_table(cuda):
    g = generator(3)
    q, k = randn(g, 6, 4, 128).to(BF16), randn(g, 6, 2, 128).to(BF16)
    table = ops.rotary_table(50, 128, device=cuda)
    positions = torch.tensor([3, -1, 49, 50, 2 ** 40, -2 ** 40], device=cuda)
    bad = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.rotary(q, k, positions, table, out=out, bad_positions=bad)
    assert bad.item() == 2
    for x, y in zip((q, k), out):
        assert (y[[1, 3, 4, 5]] == 7.0).all()
        check_rotary(x[[0, 2]], y[[0, 2]], positions[[0, 2]], table, False, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_inverse_is_the_gradient(cuda, interleaved):
    """<dy, rotary(x)> has the gradient inverse(dy): against autograd of the formula, and against differences."""
    g = generator(4)
    table = ops.rotary_table(64, 48, device=cuda, scaling={"type": "yarn", "factor": 8.0,
                                                           "original_max_position_embeddings": 16})
    positions = torch.arange(13, device=cuda)
    x, dy = randn(g, 13, 3, 64), randn(g, 13, 3, 64)
    one = dy[:, :1].clone()
    grad, _ = ops.rotary(dy.clone(), one, positions, table, interleaved=interleaved, inverse=True)
    x64 = x.double().requires_grad_()
    half, pairs = 24, (slice(0, 48, 2), slice(1, 48, 2)) if interleaved else (slice(0, 24), slice(24, 48))
    cos, sin = (table[positions][:, None, i * half:(i + 1) * half].double() for i in (0, 1))
    a, b = x64[..., pairs[0]], x64[..., pairs[1]]
    y = x64 * 0
    y = torch.cat([x64[..., 48:] * dy[..., 48:].double(),
                   (a * cos - b * sin) * dy[..., pairs[0]].double(),
                   (b * cos + a * sin) * dy[..., pairs[1]].double()], dim=-1).sum()
    y.backward()
    assert torch.allclose(grad.double(), x64.grad, rtol=0, atol=8 * 2.0 ** -22)
    # The map is linear, so a difference of any length is the derivative up to rounding.
    moved, _ = ops.rotary(x + grad, one.clone(), positions, table, interleaved=interleaved)
    still, _ = ops.rotary(x.clone(), one.clone(), positions, table, interleaved=interleaved)
    difference = ((moved.double() - still.double()) * dy.double()).sum()
    assert abs(difference - grad.double().square().sum()) <= grad.numel() * 2.0 ** -18


# ---------------------------------------------------------------------------------------------------
# store


def empty_cache(g, pages, page, heads, dim, block, filled=True):
    """A cache whose rows hold something (filled) or any bytes, NaN among them, with zero scales."""
    cache = torch.randint(0, 256, (pages, page, heads, dim), generator=g, device="cuda", dtype=torch.uint8)
    if filled:
        cache = torch.where(cache & 0x7F == NAN_BYTE, 0x30, cache).to(torch.uint8)
        scale = torch.exp2(torch.randint(-9, 3, (pages, page // block, heads), generator=g, device="cuda").float())
    else:
        scale = torch.zeros(pages, page // block, heads, device="cuda")
    return cache.view(torch.float8_e4m3fn), scale


def same_values(got, want):
    got = got.float().double().cpu()
    return torch.equal(got.nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))


def check_store(key, value, caches, slots, **options):
    (kc, ks), (vc, vs) = caches
    wants = [ref.store(x, c, s, slots) for x, (c, s) in zip((key, value), caches)]
    ops.store_kvcache_fp8(key, value, kc, vc, ks, vs, slots, **options)
    for (payload, scale), (c, s) in zip(wants, caches):
        assert torch.equal(s.double().cpu(), scale)
        assert same_values(c, payload)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,heads,dim,page,block", [
    (1, 8, 128, 256, 64), (40, 8, 128, 256, 256), (300, 2, 64, 48, 16), (77, 5, 80, 16, 1), (1500, 3, 128, 64, 32),
    (130, 1, 256, 128, 128), (9, 1, 8, 4, 2), (1100, 4, 24, 2048, 1024),
])
def test_store_matches_the_formula(cuda, dtype, tokens, heads, dim, page, block):
    g = generator(5)
    pages = -(-tokens // page) + 2
    rows = randn(g, tokens, 2 * heads * dim + 8) * torch.exp(2 * randn(g, tokens, 1))
    rows = rows.to(dtype)
    key, value = (rows[:, i * heads * dim:(i + 1) * heads * dim].view(tokens, heads, dim) for i in (0, 1))
    start = page // 2 + 1
    slots = (start + torch.arange(tokens, device=cuda)).to(torch.int32)
    slots[tokens // 3] = -1
    caches = [empty_cache(g, pages, page, heads, dim, block) for _ in range(2)]
    check_store(key, value, caches, slots)


def test_store_opens_extends_and_grows_blocks(cuda):
    """A page filled a few tokens at a time, with scales that grow in between."""
    g = generator(6)
    caches = [empty_cache(g, 3, 32, 2, 64, 16, filled=False) for _ in range(2)]
    at = 0
    for n, size in ((3, 1.0), (1, 1e-3), (1, 40.0), (7, 3.0), (1, 5e4), (9, 0.1), (5, 0.0), (5, 1e-7)):
        key, value = (size * randn(g, n, 2, 64)).to(BF16), (randn(g, n, 2, 64) / 3).to(BF16)
        check_store(key, value, caches, (32 + torch.arange(at, at + n, device=cuda)).to(torch.int32))
        at += n
    key = torch.ones(1, 2, 64, dtype=BF16, device=cuda)  # opens the block again: the large scale is gone
    check_store(key, key, caches, torch.tensor([32], dtype=torch.int32, device=cuda))
    assert caches[0][1][1, 0, 0] == 2.0 ** -8


def test_store_takes_slots_in_any_order_twice_and_skipped(cuda):
    g = generator(7)
    for tokens in (200, 1300):  # one token a CTA, and a window of them
        caches = [empty_cache(g, 12, 32, 2, 128, 32) for _ in range(2)]
        slots = torch.randint(0, 12 * 32, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        slots[::7] = -1
        slots[3] = 12 * 32
        slots[5] = 2 ** 31 - 1
        key, value = randn(g, tokens, 2, 128).to(FP16), randn(g, tokens, 2, 128).to(FP16)
        bad = torch.zeros(1, dtype=torch.int32, device=cuda)
        check_store(key, value, caches, slots, bad_slots=bad)
        assert bad.item() == 2
        unaligned = torch.empty(tokens + 1, dtype=torch.int32, device=cuda)[1:].copy_(slots)
        check_store(key, value, caches, unaligned)


def test_store_holds_what_is_not_finite_as_nan(cuda):
    g = generator(8)
    key = randn(g, 20, 2, 64).to(BF16)
    key[3, 0, 5], key[4, 0, 6], key[19, 1, 0] = math.inf, -math.inf, math.nan
    caches = [empty_cache(g, 2, 16, 2, 64, 16) for _ in range(2)]
    slots = torch.arange(4, 24, device=cuda).to(torch.int32)
    check_store(key, key.clone(), caches, slots)
    assert caches[0][0].float().isnan().sum() == 3
    check_store(key[:1] * 1e4, key[:1], caches, torch.tensor([1], dtype=torch.int32, device=cuda))  # NaN stay


def test_store_scale_is_exact_at_its_borders(cuda):
    for amax in (448.0, 450.0, 1.0, 1.75, 1.7578125, 2.0 ** -120, 3.0e38, 2.0 ** -133, 0.0):
        key = torch.zeros(1, 1, 8, device=cuda)
        key[0, 0, 3] = -amax
        caches = [empty_cache(generator(9), 1, 16, 1, 8, 16, filled=False) for _ in range(2)]
        check_store(key.to(BF16), key.to(BF16), caches, torch.zeros(1, dtype=torch.int32, device=cuda))


def test_store_leaves_other_blocks_as_they_were(cuda):
    g = generator(10)
    caches = [empty_cache(g, 4, 64, 2, 128, 16, filled=False) for _ in range(2)]
    before = [c.view(torch.uint8).clone() for c, _ in caches]
    slots = torch.arange(64 + 16, 64 + 48, device=cuda).to(torch.int32)
    key = randn(g, 32, 2, 128).to(BF16)
    ops.store_kvcache_fp8(key, key, caches[0][0], caches[1][0], caches[0][1], caches[1][1], slots)
    for (c, s), b in zip(caches, before):
        flat, old = c.view(torch.uint8).view(-1, 2, 128), b.view(-1, 2, 128)
        assert torch.equal(flat[:80], old[:80]) and torch.equal(flat[112:], old[112:])
        assert (s.view(-1, 2)[:5] == 0).all() and (s.view(-1, 2)[7:] == 0).all()


# ---------------------------------------------------------------------------------------------------
# attention


def build(g, lengths, q_heads, kv_heads, dim, page, block, dtype, spread=1.0, extra_width=1):
    """q, caches, scales, tables, contexts, starts of a batch with (new, context) lengths."""
    need = [-(-c // page) for _, c in lengths]
    pages = sum(need) + 2
    tables = torch.full((len(lengths), max(need + [1]) + extra_width), -7, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").int()
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    out = []
    for _ in range(2):
        x = randn(g, pages, page, kv_heads, dim) * torch.exp(0.7 * randn(g, kv_heads, dim))
        x *= torch.exp(spread * randn(g, pages, page // block, kv_heads)).repeat_interleave(block, 1)[..., None]
        amax = x.view(pages, page // block, block, kv_heads, dim).abs().amax((2, 4))
        scale = torch.exp2(torch.ceil(torch.log2(amax / 448)))
        if block > 16:  # scales need not be powers of two
            scale *= 1.37
        x = x / scale.repeat_interleave(block, 1)[..., None]
        out += [x.clamp(-448, 448).to(torch.float8_e4m3fn), scale]
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    q = randn(g, starts[-1], q_heads, dim).to(dtype)
    return q, out[0], out[2], out[1], out[3], tables, [c for _, c in lengths], starts


def poison(batch, lengths):
    """NaN in every row behind a context, and in the scales of blocks that no context reaches."""
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    page, block = kc.shape[1], kc.shape[1] // ks.shape[1]
    used = torch.zeros(kc.shape[0] * page, dtype=torch.bool, device="cuda")
    for i, c in enumerate(contexts):
        t = torch.arange(c, device="cuda")
        used[tables[i].long()[t // page] * page + t % page] = True
    for c, s in ((kc, ks), (vc, vs)):
        c.view(torch.uint8).view(-1, *c.shape[2:])[~used] = NAN_BYTE
        s.view(-1, s.shape[2])[~used.view(-1, block).any(1)] = math.nan


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def call(batch, lengths, decode=False, **options):
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    if not decode:
        options.update(cu_seqlens_q=int32(starts), max_seqlen_q=max(n for n, _ in lengths))
    return layer.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts), **options)


def check_attention(batch, got, lse=None, softmax_scale=None):
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    want, want_lse, weight, size = ref.attention(q, kc, vc, ks, vs, tables, contexts, starts, softmax_scale)
    dim, keys = q.shape[-1], max(contexts)
    v_most = 448 * float(vs[vs.isfinite()].max())
    bound = ref.attention_bound(want, weight, size, q.dtype, keys, v_most, dim)
    off = (got.double() - want).abs()
    assert torch.equal(got.isnan(), want.isnan())
    assert not (off > bound).any(), f"off by {(off / bound).nan_to_num().max():.2f} of the bound"
    if lse is not None:
        assert torch.equal(lse.isinf(), want_lse.isinf()) and not lse.isnan().any()
        fine = want_lse.isfinite()
        # One score's error, the exponentials' and the fp32 sum's relative error, the logarithm's.
        most = (dim + 2) * 2.0 ** -23 * size[..., 0] + 2.0 ** -20 + (keys + 512) * 2.0 ** -24 \
            + 2.0 ** -20 * want_lse.abs()
        assert ((lse.double() - want_lse).abs()[fine] <= most[fine]).all()


DECODE = [
    # lengths of the contexts, q_heads, kv_heads, dim, page, block
    ([1], 4, 1, 128, 16, 16),
    ([300], 32, 8, 128, 256, 64),
    ([0, 1, 15, 16, 17, 255, 256, 257], 8, 8, 64, 48, 16),
    ([5000, 0, 3, 1029], 16, 2, 128, 64, 32),
    ([2047, 2048, 2049], 10, 2, 128, 256, 256),
    ([9000], 2, 1, 64, 32, 16),
    ([700] * 30, 6, 2, 64, 16, 16),
    ([1500, 40], 24, 2, 128, 16, 16),
    ([130], 40, 1, 128, 128, 128),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("contexts,q_heads,kv_heads,dim,page,block", DECODE)
def test_attention_decodes(cuda, dtype, contexts, q_heads, kv_heads, dim, page, block):
    lengths = [(1, c) for c in contexts]
    batch = build(generator(11), lengths, q_heads, kv_heads, dim, page, block, dtype)
    poison(batch, lengths)
    lse = torch.full(batch[0].shape[:2], 5.0, device=cuda)
    got = call(batch, lengths, decode=True, lse=lse)
    check_attention(batch, got, lse)
    again = call(batch, lengths, lse=lse)  # the same as one token each of a ragged batch
    assert torch.equal(got, again)


EXTEND = [
    # (new tokens, context) of each sequence
    ([(3, 3)], 4, 1, 128, 16, 16),
    ([(1, 900), (5, 1200), (0, 64), (2, 2), (17, 333)], 8, 2, 128, 48, 16),
    ([(130, 130), (1, 77), (64, 1000)], 4, 4, 64, 64, 32),
    ([(40, 2100)], 32, 4, 128, 256, 64),
    ([(257, 300), (33, 4000)], 10, 2, 128, 256, 256),
    ([(700, 700)], 2, 1, 64, 16, 16),
    ([(300, 1024)], 7, 1, 128, 16, 16),
    ([(5, 3), (4, 0), (300, 200)], 4, 2, 128, 16, 16),  # more new tokens than context: the first rows are empty
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim,page,block", EXTEND)
def test_attention_extends(cuda, dtype, lengths, q_heads, kv_heads, dim, page, block):
    batch = build(generator(12), lengths, q_heads, kv_heads, dim, page, block, dtype)
    poison(batch, lengths)
    lse = torch.full(batch[0].shape[:2], 5.0, device=cuda)
    check_attention(batch, call(batch, lengths, lse=lse), lse)


@pytest.mark.parametrize("lengths", [[(1, 4000), (1, 17)], [(3, 40), (2, 1900)], [(200, 260), (90, 2500)]])
def test_attention_far_scores_and_uneven_scales(cuda, lengths):
    """One key takes nearly everything, the largest score comes late, and V's scales differ by 2^30."""
    batch = build(generator(13), lengths, 4, 1, 128, 32, 16, BF16, spread=0.0)
    q, kc, vc, ks, vs = batch[:5]
    q *= 6
    vs *= torch.exp2(torch.randint(-15, 16, vs.shape, generator=generator(14), device="cuda").float())
    check_attention(batch, call(batch, lengths, softmax_scale=0.3), softmax_scale=0.3)


@pytest.mark.parametrize("lengths", [[(1, 90)], [(6, 50), (4, 1800)], [(150, 150), (130, 2000)]])
def test_attention_nan_and_infinity_reach_only_rows_that_see_them(cuda, lengths):
    batch = build(generator(15), lengths, 4, 2, 64, 16, 16, BF16)
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    for s, (n, c) in enumerate(lengths):
        for back, cache in ((max(1, n // 2), vc), (max(1, n // 3), kc)):  # keys that only later tokens see
            t = c - back
            cache.view(torch.uint8)[tables[s, t // 16].long(), t % 16, 1, 7] = NAN_BYTE
    q[starts[1] - 1, 0, 3] = math.inf
    got = call(batch, lengths)
    want = ref.attention(q, kc, vc, ks, vs, tables, contexts, starts)[0]
    assert torch.equal(got.isnan(), want.isnan())
    assert got.isnan().any()
    fine = ~want.isnan()
    assert (got.double() - want)[fine].abs().max() <= 0.02 * want[fine].abs().max()


def test_attention_zero_scales_are_zero_keys(cuda):
    lengths = [(1, 64), (1, 1500)]
    batch = build(generator(16), lengths, 4, 1, 128, 16, 16, FP16)
    batch[3].zero_()
    check_attention(batch, call(batch, lengths))
    batch[4].zero_()
    assert (call(batch, lengths) == 0).all()


@pytest.mark.parametrize("lengths", [[(1, 400)], [(1, 3000)], [(150, 700)]])
def test_attention_skips_bad_pages(cuda, lengths):
    """Pages outside the cache are not read, and their keys count as absent."""
    batch = build(generator(17), lengths, 4, 2, 128, 16, 16, BF16)
    tables = batch[5]
    tables[0, 1], tables[0, 3], tables[0, 5] = -1, batch[1].shape[0], 2 ** 31 - 1
    check_attention(batch, call(batch, lengths))
    tables[0] = -1
    assert (call(batch, lengths) == 0).all()


@pytest.mark.parametrize("decode", [True, False])
def test_attention_strided_padded_and_cut(cuda, decode):
    """Strided q and out, wide tables, a context longer than its table, tokens behind the last sequence."""
    n = 1 if decode else 160
    lengths = [(n, 200), (n, 3 * n + 900)]
    q, kc, vc, ks, vs, tables, contexts, starts = build(generator(18), lengths, 4, 1, 128, 16, 16, BF16, extra_width=0)
    wide = torch.zeros(q.shape[0] + 5, 7 * 128, dtype=BF16, device=cuda)
    wide[:q.shape[0], :512] = q.flatten(1)
    view = wide[:q.shape[0] if decode else None, :512].unflatten(1, (4, 128))
    out = torch.full((view.shape[0], 640), 3.0, dtype=BF16, device=cuda)
    wide_tables = torch.full((2, tables.shape[1] + 9), 2 ** 30, dtype=torch.int32, device=cuda)
    wide_tables[:, :tables.shape[1]] = tables
    lse = torch.full((view.shape[0], 4), 3.0, device=cuda)
    options = {} if decode else dict(cu_seqlens_q=int32(starts), max_seqlen_q=n)
    args = (view, kc, vc, ks, vs, wide_tables[:, :tables.shape[1]], int32([contexts[0], 2 ** 30]))
    got = ops.attention_fp8(*args, out=out[:, 64:576].unflatten(1, (4, 128)), lse=lse, **options)
    full = tables.shape[1] * 16
    check_attention((q, kc, vc, ks, vs, tables, [contexts[0], full], starts), got[:q.shape[0]], lse[:q.shape[0]])
    assert (out[:, :64] == 3.0).all() and (out[:, 576:] == 3.0).all()
    assert (got[q.shape[0]:] == 3.0).all() and (lse[q.shape[0]:] == 3.0).all()


@pytest.mark.parametrize("n,announced", [(6, 2), (300, 40)])
def test_attention_rows_beyond_the_announced_longest_are_computed(cuda, n, announced):
    lengths = [(n, n + 50), (1, 60)]
    batch = build(generator(19), lengths, 4, 1, 128, 16, 16, BF16)
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    got = ops.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts), cu_seqlens_q=int32(starts),
                            max_seqlen_q=announced)
    check_attention(batch, got)


def test_attention_offsets_outside_q_are_cut(cuda):
    batch = build(generator(20), [(4, 40), (3, 1200)], 4, 1, 64, 16, 16, BF16)
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    got = ops.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts), cu_seqlens_q=int32([-5, 4, 2 ** 31 - 1]),
                            max_seqlen_q=4)
    check_attention(batch, got)
    ops.attention_fp8(q, kc, vc, ks, vs, tables, int32([-3, 40]), cu_seqlens_q=int32([9, 2, 1]), max_seqlen_q=4)
    torch.cuda.synchronize()


def test_attention_offsets_past_32_bits(cuda):
    """Pages whose byte offsets in the cache pass 2^32."""
    page, heads, dim = 256, 8, 128
    pages = (2 ** 32 + 2 ** 28) // (page * heads * dim)
    g = generator(21)
    kc = torch.zeros(pages, page, heads, dim, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.zeros(pages, 4, heads, device=cuda) for _ in range(2))
    slots = ((pages - 2) * page + torch.arange(300, device=cuda)).to(torch.int32)
    key, value = randn(g, 300, heads, dim).to(BF16), randn(g, 300, heads, dim).to(BF16)
    ops.store_kvcache_fp8(key, value, kc, vc, ks, vs, slots)
    for n in (1, 140):
        q = randn(g, n, 16, dim).to(BF16)
        tables = int32([[pages - 2, pages - 1]])
        got = ops.attention_fp8(q, kc, vc, ks, vs, tables, int32([300]), cu_seqlens_q=int32([0, n]), max_seqlen_q=n)
        check_attention((q, kc[-2:], vc[-2:], ks[-2:], vs[-2:], int32([[0, 1]]), [300], [0, n]), got)


# ---------------------------------------------------------------------------------------------------
# streams, graphs, and a layer's calls together


class Layer:
    """One layer's rotary, store and attention for sequences that grow in a paged e4m3 pool."""

    def __init__(self, g, seqs, q_heads, kv_heads, dim, page, block, pages):
        shape = (2, 1, pages, page, kv_heads, dim)
        self.pool = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        self.scales = torch.zeros(2, 1, pages, page // block, kv_heads, 1, device="cuda")
        self.kc, self.vc = self.pool[0, 0], self.pool[1, 0]
        self.ks, self.vs = self.scales[0, 0, ..., 0], self.scales[1, 0, ..., 0]
        self.table = ops.rotary_table(8192, dim, base=1e6, device="cuda")
        width = pages // seqs
        self.tables = torch.randperm(pages, generator=g, device="cuda").int()[:seqs * width].view(seqs, width)
        self.page, self.heads, self.dim = page, (q_heads, kv_heads), dim

    def rows(self, g, n):
        widths = [self.heads[0] * self.dim, self.heads[1] * self.dim, self.heads[1] * self.dim]
        qkv = randn(g, n, sum(widths)).to(BF16).split(widths, dim=1)
        return [x.view(n, -1, self.dim) for x in qkv]

    def step(self, q, k, v, positions, slots, contexts, **options):
        q, k = layer.rotary(q, k, positions, self.table)
        layer.store_kvcache_fp8(k, v, self.kc, self.vc, self.ks, self.vs, slots)
        return layer.attention_fp8(q, self.kc, self.vc, self.ks, self.vs, self.tables, contexts, **options)

    def slots_of(self, seq, positions):
        return self.tables[seq].long()[positions // self.page] * self.page + positions % self.page

    def check(self, q, got, positions_q, contexts, starts):
        turned = ref.rotary(q, positions_q, self.table)[0].to(BF16)
        # q's rounding after the rotation may differ by one step where the two sums straddle a border
        out, _, weight, size = ref.attention(turned, self.kc, self.vc, self.ks, self.vs, self.tables, contexts, starts)
        bound = ref.attention_bound(out, weight, size, BF16, max(contexts), 448 * float(self.vs.max()), self.dim)
        bound += weight * 2 * 2 * ref.half_step(BF16) * size
        assert ((got.double() - out).abs() <= bound).all()


def test_a_layer_prefills_decodes_and_moves_pages(cuda):
    """Prompts, decode steps, a page saved to the host and restored elsewhere, and more steps over it."""
    g = generator(22)
    net = Layer(g, 2, 8, 2, 128, 32, 16, 20)
    lengths, seqs = [70, 45], range(2)
    q, k, v = net.rows(g, sum(lengths))
    positions = torch.cat([torch.arange(n, device=cuda) for n in lengths])
    slots = torch.cat([net.slots_of(s, torch.arange(n, device=cuda)) for s, n in zip(seqs, lengths)]).int()
    starts = [0, 70, 115]
    kept = q.clone()
    got = net.step(q, k, v, positions, slots, int32(lengths), cu_seqlens_q=int32(starts), max_seqlen_q=70)
    net.check(kept, got, positions, lengths, starts)

    def decode():
        q, k, v = net.rows(g, 2)
        positions = torch.tensor(lengths, device=cuda)
        slots = torch.stack([net.slots_of(s, positions[s:s + 1])[0] for s in seqs]).int()
        for s in seqs:
            lengths[s] += 1
        kept = q.clone()
        got = net.step(q, k, v, positions, slots, int32(lengths))
        net.check(kept, got, positions, lengths, [0, 1, 2])
        return kept, got

    for _ in range(20):
        decode()
    # Sequence 0's first page goes to the host and comes back in an unused page, bytes and scales.
    old, new = int(net.tables[0, 0]), int(net.tables[1, -1])
    for pool in (net.pool.view(torch.uint8), net.scales):
        geometry = ops.geometry(pool)
        host = torch.empty(geometry.block_bytes, dtype=torch.uint8).pin_memory()
        ops.copy_blocks(pool, [old], [host.data_ptr()])
        torch.cuda.synchronize()
        pool[:, :, old] = 0x7F if pool.dtype == torch.uint8 else math.nan
        ops.copy_blocks(pool, [new], [host.data_ptr()], restore=True)
        torch.cuda.synchronize()
    net.tables[0, 0] = new
    net.scales[:, :, old] = 0  # the page is free again
    net.pool.view(torch.uint8)[:, :, old] = 0
    for _ in range(3):
        decode()


def test_calls_are_captured_and_replayed_with_new_lengths(cuda):
    """A decode step in a CUDA graph: contexts, slots and positions change between replays."""
    g = generator(23)
    net = Layer(g, 3, 8, 2, 64, 32, 32, 120)
    rows = net.rows(g, 3)
    static = [x.clone() for x in rows]
    positions, slots = torch.zeros(3, dtype=torch.int64, device=cuda), int32([0, 0, 0])
    contexts = int32([0, 0, 0])
    net.step(*static, positions, slots - 1, contexts)  # loads the kernels
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with the workspace of its capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(net.step(*static, positions, slots, contexts))
        graphs.append(graph)
    lengths = [0, 0, 0]
    for i in range(6):
        add = [1, 1, 0] if i % 2 else [1, 1, 1]  # a padded row: slot -1, context 0
        for x, y in zip(static, net.rows(g, 3)):
            x.copy_(y)
        kept = static[0].clone()
        positions.copy_(torch.tensor(lengths, device=cuda))
        slots.copy_(torch.stack([net.slots_of(s, torch.tensor([lengths[s]], device=cuda))[0] for s in range(3)]))
        if not add[2]:
            slots[2] = -1
        lengths = [n + a for n, a in zip(lengths, add)]
        now = lengths if add[2] else lengths[:2] + [0]
        contexts.copy_(int32(now))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        net.check(kept, outs[i % 2], positions, now, [0, 1, 2, 3])


def test_attention_on_other_streams_at_once(cuda):
    """The same call on two streams at the same time, with workspaces of their own, and through a raw handle."""
    lengths = [(1, 4000), (1, 900)]
    batch = build(generator(24), lengths, 8, 2, 128, 64, 64, BF16)
    q, kc, vc, ks, vs, tables, contexts, _ = batch
    args = (q, kc, vc, ks, vs, tables, int32(contexts))
    want = ops.attention_fp8(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        outs.append(ops.attention_fp8(*args, stream=streams[i % 2] if i < 10 else streams[i % 2].cuda_stream))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)
    check_attention(batch, want)


def test_attention_results_do_not_depend_on_the_workspace(cuda):
    lengths = [(1, 3000), (1, 1), (1, 0), (1, 7000)]
    batch = build(generator(25), lengths, 8, 2, 128, 16, 16, BF16)
    q, kc, vc, ks, vs, tables, contexts, _ = batch
    need = ops.attention_fp8_workspace(4, 1, tables.shape[1], 16, 8, 2, 128)
    outs = []
    for byte in (0, 0xFF, 0x7F):
        workspace = torch.full((need,), byte, dtype=torch.uint8, device=cuda)
        outs.append(ops.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts), workspace=workspace))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    check_attention(batch, outs[0])


def test_attention_refuses_a_workspace_that_is_too_small(cuda):
    batch = build(generator(26), [(1, 3000)], 4, 1, 64, 16, 16, BF16)
    q, kc, vc, ks, vs, tables, contexts, _ = batch
    need = ops.attention_fp8_workspace(1, 1, tables.shape[1], 16, 4, 1, 64)
    small = torch.empty(need - 1, dtype=torch.uint8, device=cuda)
    with pytest.raises(kvoff.KvoffError, match=f"workspace of {need} bytes"):
        ops.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts), workspace=small)
    got = ops.attention_fp8(q, kc, vc, ks, vs, tables, int32(contexts),
                            workspace=torch.empty(need, dtype=torch.uint8, device=cuda))
    check_attention(batch, got)


@pytest.mark.parametrize("n", [1, 20, 90])
def test_attention_is_captured_on_its_first_call_and_repeats_itself(cuda, n):
    """Two graphs of one call, replayed in turn and after other work: the same bits each time."""
    lengths = [(n, 2500 + n), (n, n), (n, 1400 + n)]
    batch = build(generator(27), lengths, 8, 2, 128, 64, 32, FP16)
    q, kc, vc, ks, vs, tables, contexts, starts = batch
    args = (q, kc, vc, ks, vs, tables, int32(contexts))
    options = dict(cu_seqlens_q=int32(starts), max_seqlen_q=n)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.attention_fp8(*args, **options))
        graphs.append(graph)
    for graph in graphs + graphs:
        graph.replay()
    eager = ops.attention_fp8(*args, **options)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], eager)
    check_attention(batch, eager)


def test_attention_many_sequences_of_every_length(cuda):
    """More sequences than threads, most of them short, so that CTAs walk over many of them."""
    g = generator(28)
    contexts = torch.randint(0, 70, (700,), generator=g, device="cuda").tolist()
    contexts[5], contexts[600] = 5000, 2600
    batch = build(g, [(1, c) for c in contexts], 2, 1, 64, 16, 16, BF16)
    check_attention(batch, call(batch, [(1, c) for c in contexts], decode=True))
    lengths = [(min(c, 1 + i % 40), c) for i, c in enumerate(contexts[:120])]
    batch = build(g, lengths, 2, 1, 64, 16, 16, BF16)
    check_attention(batch, call(batch, lengths))


def test_empty_calls_do_nothing(cuda):
    kc, ks = torch.zeros(2, 16, 1, 64, device=cuda).to(torch.float8_e4m3fn), torch.ones(2, 1, 1, device=cuda)
    none = torch.empty(0, 1, 64, dtype=BF16, device=cuda)
    ops.rotary(none, none, torch.empty(0, dtype=torch.int64, device=cuda), ops.rotary_table(4, 64, device=cuda))
    ops.store_kvcache_fp8(none, none, kc, kc.clone(), ks, ks.clone(), int32([]))
    out = ops.attention_fp8(none, kc, kc, ks, ks, int32([]).view(0, 2), int32([]))
    assert out.shape == (0, 1, 64)
    q = torch.ones(2, 1, 64, dtype=BF16, device=cuda)
    out = ops.attention_fp8(q, kc, kc, ks, ks, torch.empty(2, 0, dtype=torch.int32, device=cuda), int32([5, 0]))
    assert (out == 0).all()  # tables without pages: every context is cut to none


def test_one_token_with_any_stride(cuda):
    g = generator(31)
    q = randn(g, 1, 4, 64).to(BF16)
    odd = q.as_strided((1, 4, 64), (1, 64, 1))
    table, positions = ops.rotary_table(100, 64, device=cuda), torch.tensor([7], device=cuda)
    out = torch.empty_like(q), torch.empty_like(q)
    ops.rotary(odd, odd, positions, table, out=out)
    check_rotary(q, out[0], positions, table, False, False)
    check_rotary(q, out[1], positions, table, False, False)
