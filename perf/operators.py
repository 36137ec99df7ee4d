"""Cases of the operators that run a layer's attention over an 8-bit paged KV cache.

Three operators, in the order in which a layer calls them:

* rotary positions of q and k (`ops.rotary`),
* the store of new K and V rows into an e4m3 paged cache with one scale for each block of tokens and
  head (`ops.store_kvcache_fp8`),
* attention over that cache (`ops.attention_fp8`), one token a sequence or many.

`run` computes them in elementary torch operations, or with the framework's kernels where `own` is
true. `exact` computes them in 64 bits from their definitions.

Layouts: a cache is [pages, page, heads, dim] e4m3 with scales [pages, page / block, heads] fp32; a
sequence's pages stand in its row of the block table. A scale block is `scale_block` tokens of a page.
"""

import math
import random

import torch

own = False

FP8_MAX = 448.0
MIN_EXPONENT = -100  # of a scale: a block of zeros has the scale 2^-100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------
# cases


def _rotary(name, tokens, q_heads, kv_heads, dim, rotary_dim, interleaved, inverse, scaling, far, dtype):
    case = {"op": "rotary", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": rotary_dim, "interleaved": interleaved, "inverse": inverse,
            "scaling": scaling, "far": far, "dtype": dtype}
    return {"name": name, **case} if name else case


def _store(name, seqs, tokens, kv_heads, dim, page, scale_block, skipped, dtype):
    case = {"op": "store", "seqs": seqs, "tokens": tokens, "kv_heads": kv_heads, "dim": dim,
            "page": page, "scale_block": scale_block, "skipped": skipped, "dtype": dtype}
    return {"name": name, **case} if name else case


def _attention(name, seqs, q_len, context, ragged, q_heads, kv_heads, dim, page, scale_block, dtype):
    case = {"op": "attention", "seqs": seqs, "q_len": q_len, "context": context, "ragged": ragged,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "scale_block": scale_block, "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One decode step of four agents: latency is all of it.
        _rotary("rotary-decode", 4, 32, 8, 128, 128, False, False, "none", 40960, "bf16"),
        # A prompt chunk of an agent's first turn.
        _rotary("rotary-prefill", 4096, 32, 8, 128, 128, False, False, "yarn", 131072, "bf16"),
        # The gradient of a layer that turns half of each head in interleaved pairs, odd length.
        _rotary("rotary-partial-gradient", 1023, 16, 4, 128, 64, True, True, "llama3", 32768, "fp16"),
        # The largest batch of prompt tokens that an engine schedules at once, 64 query heads.
        _rotary("rotary-large", 16384, 64, 8, 128, 128, False, False, "linear", 65536, "bf16"),
        # Four agents append one token each, in the middle of their pages.
        _store("store-decode", 4, 4, 8, 128, 256, 64, False, "bf16"),
        # A prompt chunk of one sequence.
        _store("store-prefill", 1, 4096, 8, 128, 256, 64, False, "bf16"),
        # A full batch of ragged prompts in short pages, with padded tokens between them.
        _store("store-ragged", 24, 16384, 8, 128, 16, 16, True, "fp16"),
        # The first tokens of a short chat: a few pages, one sequence.
        _attention("attention-short", 1, 1, 300, False, 32, 8, 128, 256, 64, "bf16"),
        # One decode step of four agents with long histories.
        _attention("attention-decode", 4, 1, 34816, False, 32, 8, 128, 256, 64, "bf16"),
        # A decode batch of many chats, lengths from none (a padded row) to thousands, short pages.
        _attention("attention-decode-ragged", 64, 1, 8192, True, 64, 8, 128, 16, 16, "fp16"),
        # A tool's result of 2048 tokens over a restored history.
        _attention("attention-extend", 1, 2048, 34816, False, 32, 8, 128, 256, 64, "bf16"),
        # Ragged prompts in one batch, heads of 64.
        _attention("attention-extend-ragged", 6, 512, 8192, True, 16, 4, 64, 48, 16, "bf16"),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["rotary", "store", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "rotary":
        rotary_dim = rng.choice([dim, dim, dim // 2, dim // 4])
        return _rotary(None, _log(rng, 1, 16384), kv_heads * rng.choice([1, 2, 4, 7, 8]), kv_heads, dim, rotary_dim,
                       rng.random() < 0.5, rng.random() < 0.4, rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                       _log(rng, 4096, 131072), dtype)
    page, scale_block = rng.choice([(16, 16), (48, 16), (64, 32), (256, 16), (256, 64), (256, 256)])
    if op == "store":
        tokens = _log(rng, 1, 16384)
        return _store(None, min(tokens, _log(rng, 1, 64)), tokens, kv_heads, dim, page, scale_block,
                      rng.random() < 0.3, dtype)
    group = rng.choice([1, 2, 4, 5, 8])
    seqs, context = _log(rng, 1, 64), _log(rng, 1, 34816)
    q_len = 1 if rng.random() < 0.5 else min(context, _log(rng, 2, 2048))
    # No more scores than the largest listed case has, and no more cached values.
    while seqs > 1 and (seqs * kv_heads * group * q_len * context > 1.0e9 or seqs * context * kv_heads * dim > 1.5e8):
        seqs //= 2
    if kv_heads * group * q_len * context > 2.2e9:
        q_len = max(1, int(2.2e9 / (kv_heads * group * context)))
    return _attention(None, seqs, q_len, context, seqs > 1 and rng.random() < 0.7, kv_heads * group, kv_heads, dim,
                      page, scale_block, dtype)


# ---------------------------------------------------------------------------------------------------
# what a program has in hand


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _frequencies(case):
    """Angle per position of each pair (float64), and the factor that cos and sin carry."""
    half = case["rotary_dim"] // 2
    base, kind, factor, original = 1000000.0, case["scaling"], 4.0, max(2048, case["far"] // 4)
    if kind == "ntk":
        base *= factor ** (case["rotary_dim"] / max(1, case["rotary_dim"] - 2))
    inv = 1.0 / base ** (torch.arange(half, dtype=torch.float64) / half)
    attention = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        def pair(turns):  # the pair that turns this often over the original length
            return case["rotary_dim"] * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), case["rotary_dim"] - 1)
        ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        attention = 0.1 * math.log(factor) + 1.0
    elif kind == "llama3":
        turns = original * inv / (2 * math.pi)
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        inv = (1 - smooth) * inv / factor + smooth * inv
    return inv, attention


def _power_of_two(amax):
    """The smallest power of two s with amax <= 448 s, at least 2^MIN_EXPONENT."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, MIN_EXPONENT).clamp(min=MIN_EXPONENT)
    return torch.ldexp(torch.ones_like(amax), e)


def _cache(g, pages, case):
    """A cache that holds something in every row: payload and scales."""
    page, block, heads, dim = case["page"], case["scale_block"], case["kv_heads"], case["dim"]
    channels = torch.exp(0.7 * _randn(g, heads, dim))  # a few strong channels, as keys have
    x = _randn(g, pages, page // block, block, heads, dim).mul_(channels)
    scale = _power_of_two(x.abs().amax(dim=(2, 4)))
    x.div_(scale[:, :, None, :, None])
    return x.to(torch.float8_e4m3fn).view(pages, page, heads, dim), scale


def _lengths(case):
    """(new tokens, context) of each sequence: the case alone decides, a seed only their order."""
    n = case["seqs"]
    if not case["ragged"]:
        return [(case["q_len"], max(case["context"], case["q_len"]))] * n
    r, got = random.Random(n * 1000003 + case["context"]), []
    for i in range(n):
        q = case["q_len"] if i == 0 or case["q_len"] == 1 else _log(r, 1, case["q_len"])
        c = case["context"] if i == 0 else _log(r, 1, case["context"])
        got.append((q, max(q, c)))
    if case["q_len"] == 1 and n > 2:
        got[1] = (1, 0)  # a padded row of a captured batch: nothing to attend to
    return got


def _pages_of(case, g, contexts, total=0):
    page = case["page"]
    need = [-(-c // page) for c in contexts]
    total = max(total, sum(need) + 3)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return total, tables


def prepare(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        n, dim = case["tokens"], case["dim"]
        heads = (case["q_heads"], case["kv_heads"], case["kv_heads"])
        q, k, _ = _randn(g, n, sum(heads) * dim).to(dtype).split([h * dim for h in heads], dim=1)
        inv, attention = _frequencies(case)
        inv = inv.cuda()
        angle = torch.arange(case["far"], device="cuda", dtype=torch.float64)[:, None] * inv
        table = torch.cat([angle.cos() * attention, angle.sin() * attention], dim=1).float()
        start = torch.randint(0, max(1, case["far"] - n), (1,), generator=g, device="cuda")
        positions = (start + torch.arange(n, device="cuda")) % case["far"]
        q, k = q.view(n, heads[0], dim), k.view(n, heads[1], dim)
        return {"case": case, "q": q, "k": k, "positions": positions, "table": table, "inv": inv,
                "attention": attention, "out": (torch.empty_like(q, memory_format=torch.contiguous_format),
                                                torch.empty_like(k, memory_format=torch.contiguous_format))}
    if case["op"] == "store":
        n, seqs, page, block = case["tokens"], case["seqs"], case["page"], case["scale_block"]
        share = [n // seqs + (i < n % seqs) for i in range(seqs)]
        r = random.Random(seed)
        begin = [r.randrange(page) for _ in share]  # where in a page each sequence goes on
        most = sum(-(-(s + page - 1) // page) for s in share) + 3  # wherever they begin
        pages, tables = _pages_of(case, g, [b + s for b, s in zip(begin, share)], most)
        slots = torch.cat([tables[i].long()[(torch.arange(s, device="cuda") + b) // page] * page
                           + (torch.arange(s, device="cuda") + b) % page
                           for i, (s, b) in enumerate(zip(share, begin))]).to(torch.int32)
        if case["skipped"]:
            slots[torch.rand(n, generator=g, device="cuda") < 0.05] = -1
        width = case["kv_heads"] * case["dim"]
        rows = _randn(g, n, 2 * width)
        rows *= torch.exp(0.7 * _randn(g, 2 * width))
        key, value = rows.to(dtype).split(width, dim=1)
        shape = (n, case["kv_heads"], case["dim"])
        (kc, ks), (vc, vs) = _cache(g, pages, case), _cache(g, pages, case)
        return {"case": case, "key": key.view(shape), "value": value.view(shape), "slots": slots,
                "k_cache": kc, "k_scale": ks, "v_cache": vc, "v_scale": vs}
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    contexts = [c for _, c in lengths]
    starts = [0]
    for q, _ in lengths:
        starts.append(starts[-1] + q)
    pages, tables = _pages_of(case, g, contexts)
    (kc, ks), (vc, vs) = _cache(g, pages, case), _cache(g, pages, case)
    q = _randn(g, starts[-1], case["q_heads"], case["dim"])
    return {"case": case, "q": q.to(dtype), "k_cache": kc, "k_scale": ks, "v_cache": vc, "v_scale": vs,
            "tables": tables, "contexts": torch.tensor(contexts, dtype=torch.int32, device="cuda"),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "most": max(q for q, _ in lengths)}


# ---------------------------------------------------------------------------------------------------
# one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(op, state)
    return {"rotary": _plain_rotary, "store": _plain_store, "attention": _plain_attention}[op](state)


def _run_own(op, s):
    import sys

    if "kv-cache-offloading_b200" not in sys.path:
        sys.path.insert(0, "kv-cache-offloading_b200")
    from kvoff import ops

    case = s["case"]
    if op == "rotary":
        return ops.rotary(s["q"], s["k"], s["positions"], s["table"], interleaved=case["interleaved"],
                          inverse=case["inverse"], out=s["out"])
    if op == "store":
        ops.store_kvcache_fp8(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                              s["slots"])
        return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if case["q_len"] == 1:
        return ops.attention_fp8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"],
                                 s["contexts"])
    return ops.attention_fp8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"],
                             s["contexts"], cu_seqlens_q=s["starts"], max_seqlen_q=s["most"])


def _plain_rotary(s):
    case, half = s["case"], s["case"]["rotary_dim"] // 2
    angle = s["positions"].double()[:, None] * s["inv"]  # positions are far: 64 bits
    cos = (angle.cos() * s["attention"]).float()[:, None]
    sin = (angle.sin() * s["attention"]).float()[:, None]
    sin = -sin if case["inverse"] else sin

    def turn(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:2 * half]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([turned, y[..., 2 * half:]], dim=-1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _plain_store(s):
    block = s["case"]["scale_block"]
    kept = s["slots"] >= 0
    slots = s["slots"][kept].long()
    group = slots // block  # scale blocks tile the pages, so slots count them through
    touched, which = torch.unique(group, return_inverse=True)
    opened = torch.zeros(len(touched), dtype=torch.int32, device=slots.device)
    opened.index_reduce_(0, which, (slots % block == 0).to(torch.int32), "amax")

    def put(rows, cache, scale):
        pages, page, heads, dim = cache.shape
        x = rows[kept].float()
        size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        amax = torch.zeros(len(touched), heads, device=x.device).index_reduce_(0, which, size, "amax")
        scales = scale.view(-1, heads)
        old = torch.where(opened[:, None] > 0, 0.0, scales[touched])
        new = torch.maximum(_power_of_two(amax), old)
        payload = cache.view(torch.uint8).view(-1, block, heads, dim)
        rest = payload[touched]
        again = (rest.view(torch.float8_e4m3fn).float() * (old / new)[:, None, :, None]).to(torch.float8_e4m3fn)
        payload[touched] = torch.where(opened[:, None, None, None] > 0, rest, again.view(torch.uint8))
        y = (x / new[which][..., None]).to(torch.float8_e4m3fn)
        payload.view(-1, heads, dim)[slots] = y.view(torch.uint8)
        scales[touched] = new

    put(s["key"], s["k_cache"], s["k_scale"])
    put(s["value"], s["v_cache"], s["v_scale"])
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_attention(s):
    case = s["case"]
    heads, dim, page, block = case["kv_heads"], case["dim"], case["page"], case["scale_block"]
    group = case["q_heads"] // heads
    n, width = s["tables"].shape
    most = s["most"]

    def gather(cache, scale):  # [n, heads, keys, dim]
        at = s["tables"].long().clamp(min=0)
        x = cache.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        x = x.view(n, width, page // block, block, heads, dim) * scale[at][:, :, :, None, :, None]
        return x.view(n, width * page, heads, dim).transpose(1, 2)

    contexts, starts = s["contexts"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    at = starts[:-1, None] + torch.arange(most, device="cuda")  # the tokens, padded to the longest
    real = torch.arange(most, device="cuda") < new[:, None]
    q = s["q"][torch.where(real, at, 0)].float()  # [n, most, q_heads, dim]
    q = q.view(n, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, group * most, dim)
    scores = q @ gather(s["k_cache"], s["k_scale"]).transpose(-1, -2)
    scores = scores.mul_(1.0 / math.sqrt(dim)).view(n, heads, group, most, width * page)
    last = contexts[:, None] - new[:, None] + torch.arange(most, device="cuda")  # a token's own key
    hidden = torch.arange(width * page, device="cuda") > last[..., None]  # [n, most, keys]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores.view(n, heads, group * most, -1) @ gather(s["v_cache"], s["v_scale"])
    out = out.view(n, heads, group, most, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, case["q_heads"], dim)
    return out[real].to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------
# the least that a pass has to move and compute


def work(case):
    if case["op"] == "rotary":
        heads = case["q_heads"] + case["kv_heads"]
        row = heads * case["dim"]
        return {"bytes": case["tokens"] * (4 * row + 4 * case["rotary_dim"] + 8),
                "flops": case["tokens"] * heads * case["rotary_dim"] * 3}
    if case["op"] == "store":
        row = 2 * case["kv_heads"] * case["dim"]
        blocks = case["tokens"] / min(case["scale_block"], max(1.0, case["tokens"] / case["seqs"]))
        return {"bytes": case["tokens"] * (3 * row + 4) + 2 * 8 * blocks * case["kv_heads"],
                "flops": case["tokens"] * 3 * row}
    keys = sum(c for _, c in _lengths(case))
    rows = sum(q for q, _ in _lengths(case))
    pairs = sum(q * c - q * (q - 1) // 2 for q, c in _lengths(case) if c)
    cache = 2 * keys * case["kv_heads"] * (case["dim"] + 4 / case["scale_block"])
    return {"bytes": cache + 4 * rows * case["q_heads"] * case["dim"] + 4 * keys / case["page"],
            "flops": 4 * case["dim"] * case["q_heads"] * pairs}


# ---------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "store": _exact_store, "attention": _exact_attention}[case["op"]](case, s)


def _exact_rotary(case, s):
    # A pair is a complex number, and a position turns it by an angle and stretches it.
    half = case["rotary_dim"] // 2
    inv, stretch = _frequencies(case)
    angle = torch.outer(s["positions"].double(), inv.cuda())
    turn = torch.polar(torch.full_like(angle, stretch), -angle if case["inverse"] else angle)

    def one(x):
        y = x.double().clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return one(s["q"]), one(s["k"])


def _round_e4m3(x):
    """float64 -> the nearest e4m3 value, ties to even: 3 bits after the leading one, steps of 2^-9 at least."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-FP8_MAX, FP8_MAX)


def _exact_store(case, s):
    block, heads = case["scale_block"], case["kv_heads"]
    members = {}
    for i, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            members.setdefault(slot // block, []).append((slot % block, i))

    def one(rows, cache, scale):
        rows, dim = rows.double().cpu(), case["dim"]
        payload = cache.float().double().cpu().view(-1, block, heads, dim)
        scales = scale.double().cpu().view(-1, heads)
        for at, found in members.items():
            offsets, tokens = [o for o, _ in found], [i for _, i in found]
            x = rows[tokens]
            need = torch.log2(x.abs().amax(dim=(0, 2)) / FP8_MAX).ceil().clamp(min=MIN_EXPONENT)
            new = torch.exp2(need)
            if 0 not in offsets:
                new = torch.maximum(new, scales[at])
                payload[at] = _round_e4m3(payload[at] * (scales[at] / new)[None, :, None])
            scales[at] = new
            payload[at, offsets] = _round_e4m3(x / new[None, :, None])
        return payload.view(cache.shape), scales.view(scale.shape)

    (k, ks), (v, vs) = one(s["key"], s["k_cache"], s["k_scale"]), one(s["value"], s["v_cache"], s["v_scale"])
    return k, v, ks, vs


def _exact_attention(case, s):
    group, page, block = case["q_heads"] // case["kv_heads"], case["page"], case["scale_block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, contexts = s["starts"].tolist(), s["contexts"].tolist()
    for i, keys in enumerate(contexts):
        a, b = starts[i], starts[i + 1]
        if not keys or a == b:
            continue
        t = torch.arange(keys, device="cuda")
        where = s["tables"][i].long()[t // page]
        limit = keys - (b - a) + 1 + torch.arange(b - a, device="cuda")  # keys that each token sees
        for h in range(case["kv_heads"]):
            k = s["k_cache"][:, :, h].float()[where, t % page].double()
            v = s["v_cache"][:, :, h].float()[where, t % page].double()
            k *= s["k_scale"][where, t % page // block, h].double()[:, None]
            v *= s["v_scale"][where, t % page // block, h].double()[:, None]
            for j in range(h * group, (h + 1) * group):
                x = s["q"][a:b, j].double() @ k.T / case["dim"] ** 0.5
                x.masked_fill_(t >= limit[:, None], -math.inf)
                out[a:b, j] = torch.softmax(x, dim=-1) @ v
    return out
