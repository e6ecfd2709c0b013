"""The operators that keep keys and values in 8 bits and attend over them, as cases that can be timed and checked.

Two operators. ``append`` is what a layer does between its input product and its attention: the queries and keys of a step's rows are
turned by their positions, and keys and values go into the pages of a cache that holds them as 8-bit floating-point numbers with a scale
for every block of 16 tokens of a head (a block that grows past its scale is scaled over). ``attend`` is causal attention over such a
cache, through block tables, for rows that decode, for portions of prompts and for both in one step.

The cache's layout. A block is 16 tokens of one head. keys: [pages, kv heads, page / 16, head / 16, 16 tokens, 16 elements]; values: [pages, kv
heads, page / 16, head elements, 16 tokens]; scales: float32 [pages, kv heads, page / 16], powers of two, for keys and for values. A
block's scale is the smallest 2^e, e from -110 to 118, with 448 * 2^e at least as large as the largest magnitude in it.

The sizes: heads of GPT-2 (64 elements, 12 of them or 25) and grouped heads of 64 to 128 as the other designs have them, positions up to
some ten thousand, pages of 64 tokens (the engine's own)."""

from __future__ import annotations

import random

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 16            # tokens that share a scale
E_LOW, E_HIGH = -110, 118
LARGEST = 448.0       # of a number in 8 bits
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def _append(name, dtype, heads, kv_heads, head, rot, pairing, requests, new_low, new_high, lengths):
    case = {"op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head, "rot": rot, "pairing": pairing, "page": 64,
            "requests": requests, "new_low": new_low, "new_high": new_high, "lengths": lengths}
    return {"name": name, **case} if name else case


def _attend(name, dtype, heads, kv_heads, head, requests, context_low, context_high, new_low, new_high, lengths, alone=0, window=0, keep=0, chunk=0,
            softcap=0.0, sinks=False):
    """``alone``: so many of the requests bring one token however many the others bring."""
    case = {"op": "attend", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head, "page": 64, "requests": requests, "context_low": context_low,
            "context_high": context_high, "new_low": new_low, "new_high": new_high, "lengths": lengths, "alone": alone, "window": window, "keep": keep,
            "chunk": chunk, "softcap": softcap, "sinks": sinks}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one token of a chat with GPT-2 small: nothing to turn, the call's own time
        _append("append_one_token", "bf16", 12, 12, 64, 0, "half", 1, 1, 1, 1),
        # a decode step of 64 requests, grouped heads that turn; where in its block each token lies is spread
        _append("append_decode_64", "f32", 16, 4, 64, 64, "half", 64, 1, 1, 2),
        # a full step of prompt portions of ragged lengths, as the scheduler cuts them (2,048 tokens)
        _append("append_prompts_ragged", "f32", 12, 12, 64, 32, "half", 5, 150, 600, 3),
        # a long prompt, wide grouped heads, pairs of neighbours
        _append("append_prompt_8192", "bf16", 32, 8, 128, 128, "neighbours", 1, 8192, 8192, 4),
        # one token of a chat with GPT-2 small, a thousand tokens in
        _attend("decode_one_row", "bf16", 12, 12, 64, 1, 1000, 1000, 1, 1, 5),
        # a decode step of 64 requests of all lengths up to GPT-2's positions
        _attend("decode_64_ragged", "bf16", 12, 12, 64, 64, 0, 1023, 1, 1, 6),
        # long documents with grouped heads: what a cache of 8 bits is for
        _attend("decode_16_long_grouped", "bf16", 32, 8, 128, 16, 20000, 32000, 1, 1, 7),
        # scoring in 32 bits, GPT-2 XL's 25 heads
        _attend("decode_8_f32", "f32", 25, 25, 64, 8, 200, 1000, 1, 1, 8),
        # a whole prompt
        _attend("prompt_2048", "bf16", 12, 12, 64, 1, 0, 0, 2048, 2048, 9),
        # a long prompt of wide grouped heads
        _attend("prompt_8192_grouped", "bf16", 16, 2, 128, 1, 0, 0, 8191, 8191, 10),
        # portions behind what is stored, over a window that keeps the first keys, capped scores and sinks
        _attend("portions_window", "bf16", 16, 4, 64, 4, 100, 3000, 100, 700, 11, window=512, keep=4, softcap=30.0, sinks=True),
        # a step of 33 requests that decode and three portions, 32 bits
        _attend("mixed_step_f32", "f32", 12, 12, 64, 36, 10, 900, 60, 200, 12, alone=33),
    ]


def _spread(rng, low, high):
    """A whole number of low .. high, even over its logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    heads, kv_heads, head = rng.choice([(12, 12, 64), (16, 16, 64), (25, 25, 64), (16, 4, 64), (32, 8, 128), (16, 2, 128), (8, 8, 128), (9, 3, 80), (6, 2, 48), (4, 1, 256)])
    dtype, lengths = rng.choice(["bf16", "bf16", "f32"]), rng.randrange(1 << 30)
    kind = rng.choice(["append_tokens", "append_prompts", "decode", "decode", "prompts", "prompts", "mixed"])
    if kind == "append_tokens":
        return _append(None, dtype, heads, kv_heads, head, rng.choice([0, 16, head]), rng.choice(["half", "neighbours"]), _spread(rng, 1, 256), 1, 1, lengths)
    if kind == "append_prompts":
        longest = _spread(rng, 2, 8192 * 48 // (heads + 2 * kv_heads) * 128 // head)
        requests = rng.randint(1, max(1, min(8, 8192 // longest)))
        return _append(None, dtype, heads, kv_heads, head, rng.choice([0, 16, head]), rng.choice(["half", "neighbours"]), requests, max(1, longest // 3), min(longest, 8192), lengths)
    options = {}
    pick = rng.random()
    if pick < 0.2:
        options = {"window": _spread(rng, 16, 2048), "keep": rng.choice([0, 4])}
    elif pick < 0.3:
        options = {"chunk": _spread(rng, 16, 2048)}
    if rng.random() < 0.2:
        options["softcap"] = 30.0
    if rng.random() < 0.2:
        options["sinks"] = True
    if kind == "decode":
        requests = _spread(rng, 1, 128)
        longest = _spread(rng, 16, max(16, min(32000, 16 * 32000 * 8 * 128 // (requests * kv_heads * head))))
        return _attend(None, dtype, heads, kv_heads, head, requests, longest // rng.choice([1, 2, 16]), longest, 1, 1, lengths, **options)
    if kind == "prompts":
        longest = _spread(rng, 9, 4096)
        requests = rng.randint(1, max(1, min(6, 4096 // longest)))
        return _attend(None, dtype, heads, kv_heads, head, requests, 0, rng.choice([0, _spread(rng, 1, 4096)]), max(9, longest // 3), longest, lengths, **options)
    alone = _spread(rng, 1, 60)
    return _attend(None, dtype, heads, kv_heads, head, alone + rng.randint(1, 3), 0, _spread(rng, 16, 1500), 9, _spread(rng, 9, 300), lengths, alone=alone, **options)


# ---- sizes that follow from a case alone -------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens stored before the step, tokens of the step) of each request; those that bring one token come first."""
    rng = random.Random(case["lengths"])
    if case["op"] == "append":
        return [rng.randrange(20000) for _ in range(case["requests"])], [rng.randint(case["new_low"], case["new_high"]) for _ in range(case["requests"])]
    contexts = [rng.randint(case["context_low"], case["context_high"]) for _ in range(case["requests"])]
    news = [1 if i < case["alone"] else rng.randint(case["new_low"], case["new_high"]) for i in range(case["requests"])]
    return contexts, news


def _first_key(case, position):
    if case["chunk"]:
        return position - position % case["chunk"]
    return max(0, position - case["window"] + 1) if case["window"] else 0


def work(case):
    heads, kv_heads, head, size = case["heads"], case["kv_heads"], case["head"], BYTES[case["dtype"]]
    contexts, news = _lengths(case)
    rows = sum(news)
    if case["op"] == "append":
        read = sum((c % BLOCK) + n for c, n in zip(contexts, news))   # tokens of the blocks that are written
        return {"bytes": rows * ((2 * heads + 2 * kv_heads) * head * size) + read * 2 * kv_heads * head * (1 + 2), "flops": 3 * rows * (heads + kv_heads) * case["rot"]}
    keys = pairs = 0
    for c, n in zip(contexts, news):
        seen = sum(min(case["keep"], _first_key(case, p)) + p - _first_key(case, p) + 1 for p in range(c, c + n))
        pairs += seen
        keys += c + n - _first_key(case, c) + min(case["keep"], _first_key(case, c))
    return {"bytes": keys * 2 * kv_heads * (head + 4 / BLOCK) + 2 * rows * heads * head * size, "flops": 4 * pairs * heads * head}


# ---- numbers in 8 bits with a scale a block -----------------------------------------------------------------------------------
def _exponent(largest):
    """The smallest e with 448 * 2^e >= largest (448 = 0.875 * 2^9), inside its bounds."""
    part, power = torch.frexp(largest)
    return torch.where(largest > 0, power - 9 + (part > 0.875).to(power.dtype), E_LOW).clamp(E_LOW, E_HIGH)


def _largest(values, dims):
    size = values.abs()
    return torch.where(torch.isfinite(size), size, 0.0).amax(dims)


def _codes(values, exponent):
    """values * 2^-exponent rounded to 8 bits; infinities, which the type has none of, become NaN."""
    scaled = torch.ldexp(values, -exponent)
    scaled = torch.where(torch.isinf(values), float("nan"), scaled.clamp(-LARGEST, LARGEST))
    return scaled.to(torch.float32).to(torch.float8_e4m3fn)


def _lay_keys(codes):
    """[..., tokens, head] -> [..., tokens / 16, head / 16, 16, 16]."""
    *front, tokens, head = codes.shape
    return codes.view(torch.uint8).reshape(*front, tokens // BLOCK, BLOCK, head // 16, 16).transpose(-3, -2).contiguous().view(torch.float8_e4m3fn)


def _lay_values(codes):
    """[..., tokens, head] -> [..., tokens / 16, head, 16]."""
    *front, tokens, head = codes.shape
    return codes.view(torch.uint8).reshape(*front, tokens // BLOCK, BLOCK, head).transpose(-2, -1).contiguous().view(torch.float8_e4m3fn)


def _key_numbers(codes):
    """The code numbers (uint8) of [..., tokens / 16, head / 16, 16, 16] as [..., tokens, head] of float8."""
    *front, blocks, pieces, _, _ = codes.shape
    return codes.transpose(-3, -2).reshape(*front, blocks * BLOCK, pieces * 16).view(torch.float8_e4m3fn)


def _value_numbers(codes):
    *front, blocks, head, _ = codes.shape
    return codes.transpose(-2, -1).reshape(*front, blocks * BLOCK, head).view(torch.float8_e4m3fn)


# ---- states --------------------------------------------------------------------------------------------------------------------
def _channels(shape, generator, size=1.0):
    """Numbers as products leave them: normal, a few channels of each head many times larger than the rest."""
    x = torch.randn(shape, generator=generator, device=DEVICE) * size
    gain = torch.exp(0.5 * torch.randn(shape[1:], generator=generator, device=DEVICE))
    return x * gain


def _tables(case, contexts, news, pages_of):
    """A page for every 64 tokens, in no order, and the block tables [requests, most]; the page that no request holds comes last."""
    rng = random.Random(case["lengths"] + 1)
    total = sum(pages_of)
    order = list(range(total))
    rng.shuffle(order)
    most, at, rows = max(pages_of), 0, []
    for n in pages_of:
        rows.append(order[at : at + n] + [0] * (most - n))
        at += n
    return total, rows


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, heads, kv_heads, head, page = TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head"], case["page"]
    contexts, news = _lengths(case)
    skipped = [c // page * page for c in contexts] if case["op"] == "append" else [0] * len(contexts)   # pages before these the step does not touch
    pages_of = [-(-(c + n - s) // page) for c, n, s in zip(contexts, news, skipped)]
    total, rows = _tables(case, contexts, news, pages_of)
    state = {"case": case, "tables": torch.tensor(rows, dtype=torch.int32, device=DEVICE)}
    held = {}
    for plane, size in (("k", 1.0), ("v", 0.5)):   # every place of every page holds something, as in a cache that has been in use
        x = _channels((total, page, kv_heads, head), generator, size).transpose(1, 2).reshape(total, kv_heads, page // BLOCK, BLOCK, head)
        exponent = _exponent(_largest(x, (-2, -1)))
        codes = _codes(x, exponent[..., None, None]).view(torch.uint8).reshape(total, kv_heads, page, head).view(torch.float8_e4m3fn)
        held[plane] = ((_lay_keys if plane == "k" else _lay_values)(codes), torch.ldexp(torch.ones((), device=DEVICE), exponent).contiguous())
        del x, codes
    state["k_codes"], state["k_scales"] = held["k"]
    state["v_codes"], state["v_scales"] = held["v"]
    n = sum(news)
    positions, requests, places = [], [], []
    for b, (c, m, s) in enumerate(zip(contexts, news, skipped)):
        positions += range(c, c + m)
        requests += [b] * m
        places += [rows[b][(p - s) // page] * page + p % page for p in range(c, c + m)]
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)
    state["positions"] = ints(positions)
    if case["op"] == "append":
        state["slots"] = ints(places)
        read = []   # the tokens that the written blocks hold behind the step
        for b, (c, m, s) in enumerate(zip(contexts, news, skipped)):
            read += [rows[b][(p - s) // page] * page + p % page for p in range(c // BLOCK * BLOCK, c + m)]
        state["read"] = ints(read)
        state["rows"] = torch.cat([_channels((n, count, head), generator, size).reshape(n, count * head)
                                   for count, size in ((heads, 1.0), (kv_heads, 1.0), (kv_heads, 0.5))], dim=1).to(dtype)
        rot = case["rot"]
        state["frequencies"] = (10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1))).to(DEVICE) if rot else None
        return state
    state["q"] = _channels((n, heads, head), generator, 1.0).reshape(n, heads * head).to(dtype)
    state["requests"], state["contexts"] = ints(requests), ints(contexts)
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    state["starts"] = ints(starts)
    state["sinks"] = torch.randn(heads, generator=generator, device=DEVICE) if case["sinks"] else None
    state["longest"], state["most_new"] = max(c + m for c, m in zip(contexts, news)), max(news)
    state["short_rows"], state["short_requests"] = sum(m for m in news if m <= 8), sum(m <= 8 for m in news)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
def _turned(x, positions, frequencies, rot, pairing):
    """x [rows, heads, head] in 32 bits, its first ``rot`` elements turned in pairs; the angles in 64 bits."""
    if not rot:
        return x
    angle = torch.remainder(positions.double()[:, None] * frequencies, 2.0 * torch.pi)
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if pairing == "half":
        u, v = x[..., : rot // 2], x[..., rot // 2 : rot]
        return torch.cat([u * c - v * s, v * c + u * s, x[..., rot:]], dim=-1)
    u, v = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([u * c - v * s, v * c + u * s], dim=-1).flatten(-2), x[..., rot:]], dim=-1)


def _kept(new, codes, scales, slots, read, numbers, page):
    """What the read slots hold once ``new`` [rows, kv heads, head] has gone to ``slots``."""
    pages, kv_heads, blocks_a_page = scales.shape
    head = new.shape[-1]
    block, offset = (slots // BLOCK).long(), (slots % BLOCK).long()
    n_blocks = pages * blocks_a_page
    first = torch.full((n_blocks,), BLOCK, dtype=torch.int64, device=new.device).scatter_reduce_(0, block, offset, "amin")
    largest = torch.zeros((n_blocks, kv_heads), device=new.device).scatter_reduce_(0, block[:, None].expand(-1, kv_heads), _largest(new, -1), "amax")
    old = torch.frexp(scales.transpose(1, 2).reshape(n_blocks, kv_heads))[1] - 1
    need = _exponent(largest)
    exponent = torch.where((first > 0)[:, None], torch.maximum(old, need), need)
    exponent = torch.where((first < BLOCK)[:, None], exponent, old)   # [blocks, kv heads]; blocks without a new token stay
    held = numbers(codes.view(torch.uint8)).float().reshape(pages, kv_heads, blocks_a_page, BLOCK, head).transpose(1, 2).reshape(n_blocks, kv_heads, BLOCK, head)
    held = torch.ldexp(held, (old - exponent)[..., None, None]).to(torch.float8_e4m3fn).float()
    fresh = _codes(new, exponent[block][..., None]).float()
    held[block, :, offset] = fresh
    held = torch.ldexp(held, exponent[..., None, None])
    return held[(read // BLOCK).long(), :, (read % BLOCK).long()].to(torch.bfloat16)


def _append_plain(state):
    case = state["case"]
    heads, kv_heads, head, rot = case["heads"], case["kv_heads"], case["head"], case["rot"]
    rows = state["rows"].float()
    n = rows.shape[0]
    q, k, v = rows.split([heads * head, kv_heads * head, kv_heads * head], dim=1)
    q = _turned(q.view(n, heads, head), state["positions"], state["frequencies"], rot, case["pairing"])
    k = _turned(k.view(n, kv_heads, head), state["positions"], state["frequencies"], rot, case["pairing"])
    kept_k = _kept(k, state["k_codes"], state["k_scales"], state["slots"], state["read"], _key_numbers, case["page"])
    kept_v = _kept(v.view(n, kv_heads, head), state["v_codes"], state["v_scales"], state["slots"], state["read"], _value_numbers, case["page"])
    return {"q": q.reshape(n, heads * head).to(state["rows"].dtype), "k": kept_k, "v": kept_v}


def _append_own(state):
    from mini_llm_amd.ops import kernels

    case = state["case"]
    heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
    k_pages, v_pages = kernels.ScaledPages(state["k_codes"], state["k_scales"]), kernels.ScaledPages(state["v_codes"], state["v_scales"])
    q = kernels.scaled_append(state["rows"], 0, heads * head, (heads + kv_heads) * head, k_pages, v_pages, state["slots"], state["positions"], heads, kv_heads, head,
                              head, frequencies=state["frequencies"], rot_dims=case["rot"], pairing=case["pairing"])
    k, v = kernels.scaled_rows(k_pages, v_pages, state["read"])
    return {"q": q, "k": k, "v": v}


def _gathered(codes, scales, tables, numbers):
    """[requests, kv heads, tokens, head] in 32 bits: what a request's pages hold."""
    at = tables.long()
    held = numbers(codes.view(torch.uint8)[at]).float()                   # [requests, pages, kv heads, page, head]
    b, pages, kv_heads, page, head = held.shape
    held = held * scales[at].repeat_interleave(BLOCK, dim=-1)[..., None]
    return held.transpose(1, 2).reshape(b, kv_heads, pages * page, head)


def _attend_plain(state):
    case = state["case"]
    heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
    b, q_most, group = case["requests"], state["most_new"], heads // kv_heads
    request, position = state["requests"].long(), state["positions"].long()
    place = position - state["contexts"].long()[request]
    q = torch.zeros((b, q_most, heads, head), device=DEVICE)
    q[request, place] = state["q"].float().view(-1, heads, head)
    q = q.view(b, q_most, kv_heads, group, head).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, group * q_most, head)
    k = _gathered(state["k_codes"], state["k_scales"], state["tables"], _key_numbers)
    score = torch.matmul(q, k.transpose(-1, -2)) * head ** -0.5
    del k
    tokens = score.shape[-1]
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    at = state["contexts"].long()[:, None] + torch.arange(q_most, device=DEVICE)        # [requests, rows]
    key = torch.arange(tokens, device=DEVICE)
    first = at - at % case["chunk"] if case["chunk"] else (at - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(at)
    seen = (key <= at[..., None]) & ((key >= first[..., None]) | (key < case["keep"]))
    score = score.view(b, kv_heads, group, q_most, tokens).masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sinks = state["sinks"].view(1, kv_heads, group, 1, 1)
        top = torch.maximum(top, sinks)
    weight = torch.exp(score - top)
    del score
    total = weight.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sinks - top)
    v = _gathered(state["v_codes"], state["v_scales"], state["tables"], _value_numbers)
    out = torch.matmul(weight.view(b, kv_heads, group * q_most, tokens), v).view(b, kv_heads, group, q_most, head) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(b, q_most, heads * head)
    return out[request, place].to(state["q"].dtype)


def _attend_own(state):
    from mini_llm_amd.ops import kernels

    case = state["case"]
    k_pages, v_pages = kernels.ScaledPages(state["k_codes"], state["k_scales"]), kernels.ScaledPages(state["v_codes"], state["v_scales"])
    mixed = {"short_rows": state["short_rows"], "short_requests": state["short_requests"]} if state["most_new"] > 8 else {}
    return kernels.paged_attention(state["q"], k_pages, v_pages, state["requests"], state["positions"], state["tables"], case["heads"], case["kv_heads"], case["head"],
                                   case["head"] ** -0.5, window=case["window"], max_q_len=state["most_new"], max_len=state["longest"], q_starts=state["starts"],
                                   context_lens=state["contexts"], softcap=case["softcap"], sinks=state["sinks"], chunk=case["chunk"], keep_first=case["keep"], **mixed)


def run(state):
    if state["case"]["op"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


# ---- in 64 bits ---------------------------------------------------------------------------------------------------------------------
def _exact_turn(x, position, rot, pairing):
    """x [rows, heads, head] as complex pairs times e^(i position f)."""
    if not rot:
        return x
    pair = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    e = torch.polar(torch.ones_like(pair)[None].expand(len(position), -1), position.double()[:, None] * 10000.0 ** (-2.0 * pair / rot))[:, None]
    first, second = (pair.long(), pair.long() + rot // 2) if pairing == "half" else (2 * pair.long(), 2 * pair.long() + 1)
    z = torch.complex(x[..., first], x[..., second]) * e
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_round(x):
    """x, at most 448 in size, to the nearest number of 8 bits (three bits behind the leading one, none below 2^-9), ties to even."""
    step = torch.pow(2.0, torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(x / step) * step


def _exact_exponent(largest):
    return max(E_LOW, min(E_HIGH, next(e for e in range(E_LOW, E_HIGH + 1) if LARGEST * 2.0**e >= largest)))


def _exact_append(case, state):
    heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
    rows = state["rows"].double()
    n = rows.shape[0]
    position = state["positions"].long()
    q = _exact_turn(rows[:, : heads * head].reshape(n, heads, head), position, case["rot"], case["pairing"])
    k = _exact_turn(rows[:, heads * head : (heads + kv_heads) * head].reshape(n, kv_heads, head), position, case["rot"], case["pairing"])
    v = rows[:, (heads + kv_heads) * head :].reshape(n, kv_heads, head)
    block = (state["slots"] // BLOCK).tolist()
    runs, at = [], 0
    while at < n:   # rows that fall into one block
        end = at
        while end < n and block[end] == block[at]:
            end += 1
        runs.append((at, end))
        at = end
    if len(runs) * kv_heads > 8000:
        return None
    first_slot = state["slots"].tolist()
    out = []
    for x, codes, scales, keys in ((k, state["k_codes"], state["k_scales"], True), (v, state["v_codes"], state["v_scales"], False)):
        got = []
        size = x.abs().amax(-1).tolist()
        flat = scales.double()
        for a, e in runs:
            page, inside = divmod(block[a], case["page"] // BLOCK)
            lead = first_slot[a] % BLOCK
            raw = codes.view(torch.uint8)[page, :, inside].view(torch.float8_e4m3fn).double()
            held = raw.transpose(1, 2).reshape(kv_heads, BLOCK, head) if keys else raw.transpose(1, 2)
            old = torch.log2(flat[page, :, inside]).round().tolist()
            power = []
            for g in range(kv_heads):
                need = _exact_exponent(max(size[r][g] for r in range(a, e)))
                power.append(max(need, int(old[g])) if lead else need)
            power = torch.tensor(power, dtype=torch.float64, device=x.device)
            scale = torch.pow(2.0, power)[:, None, None]
            before = held[:, :lead]
            if lead:
                before = _exact_round(before * torch.pow(2.0, torch.tensor(old, dtype=torch.float64, device=x.device) - power)[:, None, None])
            fresh = _exact_round(x[a:e].transpose(0, 1) / scale)
            got.append((torch.cat([before, fresh], dim=1) * scale).transpose(0, 1))
        out.append(torch.cat(got))
    return {"q": q.reshape(n, heads * head), "k": out[0], "v": out[1]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, state)
    heads, kv_heads, head, page = case["heads"], case["kv_heads"], case["head"], case["page"]
    contexts, news = _lengths(case)
    if sum(n * (c + n) for c, n in zip(contexts, news)) * heads * head > 4e12:
        return None
    group, at, out = heads // kv_heads, 0, []
    for b, (c, n) in enumerate(zip(contexts, news)):
        pages = state["tables"][b, : -(-(c + n) // page)].long()
        q = state["q"][at : at + n].double().view(n, heads, head)
        at += n
        row = torch.arange(c, c + n, device=DEVICE)[:, None]
        col = torch.arange(c + n, device=DEVICE)[None]
        low = row // case["chunk"] * case["chunk"] if case["chunk"] else row - case["window"] + 1 if case["window"] else row * 0
        hidden = (col > row) | ((col < low) & (col >= case["keep"]))
        heads_out = []
        for h in range(heads):
            g = h // group
            k8 = state["k_codes"].view(torch.uint8)[pages, g].view(torch.float8_e4m3fn).double()      # [pages, blocks, head / 16, 16, 16]
            k = (k8.transpose(2, 3).flatten(3) * state["k_scales"][pages, g].double()[..., None, None]).reshape(-1, head)[: c + n]
            v8 = state["v_codes"].view(torch.uint8)[pages, g].view(torch.float8_e4m3fn).double()      # [pages, blocks, head, 16]
            v = (v8.transpose(2, 3) * state["v_scales"][pages, g].double()[..., None, None]).reshape(-1, head)[: c + n]
            s = q[:, h] @ k.T / head**0.5
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            s[hidden] = -float("inf")
            if case["sinks"]:
                s = torch.cat([s, state["sinks"][h].double().expand(n, 1)], dim=1)
            p = torch.softmax(s, dim=1)[:, : c + n]
            heads_out.append(p @ v)
        out.append(torch.stack(heads_out, dim=1).reshape(n, heads * head))
    return torch.cat(out)
