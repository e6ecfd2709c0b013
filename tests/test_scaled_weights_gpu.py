"""How exact the softmax weights of attention over a cache of 8 bits are, by bounds on each result that follow from its own weights and values."""

import pytest
import torch

from test_scaled_attention_gpu import Batch, kernels

pytestmark = pytest.mark.gpu


def wanted_and_spread(batch, window=0, keep=0):
    """Of every result: itself, the weighted distance of its values from it (sum of p |v - out|), and their weighted size (sum of p |v|), in 64 bits."""
    k_held, v_held = (p.held() for p in batch.planes)
    q = batch.q.double().view(-1, batch.heads, batch.size)
    out, spread, size = (torch.zeros_like(q) for _ in range(3))
    for r in range(len(q)):
        p, b = int(batch.positions[r]), int(batch.requests[r])
        keys = torch.arange(p + 1)
        if window:
            keys = keys[(keys > p - window) | (keys < keep)]
        pages = batch.tables[b].long()[keys // batch.page]
        k, v = (t[pages, :, keys % batch.page].repeat_interleave(batch.heads // batch.kv_heads, dim=1) for t in (k_held, v_held))
        w = torch.softmax(torch.einsum("hd,khd->hk", q[r], k) * batch.size**-0.5, dim=1)
        out[r] = torch.einsum("hk,khd->hd", w, v)
        spread[r] = torch.einsum("hk,khd->hd", w, (v - out[r]).abs())
        size[r] = torch.einsum("hk,khd->hd", w, v.abs())
    return [t.reshape(len(q), -1) for t in (out, spread, size)]


def within(got, batch, weight_error, **options):
    """got: float32 results of bfloat16 queries. A weight is off by ``weight_error`` of itself as it is rounded, and with its score: a sum of exact products in 32-bit with
    at most 16 roundings in a row for every 64 elements, its scaling, the maximum's subtraction and the power, four more, each 2^-24 of |q| |k| scale at most, and twice that as
    numerator and denominator both have it. Where every weight p_j is off by e_j of itself, their weighted mean is off by at most max |e_j| sum p_j |v_j - mean| / (1 - max |e_j|).
    Sums over keys, lanes, waves and runs, and the division: 32 roundings of sum p |v|."""
    want, spread, size = wanted_and_spread(batch, **options)
    score = float(batch.q.double().view(-1, batch.size).norm(dim=1).max() * batch.planes[0].held().norm(dim=-1).max()) * batch.size**-0.5
    error = weight_error + 2.0**-24 * 2 * (16 * max(1.0, batch.size / 64) + 4) * score
    off, bound = (got.double().cpu() - want).abs(), error / (1 - error) * spread + 32 * 2.0**-24 * size
    assert bool((off <= bound).all()), f"{float((off / bound).max()):.3g} times what is allowed"


@pytest.mark.parametrize("heads,kv_heads,size,page", [(4, 4, 64, 64), (8, 2, 128, 64), (20, 1, 64, 16), (2, 1, 80, 32), (2, 2, 256, 64)])
@pytest.mark.parametrize("runs", [False, True], ids=["whole", "runs"])
def test_rows_keep_their_weights_to_sixteen_bits(heads, kv_heads, size, page, runs, monkeypatch):
    """What decodes: weights as two numbers of bfloat16, the second what the first leaves: off by 2^-8 of 2^-8 of themselves."""
    if runs:
        monkeypatch.setattr(kernels(), "scaled_cut", lambda *_: (1, 2, 10))
    batch = Batch("bf16", heads, kv_heads, size, page, [0, 15, 63, 64, 200, 900], [1] * 6, seed=size + heads)
    within(batch.run(wide_out=True), batch, 2.0**-16)
    within(batch.run(wide_out=True, window=90, keep_first=20), batch, 2.0**-16, window=90, keep=20)


def test_rows_beside_portions_keep_theirs():
    batch = Batch("bf16", 4, 2, 64, 64, [300, 7, 40], [1, 3, 30], seed=2)
    before = kernels().launch_counts()
    got = batch.run(wide_out=True, short_rows=4, short_requests=2)
    assert "scaled_attention_mixed" in kernels().launches_since(before)
    within(got, batch, 2.0**-8)
    batch.q, batch.positions, batch.requests = (t[:4] for t in (batch.q, batch.positions, batch.requests))
    within(got[:4], batch, 2.0**-16)


@pytest.mark.parametrize("heads,kv_heads,size,page", [(4, 4, 64, 64), (8, 2, 128, 64), (40, 2, 64, 16), (104, 2, 128, 64), (2, 1, 80, 32), (2, 2, 256, 64)])
def test_portions_round_their_weights_once(heads, kv_heads, size, page):
    """Half a step of bfloat16, 2^-8, of each weight; in launches of few blocks, of more, and of plenty."""
    batch = Batch("bf16", heads, kv_heads, size, page, [0, 37], [260, 61] if heads <= 8 else [520, 61], seed=size + heads)
    within(batch.run(wide_out=True), batch, 2.0**-8)
