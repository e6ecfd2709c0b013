"""Runs of a row's keys over a cache of 8 bits, put together by a kernel of their own: with everything that the put-together results are given besides."""

import pytest
import torch

from plain_scaled import attended
from test_scaled_attention_gpu import DEVICE, Batch, check, close, kernels

SINKS = torch.tensor([0.5, -3.0, 4.0, 0.0, 6.0, -1.0])
OPTIONS = [dict(sinks=SINKS), dict(softcap=3.0), dict(window=900), dict(window=300, keep_first=130), dict(window=64 * 5, keep_first=64), dict(chunk=700), dict(chunk=64),
           dict(window=777, keep_first=5, softcap=4.0, sinks=SINKS)]
CUTS = [(1, 1, 40), (2, 3, 14), (8, 5, 8), (1, 7, 3)]


def long_rows(dtype, size=64, page=64, seed=9):
    return Batch(dtype, 6, 3, size, page, [2500, 0, 64 * 7 - 1, 64 * 7, 1000, 63], [1] * 6, seed=seed)


def on_device(options):
    return {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in options.items()}


def merged(batch, **options):
    """The batch's results, from runs that were put together."""
    before = kernels().launch_counts()
    got = batch.run(**on_device(options))
    assert "scaled_attention_merge" in kernels().launches_since(before)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("cut", CUTS, ids=str)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(k if isinstance(v, torch.Tensor) else f"{k}{v}" for k, v in o.items()))
def test_runs_with_masks_caps_and_sinks(options, dtype, cut, monkeypatch):
    batch = long_rows(dtype)
    monkeypatch.setattr(kernels(), "scaled_cut", lambda *_: cut)
    check(batch, merged(batch, **options), **options)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size,page", [("bf16", 128, 64), ("bf16", 80, 16), ("f32", 48, 32), ("bf16", 256, 16), ("f32", 208, 64)])
def test_runs_of_other_heads(dtype, size, page, monkeypatch):
    batch = long_rows(dtype, size, page, seed=size)
    monkeypatch.setattr(kernels(), "scaled_cut", lambda *_: (1, 3, 14))
    for options in (OPTIONS[3], OPTIONS[-1]):
        check(batch, merged(batch, **options), **options)


@pytest.mark.gpu
@pytest.mark.parametrize("cut", CUTS, ids=str)
def test_runs_into_every_kind_of_result(cut, monkeypatch):
    """Wide results, columns of a wider tensor on no 16 bytes, and rows in the packed layout, which the next product takes."""
    K, batch, options = kernels(), long_rows("bf16"), OPTIONS[-1]
    monkeypatch.setattr(K, "scaled_cut", lambda *_: cut)
    plain = merged(batch, **options)
    wide = merged(batch, wide_out=True, **options)
    assert wide.dtype == torch.float32 and torch.equal(wide.bfloat16(), plain)
    into = torch.full((6, 500), 5.0, dtype=torch.bfloat16, device=DEVICE)
    merged(batch, out=into[:, 7 : 7 + 384], **options)
    assert torch.equal(into[:, 7 : 7 + 384], plain) and bool((into[:, :7] == 5.0).all()) and bool((into[:, 7 + 384 :] == 5.0).all())
    packed = merged(batch, packed_out=True, **options)
    assert isinstance(packed, K.PackedRows)
    assert torch.equal(K.linear(packed, K.pack_matrix(torch.eye(384, dtype=torch.bfloat16, device=DEVICE)), out_dtype=torch.float32), plain.float())
    check(batch, plain, **options)


@pytest.mark.gpu
def test_rows_that_see_nothing_among_rows_of_runs(monkeypatch):
    batch = long_rows("bf16")
    monkeypatch.setattr(kernels(), "scaled_cut", lambda *_: (2, 3, 14))
    want = batch.want(**OPTIONS[0])
    batch.requests[0], batch.positions[4] = -1, -1
    got = merged(batch, **OPTIONS[0])
    assert not bool(got[0].any()) and not bool(got[4].any())
    kept = [1, 2, 3, 5]
    close(got[kept], want[kept], batch)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_the_cut_that_calls_choose_reaches_the_runs(dtype):
    """As the engine asks for it, nothing replaced: 17 rows of 12 heads, the longest with 4,096 keys; 48 rows of grouped heads."""
    for heads, kv_heads, rows in ((12, 12, 17), (8, 1, 48)):
        batch = Batch(dtype, heads, kv_heads, 64, 64, [4095, 100, 2000] + [30 * r for r in range(rows - 3)], [1] * rows, seed=rows)
        sinks = torch.linspace(-2.0, 5.0, heads)
        for options in (dict(sinks=sinks), dict(window=3500, keep_first=9, sinks=sinks)):
            check(batch, merged(batch, **options), **options)


def test_what_these_tests_would_notice():
    """A sink left out, counted twice or given to the wrong head, a window, a chunk or a cap that is not there, are all outside the tolerance (a window that is off by one
    key of 300 outside that of 32 bits alone)."""
    for dtype in ("bf16", "f32"):
        batch = long_rows(dtype)
        q, held = batch.q.double().view(-1, batch.heads, batch.size), [p.held() for p in batch.planes]

        def plain(**options):
            return attended(q, *held, batch.requests, batch.positions, batch.tables, batch.size**-0.5, **options).reshape(len(q), -1)

        for wanted, planted in ((dict(sinks=SINKS), dict()), (dict(sinks=SINKS), dict(sinks=SINKS + 0.6931)), (dict(sinks=SINKS), dict(sinks=SINKS.roll(1))),
                                (dict(window=300, keep=130), dict(window=300)), (dict(window=300, keep=130), dict(window=299, keep=130)), (dict(chunk=700), dict()),
                                (dict(softcap=3.0), dict()), (dict(softcap=3.0), dict(softcap=3.5))):
            if dtype == "bf16" and planted.get("window") == 299:
                continue
            with pytest.raises(AssertionError):
                close(plain(**planted), plain(**wanted), batch)
