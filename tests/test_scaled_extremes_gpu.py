"""Attention over a cache of 8 bits where a sink is far above or far below every score, against the plain implementation in 64 bits."""

import pytest
import torch

from test_scaled_attention_gpu import DEVICE, Batch, check, kernels

pytestmark = pytest.mark.gpu
SINKS = [60.0, 88.0, 91.0, 130.0, 1000.0, 3e38, -60.0, -1000.0, -3e38, 0.0, 100.5, 200.25]   # e^88.8 is past the largest number of 32 bits


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("way", ["rows", "runs", "portions", "both", "both-in-two"])
def test_sinks_far_from_the_scores(dtype, size, way, monkeypatch):
    K = kernels()
    contexts, news = {"rows": ([0, 40, 300], [1, 1, 1]), "runs": ([0, 700, 1300], [1, 1, 1]), "portions": ([0, 90], [70, 33])}.get(way, ([700, 0, 40], [1, 50, 20]))
    batch = Batch(dtype, 12, 4, size, 64, contexts, news, seed=31)
    sinks = torch.tensor(SINKS)
    options = {}
    if way == "runs":
        monkeypatch.setattr(K, "scaled_cut", lambda *_: (1, 3, 8))
    if way.startswith("both"):
        monkeypatch.setattr(K, "scaled_mixes", lambda *_: way == "both")
        options = dict(short_rows=1, short_requests=1)
    before = K.launch_counts()
    got = batch.run(sinks=sinks.to(DEVICE), **options)
    ran = K.launches_since(before)
    assert ("scaled_attention_mixed" in ran) == (way == "both") and (way != "runs" or "scaled_attention_merge" in ran)
    check(batch, got, sinks=sinks)
