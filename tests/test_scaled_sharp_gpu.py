"""GPT-2 over a cache of 8 bits with weights whose softmaxes are sharp: a wrong key, page or scale moves the logits by much more than rounding does."""

import json

import numpy as np
import pytest

import plain_gpt2
from conftest import TINY_A, random_tokens, sharpen_attention
from test_scaled_engine_gpu import STEPS, plain_gpt2_step, runner_for, step_and_held

# 32-bit: sums in another order than numpy's. bfloat16: the engine rounds where the plain run does, and may round the other way: every rounded number off by up to half a step
# moves these logits by 0.004 (test_what_these_tolerances_would_notice)
TOLERANCE = {"float32": 3e-4, "bfloat16": 1e-2}


def sharp_weights(dtype, seed=3):
    weights = plain_gpt2.random_weights(dict(TINY_A), seed)
    sharpen_attention(weights, TINY_A)
    return plain_gpt2.bf16_weights(weights) if dtype == "bfloat16" else weights


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", STEPS, ids=str)
@pytest.mark.parametrize("page_size", [16, 64])
def test_sharp_gpt2_steps(dtype, steps, page_size, tmp_path):
    weights = sharp_weights(dtype)
    rounded = plain_gpt2.stored_as_bf16 if dtype == "bfloat16" else (lambda x: x)
    w = {name: t.astype(np.float64) for name, t in weights.items()}
    model, cache, runner = runner_for(dict(TINY_A), weights, dtype, tmp_path, page_size=page_size)
    tokens = {name: random_tokens(i, 128, TINY_A["vocab_size"]) for i, name in enumerate("ab")}
    done = {"a": 0, "b": 0}
    for step in STEPS[steps]:
        entries = []
        for name, n in step:
            if not cache.has(name):
                cache.open(name)
            entries.append((name, tokens[name][done[name] : done[name] + n]))
        logits, held = step_and_held(model, cache, runner, entries)
        row = 0
        for name, new in entries:
            want, _ = plain_gpt2_step(TINY_A, w, new, done[name], {i: held[i][name] for i in held}, rounded)
            off = np.abs(logits[row : row + len(new)] - want).max()
            assert off <= TOLERANCE[dtype] * max(np.abs(want).max(), 1.0), (name, off)
            row += len(new)
            done[name] += len(new)


def engine_for(tmp_path, weights, dtype, **options):
    from mini_llm_amd.engine.engine import Engine, EngineOptions

    if not (tmp_path / "config.json").exists():
        (tmp_path / "config.json").write_text(json.dumps(TINY_A))
        plain_gpt2.write_safetensors(tmp_path / "model.safetensors", weights)
    return Engine(tmp_path, EngineOptions(dtype=dtype, **{"max_sessions": 40, "max_length": 120, "cache_dtype": "float8", **options}))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sharp_captured_steps_are_the_eager_ones(dtype, tmp_path):
    prompts = [random_tokens(20 + i, n, TINY_A["vocab_size"]) for i, n in enumerate((3, 17, 40, 64, 1, 33))]
    weights = sharp_weights(dtype)
    with engine_for(tmp_path, weights, dtype, use_graphs=False, step_ahead=False) as engine:
        want = engine.generate(prompts, max_new_tokens=40)
    with engine_for(tmp_path, weights, dtype, portion_graph_after=1, page_size=16) as engine:
        assert engine.generate(prompts, max_new_tokens=40) == want
        assert engine.generate(prompts, max_new_tokens=40) == want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sharp_decoding_in_two_groups_side_by_side(dtype, tmp_path):
    prompts = [random_tokens(300 + i, 21, TINY_A["vocab_size"]) for i in range(40)]
    weights, results = sharp_weights(dtype), []
    for lanes in (None, 32):
        with engine_for(tmp_path, weights, dtype, page_size=16, decode_lanes_from=lanes) as engine:
            handles = [engine.try_take_cache() for _ in prompts]
            got = [[engine.prefill_greedy(h, p)] for h, p in zip(handles, prompts)]
            engine.decode_batch_enqueue(handles)
            for step in range(40):
                if step < 39:
                    engine.decode_batch_enqueue(handles)
                for tokens, token in zip(got, engine.take()):
                    tokens.append(token)
            graph, = [g for key, g in engine.runner._graphs.items() if key[:2] == (64, True)]
            assert (graph.lanes is not None) == (lanes is not None)
            results.append(got)
    assert results[0] == results[1]


def test_what_these_tolerances_would_notice():
    """In 64 bits on the CPU: keys in another order, at twice their scale, of the neighbouring page, or none at all, against the tolerances; and what rounding the other way does."""
    weights, n, heads = sharp_weights("bfloat16"), 70, TINY_A["n_head"]
    w = {name: t.astype(np.float64) for name, t in weights.items()}
    tokens = random_tokens(0, 128, TINY_A["vocab_size"])[:n]
    rng = np.random.default_rng(1)
    nothing = np.zeros((n, heads, TINY_A["n_embd"] // heads))
    held = {i: (nothing, nothing) for i in range(TINY_A["n_layer"])}
    for i in held:   # a layer's keys and values follow from what the layers below attend over
        held[i] = plain_gpt2_step(TINY_A, w, tokens, 0, held, plain_gpt2.stored_as_bf16)[1][i]

    def logits(change=lambda k: k, rounded=plain_gpt2.stored_as_bf16):
        return plain_gpt2_step(TINY_A, w, tokens, 0, {i: (change(k), v) for i, (k, v) in held.items()}, rounded)[0]

    def either_way(x):
        y = plain_gpt2.stored_as_bf16(x)
        return y + np.abs(y) * 2.0**-8 * rng.integers(-1, 2, size=y.shape)

    want = logits()
    scale = max(np.abs(want).max(), 1.0)
    assert max(np.abs(logits(rounded=either_way) - want).max() for _ in range(3)) <= 0.7 * TOLERANCE["bfloat16"] * scale
    order = rng.permutation(n)
    for planted in (lambda k: k[order], lambda k: 0 * k, lambda k: np.concatenate([k[:16], 2 * k[16:32], k[32:]]), lambda k: np.concatenate([k[16:32], k[:16], k[32:]])):
        wrong = logits(planted)
        assert np.abs(wrong - want).max() >= 8 * TOLERANCE["bfloat16"] * scale
        assert (wrong.argmax(1) != want.argmax(1)).mean() >= 0.02   # and a share of the tokens that are chosen: of 240 to 1,600 that a test compares, some
