"""Models over a cache of 8 bits: steps through the engine's own step function against the plain implementations, which attend over what the
cache holds at every layer of every step; and the engine's ways of running such steps against each other."""

import json

import numpy as np
import pytest
import torch

import plain_dizizen
import plain_gevulorn
import plain_gpt2
from conftest import TINY_A, random_tokens
from dizizen_cases import CASES as DIZIZEN
from gevulorn_cases import CASES as GEVULORN
from plain_scaled import coded, exponent_for

pytestmark = pytest.mark.gpu


def runner_for(config, weights, dtype, tmp_path, *, page_size=16, max_requests=4, max_length=200, graphs=True):
    from mini_llm_amd.engine import ModelRunner
    from mini_llm_amd.engine.loading import load_model, make_cache

    tmp_path.mkdir(parents=True, exist_ok=True)
    (tmp_path / "config.json").write_text(json.dumps(config))
    plain_gpt2.write_safetensors(tmp_path / "model.safetensors", weights)
    model = load_model(tmp_path, dtype)
    limit = min(max_length, model.max_positions() or max_length)
    cache = make_cache(model, max_tokens=max_requests * (limit + page_size), page_size=page_size, max_requests=max_requests, max_length=limit, cache_dtype="float8")
    return model, cache, ModelRunner(model, cache, "cuda:0", use_graphs=graphs)


def step_and_held(model, cache, runner, entries):
    """The step's logits, and of every layer call that attends what the cache held for each request when it did: {index: {request: (k, v)}}."""
    from mini_llm_amd.engine import StepEntry
    from mini_llm_amd.ops import kernels

    held = {}
    until = {name: cache.length(name) + len(tokens) for name, tokens in entries}

    def look(index, _):
        if index != "embedding" and model.schedule[index].cache in cache.group_of_layer:
            layer, shown = model.schedule[index].cache, {}
            group = cache.group_of_layer[layer]
            for name, _tokens in entries:
                pages = cache.block_table(name, group)
                slots = [pages[p // cache.page_size] * cache.page_size + p % cache.page_size if pages[p // cache.page_size] >= 0 else -1 for p in range(until[name])]
                k, v = kernels.scaled_rows(cache.k_pages[layer], cache.v_pages[layer], torch.tensor(slots, dtype=torch.int32, device="cuda:0"), out_dtype=torch.float32)
                shown[name] = (k.double().cpu().numpy(), v.double().cpu().numpy())   # (zeros where a window has given the page back)
            held[index] = shown

    logits = runner.step([StepEntry(name, tokens, list(range(len(tokens)))) for name, tokens in entries], observer=look)
    return logits.double().cpu().numpy(), held


STEPS = {"whole": [[("a", 70), ("b", 33)]], "then_tokens": [[("a", 40)], [("a", 1), ("b", 17)], [("a", 1), ("b", 1)], [("a", 1), ("b", 1)]],
         "portions": [[("a", 30), ("b", 5)], [("a", 25), ("b", 1)], [("b", 40), ("a", 1)], [("b", 3), ("a", 20)]]}


def plain_gpt2_step(config, w, tokens, position, held, rounded):
    """A step of one request in 64 bits; attention over ``held``. Returns logits and the step's exact (k, v) of every layer."""
    heads, width, eps = config["n_head"], config["n_embd"], config["layer_norm_epsilon"]
    size = width // heads
    x = plain_gpt2.embed(tokens, w["wte.weight"], w["wpe.weight"], position)
    made = []
    for i in range(config["n_layer"]):
        p = f"h.{i}."
        h = rounded(plain_gpt2.layernorm(x, w[p + "ln_1.weight"], w[p + "ln_1.bias"], eps))
        qkv = rounded(plain_gpt2.linear(h, w[p + "attn.c_attn.weight"], w[p + "attn.c_attn.bias"]))
        q, k, v = (t.reshape(-1, heads, size) for t in np.split(qkv, 3, axis=1))
        made.append((k, v))
        held_k, held_v = held[i]
        out = np.zeros_like(q)
        for r in range(len(q)):
            for g in range(heads):
                s = held_k[: position + r + 1, g] @ q[r, g] / size**0.5
                weight = np.exp(s - s.max())
                out[r, g] = (weight / weight.sum()) @ held_v[: position + r + 1, g]
        x = x + plain_gpt2.linear(rounded(out.reshape(len(q), width)), w[p + "attn.c_proj.weight"], w[p + "attn.c_proj.bias"])
        h = rounded(plain_gpt2.layernorm(x, w[p + "ln_2.weight"], w[p + "ln_2.bias"], eps))
        h = rounded(plain_gpt2.ACTIVATIONS[config["activation_function"]](plain_gpt2.linear(h, w[p + "mlp.c_fc.weight"], w[p + "mlp.c_fc.bias"])))
        x = x + plain_gpt2.linear(h, w[p + "mlp.c_proj.weight"], w[p + "mlp.c_proj.bias"])
    return plain_gpt2.lm_head(rounded(plain_gpt2.layernorm(x, w["ln_f.weight"], w["ln_f.bias"], eps)), w["wte.weight"]), made


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("steps", STEPS, ids=str)
def test_gpt2_steps(dtype, steps, tmp_path):
    config = dict(TINY_A)
    weights = plain_gpt2.random_weights(config, 3)
    if dtype == "bfloat16":
        weights = plain_gpt2.bf16_weights(weights)
    rounded = plain_gpt2.stored_as_bf16 if dtype == "bfloat16" else (lambda x: x)
    w = {name: t.astype(np.float64) for name, t in weights.items()}
    model, cache, runner = runner_for(config, weights, dtype, tmp_path)
    tokens = {name: random_tokens(i, 128, config["vocab_size"]) for i, name in enumerate("ab")}
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
            want, made = plain_gpt2_step(config, w, new, done[name], {i: held[i][name] for i in held}, rounded)
            for i, (k, v) in enumerate(made):
                for plane, exact in zip(held[i][name], (k, v)):
                    got = plane[done[name] :]
                    # half a code's step of the number (2^-4 of it), or half the smallest step (2^-10 scale, twice if the block has grown; scale is at most its
                    # largest / 224), and the number as it is made (32-bit, or two roundings of bfloat16: 2^-8 each)
                    largest = np.abs(plane).max()
                    assert np.all(np.abs(got - exact) <= (2.0**-4 + 2.0**-6) * np.abs(exact) + 2 * 2.0**-10 * largest / 224 + (2.0**-7 if dtype == "bfloat16" else 2.0**-18) * largest)
            off = np.abs(logits[row : row + len(new)] - want)
            scale = np.abs(want).max()
            # 32-bit: sums in another order than numpy's. bfloat16: the engine rounds where the plain run does, a half step either way
            assert off.max() <= (3e-4 if dtype == "float32" else 2e-2) * max(scale, 1.0), (name, off.max(), scale)
            row += len(new)
            done[name] += len(new)
        for name, new in entries:
            assert cache.length(name) == done[name]


def engine_for(config, seed, dtype, **options):
    from mini_llm_amd.config import config_from_dict
    from mini_llm_amd.engine.engine import Engine, EngineOptions

    return Engine.from_random(config_from_dict(config), seed, EngineOptions(dtype=dtype, **{"max_sessions": 8, "max_length": 120, "cache_dtype": "float8", **options}))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["gpt2", "dizizen", "gevulorn"])
def test_captured_steps_are_the_eager_ones(name, dtype):
    """Prompts, portions and decoding through the scheduler, replayed from graphs, ahead of the host and in lanes, against the same eagerly."""
    config = {"gpt2": TINY_A, "dizizen": DIZIZEN["mixed"], "gevulorn": GEVULORN["mixed"]}[name]
    vocab = config.get("vocab_size", config.get("vocab"))
    prompts = [random_tokens(20 + i, n, vocab) for i, n in enumerate((3, 17, 40, 64, 1))]
    with engine_for(config, 5, dtype, use_graphs=False, step_ahead=False) as engine:
        want = engine.generate(prompts, max_new_tokens=24)
    with engine_for(config, 5, dtype, portion_graph_after=1, page_size=16) as engine:
        assert engine.generate(prompts, max_new_tokens=24) == want
        assert engine.generate(prompts, max_new_tokens=24) == want   # captured by now, in pages that were used before


@pytest.mark.parametrize("case", [*(f"dizizen-{n}" for n in DIZIZEN), *(f"gevulorn-{n}" for n in GEVULORN)])
def test_designs_over_what_the_cache_holds(case, tmp_path, monkeypatch):
    """A prompt, whole, in 32 bits: the plain implementation with every attention's keys and values replaced by what the cache held."""
    design, _, which = case.partition("-")
    config = {"dizizen": DIZIZEN, "gevulorn": GEVULORN}[design][which]
    plain = {"dizizen": plain_dizizen, "gevulorn": plain_gevulorn}[design]
    weights = plain.random_weights(config, 31)
    model, cache, runner = runner_for(config, weights, "float32", tmp_path, max_length=160)
    tokens = random_tokens(8, 90, config["vocab"])
    cache.open("r")
    logits, held = step_and_held(model, cache, runner, [("r", tokens)])
    calls = iter(sorted(held))   # layer calls that attend, in order

    def held_now(k, v):
        index = next(calls)
        hk, hv = (t[:, : x.shape[1], : x.shape[2]] for t, x in zip(held[index]["r"], (k, v)))
        for got, exact in zip((hk, hv), (k, v)):
            largest = np.abs(exact).max()
            assert np.all(np.abs(got - exact) <= (2.0**-4 + 2.0**-6) * np.abs(exact) + (2.0**-10 / 224 + 2.0**-16) * largest), index
        return hk, hv

    if design == "dizizen":
        attend = plain.causal_attention
        monkeypatch.setattr(plain, "causal_attention", lambda q, k, v, scale: attend(q, *held_now(k, v), scale))
    else:
        attend = plain.sink_attention
        monkeypatch.setattr(plain, "sink_attention", lambda q, k, v, *rest: attend(q, *held_now(k, v), *rest))
    want = plain.forward(config, plain.as_float64(weights), tokens)
    assert next(calls, None) is None
    # sums in another order than numpy's (one position in a hundred may be up to five times off: a router whose two candidates lie within
    # rounding of each other picks the other one)
    off = (np.abs(logits - want) / (3e-4 + 2e-4 * np.abs(want))).max(axis=1)
    assert np.quantile(off, 0.99) <= 1.0 and off.max() <= 5.0, off.max()


def test_the_cache_takes_half_the_memory_and_reads_back_what_it_holds(tmp_path):
    from mini_llm_amd.engine.loading import cache_bytes_per_token

    with engine_for(TINY_A, 1, "bfloat16", cache_gib=0.01) as engine, engine_for(TINY_A, 1, "bfloat16", cache_gib=0.01, cache_dtype=None) as plain:
        groups = engine.model.cache_groups()
        assert cache_bytes_per_token(groups, 2, scaled=True) == 2 * 2 * 4 * (16 + 0.25) and cache_bytes_per_token(groups, 2) == 2 * 2 * 4 * 16 * 2
        assert engine.cache.pools[0].num_pages > 1.9 * plain.cache.pools[0].num_pages
        tokens = random_tokens(3, 50, 512)
        kept = []
        for e in (engine, plain):
            with e.open_session() as session:
                session.prefill(tokens)
                kept.append(e.cache.read_kv(session._handle, 0, 50))
        for got, exact in zip(*kept):
            exact = exact.double().cpu()
            e = exponent_for(torch.stack([b.abs().amax((0, 2)) for b in exact.split(16)]))          # [blocks, heads]
            want = torch.cat([coded(b.transpose(0, 1), e[i][:, None, None]).transpose(0, 1) * 2.0 ** e[i].double()[None, :, None] for i, b in enumerate(exact.split(16))])
            assert torch.equal(got.double().cpu(), want)


def test_command_line(tmp_path, capsys):
    from mini_llm_amd.cli.complete import main

    config = dict(TINY_A)
    (tmp_path / "config.json").write_text(json.dumps(config))
    plain_gpt2.write_safetensors(tmp_path / "model.safetensors", plain_gpt2.random_weights(config, 3))
    assert main(["--model", str(tmp_path), "--tokens", "5,17,3", "--max-new-tokens", "6", "--temperature", "0", "--cache-dtype", "float8"]) == 0
    assert len(capsys.readouterr().out.strip().split(",")) == 6


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["gpt2", "dizizen"])
def test_decoding_in_two_groups_side_by_side(name, dtype):
    """40 sequences whose captured step takes its requests through the layers in two groups on two streams, against one group."""
    config = {"gpt2": TINY_A, "dizizen": DIZIZEN["mixed"]}[name]
    prompts = [random_tokens(300 + i, 21, config.get("vocab_size", config.get("vocab"))) for i in range(40)]
    results = []
    for lanes in (None, 32):
        with engine_for(config, 5, dtype, max_sessions=40, page_size=16, decode_lanes_from=lanes) as engine:
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
