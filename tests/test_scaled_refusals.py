"""Pages of 8 bits: what the calls refuse, and the bookkeeping that needs no GPU."""

import pytest
import torch

from mini_llm_amd.ops import kernels as K


def codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_shapes_of_pages():
    k, v = K.scaled_pages(3, 2, 64, 48, "cpu")
    assert k.shape == v.shape == (3, 2, 64, 48) and k.is_keys and not v.is_keys
    assert k.codes.shape == (3, 2, 4, 3, 16, 16) and v.codes.shape == (3, 2, 4, 48, 16) and k.scales.shape == (3, 2, 4)
    assert k.dtype == torch.float8_e4m3fn and bool((v.scales == 1).all())


@pytest.mark.parametrize("args", [(0, 1, 16, 16), (1, 0, 16, 16), (1, 1, 8, 16), (1, 1, 48, 16), (1, 1, 16, 24), (1, 1, 16, 0), (1, 1, 16, 272)])
def test_pages_that_cannot_be(args):
    with pytest.raises(K.OperandError):
        K.scaled_pages(*args, "cpu")


@pytest.mark.parametrize("make", [
    lambda: (torch.zeros((1, 1, 1, 1, 16, 16)), torch.ones((1, 1, 1))),
    lambda: (codes(1, 1, 1, 1, 16, 16), torch.ones((1, 1, 1), dtype=torch.float64)),
    lambda: (codes(1, 1, 1, 1, 16, 16), torch.ones((1, 1, 2))),
    lambda: (codes(1, 1, 1, 16), torch.ones((1, 1, 1))),
    lambda: (codes(1, 1, 1, 16, 8), torch.ones((1, 1, 1))),
    lambda: (codes(1, 1, 3, 16, 16), torch.ones((1, 1, 3))),
    lambda: (codes(1, 1, 1, 24, 16), torch.ones((1, 1, 1))),
    lambda: (codes(1, 2, 3, 16, 16).transpose(1, 2), torch.ones((1, 3, 2))),
    lambda: ("codes", torch.ones((1, 1, 1)))])
def test_codes_and_scales_that_do_not_fit(make):
    with pytest.raises(K.OperandError):
        K.ScaledPages(*make())


def test_the_cpu_is_refused():
    k, v = K.scaled_pages(1, 1, 16, 16, "cpu")
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(K.OperandError, match="GPU"):
        K.scaled_append(torch.zeros((1, 48)), 0, 16, 32, k, v, ints, ints, 1, 1, 16, 16)
    with pytest.raises(K.OperandError, match="GPU"):
        K.paged_attention(torch.zeros((1, 16)), k, v, ints, ints, ints[None], 1, 1, 16, 0.25)
    with pytest.raises(K.OperandError, match="GPU"):
        K.scaled_rows(k, v, ints)


def test_planes_in_the_wrong_place_are_refused():
    k, v = K.scaled_pages(1, 1, 16, 16, "cpu")
    plain = torch.zeros((1, 1, 16, 16))
    ints = torch.zeros(1, dtype=torch.int32)
    for pair in ((v, k), (k, k), (k, plain)):
        with pytest.raises(K.OperandError):
            K.paged_attention(torch.zeros((1, 16)), *pair, ints, ints, ints[None], 1, 1, 16, 0.25)
        with pytest.raises(K.OperandError):
            K.scaled_append(torch.zeros((1, 48)), 0, 16, 32, *pair, ints, ints, 1, 1, 16, 16)
    with pytest.raises(K.OperandError):
        K.scaled_rows(k, K.scaled_pages(2, 1, 16, 16, "cpu")[1], ints)


@pytest.mark.parametrize("blocks", [1, 12, 100, 1000, 100000])
@pytest.mark.parametrize("tiles", [1, 2, 16, 17, 500, 16384])
@pytest.mark.parametrize("head_size,columns", [(16, 1), (64, 16), (128, 4), (128, 16), (256, 1), (256, 16)])
def test_cuts_fit_what_the_kernel_takes(blocks, tiles, head_size, columns):
    waves, run, runs = K.scaled_cut(blocks, tiles, head_size, columns)
    assert K.scaled_cut(blocks, tiles, head_size, columns, True)[0] <= (8 if head_size <= 128 else 4)
    assert 1 <= waves <= 16 and waves & (waves - 1) == 0 and waves * columns * (head_size + 4) * 4 <= 65536
    assert run >= 1 and run * runs >= tiles and run * (runs - 1) < tiles and 1 <= runs <= 65535


def test_models_whose_mixers_keep_other_rows_are_refused():
    from conftest import TINY_A, TINY_D
    from gimozen_cases import CASES as GIMOZEN
    from ketolix_cases import CASES as KETOLIX
    from mini_llm_amd.config import config_from_dict
    from mini_llm_amd.engine.loading import build_model, scaled_cache

    assert scaled_cache(build_model(config_from_dict(TINY_A), "bfloat16"), "float8")
    assert not scaled_cache(build_model(config_from_dict(TINY_A), "bfloat16"), None)
    for config in (*GIMOZEN.values(), *KETOLIX.values()):
        with pytest.raises(ValueError, match="8 bits"):
            scaled_cache(build_model(config_from_dict(config), "bfloat16"), "float8")
    with pytest.raises(ValueError, match="unknown cache type"):
        scaled_cache(build_model(config_from_dict(TINY_A), "bfloat16"), "int4")


@pytest.mark.parametrize("head_size,page_size,planes", [(14, 64, 2), (272, 64, 2), (16, 8, 2), (64, 64, 1)])
def test_groups_that_a_cache_of_8_bits_does_not_hold(head_size, page_size, planes):
    from mini_llm_amd.cache import CacheManager
    from mini_llm_amd.models.base import CacheGroupSpec

    with pytest.raises(ValueError, match="8 bits"):
        CacheManager([CacheGroupSpec("g", (0,), 2, head_size, None, planes)], {}, num_pages=4, page_size=page_size, max_requests=2, scaled=True)


def test_bookkeeping_of_a_cache_of_8_bits():
    from mini_llm_amd.cache import CacheManager
    from mini_llm_amd.models.base import CacheGroupSpec

    cache = CacheManager([CacheGroupSpec("g", (0, 1), 2, 32, None)], {}, num_pages=4, page_size=16, max_requests=2, device="cpu", max_length=64, scaled=True)
    assert cache.k_pages[0].is_keys and not cache.v_pages[1].is_keys and cache.k_pages[1].shape == (4, 2, 16, 32)


def test_plain_key_pages_beside_value_pages_of_8_bits_are_refused():
    _, v = K.scaled_pages(1, 1, 16, 16, "cpu")
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(K.OperandError, match="8 bits"):
        K.paged_attention(torch.zeros((1, 16)), torch.zeros((1, 1, 16, 16)), v, ints, ints, ints[None], 1, 1, 16, 0.25)


@pytest.mark.parametrize("rows,requests,longest,heads,size,wide,one", [
    (64, 1, 64, 12, 64, False, True), (2048, 1, 2048, 12, 64, False, True), (8192, 1, 8192, 12, 64, False, False),
    (2048, 1, 2048, 32, 128, False, False), (512, 4, 128, 8, 256, False, False), (64, 1, 64, 12, 64, True, True)])
def test_steps_of_both_kinds_go_in_one_launch_where_the_portions_are_few(rows, requests, longest, heads, size, wide, one):
    assert K.scaled_mixes(12, rows, requests, longest, heads, size, wide) == one
    assert not K.scaled_mixes(100000, rows, requests, longest, heads, size, wide)
