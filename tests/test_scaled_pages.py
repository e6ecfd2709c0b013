"""What pages of 8 bits are made of, and stay."""

import pytest
import torch

from mini_llm_amd.ops import kernels as K


@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("which", ["codes", "scales"])
@pytest.mark.parametrize("how", ["data", "set"])
def test_pages_whose_tensors_have_other_memory_are_refused(keys, which, how):
    k, v = K.scaled_pages(3, 2, 64, 16, "cpu")
    pages, ints = k if keys else v, torch.zeros(1, dtype=torch.int32)
    with pytest.raises(K.OperandError, match="GPU"):
        K.scaled_rows(k, v, ints)
    tensor = pages.codes if which == "codes" else pages.scales
    other = tensor[:1].clone()
    if how == "data":
        tensor.data = other
    else:
        tensor.set_(other)
    for call in (lambda: K.scaled_rows(k, v, ints), lambda: K.scaled_append(torch.zeros((1, 96)), 0, 32, 64, k, v, ints, ints, 2, 2, 16, 16),
                 lambda: K.paged_attention(torch.zeros((1, 32)), k, v, ints, ints, ints[None], 2, 2, 16, 0.25)):
        with pytest.raises(K.OperandError, match="other memory"):
            call()


@pytest.mark.gpu
def test_calls_over_pages_whose_tensors_have_other_memory_are_refused():
    k, v = K.scaled_pages(4, 1, 16, 16, "cuda:0")
    ints = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    rows = torch.ones((1, 48), device="cuda:0")
    K.scaled_append(rows, 0, 16, 32, k, v, ints, ints, 1, 1, 16, 16)
    v.codes.data = v.codes[:1].clone()
    for call in (lambda: K.scaled_append(rows, 0, 16, 32, k, v, ints, ints, 1, 1, 16, 16), lambda: K.scaled_rows(k, v, ints),
                 lambda: K.paged_attention(rows[:, :16], k, v, ints, ints, ints[None], 1, 1, 16, 0.25)):
        with pytest.raises(K.OperandError, match="other memory"):
            call()


def test_a_rotation_without_frequencies_is_refused():
    assert K._rotation(None, 0, 64, "half", "values", 0) == (None, 0)
    with pytest.raises(K.OperandError, match="frequencies of values"):
        K._rotation(None, 16, 64, "half", "values", 0)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rot_dims", "v_rot_dims"])
def test_calls_with_a_rotation_without_frequencies_are_refused(name):
    pages = K.scaled_pages(1, 1, 16, 16, "cuda:0")
    ints = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    with pytest.raises(K.OperandError, match="frequencies"):
        K.scaled_append(torch.ones((1, 48), device="cuda:0"), 0, 16, 32, *pages, ints, ints, 1, 1, 16, 16, **{name: 16})
    assert not bool(pages[0].codes.view(torch.uint8).any())
