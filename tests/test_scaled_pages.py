"""What pages of 8 bits are made of, and stay."""

import gc

import pytest
import torch

from mini_llm_amd.ops import kernels as K


@pytest.mark.parametrize("keys", [True, False])
def test_pages_keep_their_memory_when_the_callers_tensors_become_others(keys):
    codes = torch.zeros((3, 2, 4, 1, 16, 16) if keys else (3, 2, 4, 16, 16), dtype=torch.uint8).view(K.E4M3)
    scales = torch.ones((3, 2, 4))
    pages, at = K.ScaledPages(codes, scales), (codes.data_ptr(), scales.data_ptr())
    scales[1, 0, 2] = 4.0
    assert pages.scales[1, 0, 2] == 4.0
    codes.data = torch.ones((1, 1), dtype=torch.uint8).view(K.E4M3)
    scales.set_(torch.zeros(2))
    del codes, scales
    gc.collect()
    assert pages.addresses == at == (pages.codes.data_ptr(), pages.scales.data_ptr())
    assert pages.codes.numel() == 3 * 2 * 64 * 16 and pages.scales.shape == (3, 2, 4) and pages.scales[1, 0, 2] == 4.0 and not bool(pages.codes.view(torch.uint8).any())


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
