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
