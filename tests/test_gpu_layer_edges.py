"""Calls of the operators around a layer's products at the ends of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def K():
    from fms_mo_amd import kernels

    return kernels


@pytest.mark.parametrize("code", [I8, E4M3])
def test_tokens_of_no_elements_have_a_scale(dev, code):
    """The scale of rows of zeros, not what the memory held before."""
    held = [torch.full((4096,), 7.0, device=dev) for _ in range(64)]  # (memory that the results may be made in)
    del held
    zeros = K().add_rms_norm_quant(torch.zeros(3, 64, device=dev).half(), torch.ones(64, device=dev).half(), dtype=code)[1]
    x, w = torch.empty(3, 0, device=dev).half(), torch.empty(0, device=dev).half()
    for res in (None, x):
        q, s, h, n = K().add_rms_norm_quant(x, w, res, dtype=code, want_normed=True)
        assert q.shape == (3, 0) and n.shape == (3, 0) and (h is None) == (res is None)
        assert torch.equal(s, zeros)
