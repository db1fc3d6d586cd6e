"""Calls of the operators around a layer's products at the ends of what they take."""
import pytest
import torch

import layer_reference as R

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


@pytest.mark.parametrize("code", [I8, E4M3])
def test_more_tokens_than_the_expert_block_takes(dev, code):
    """The refusal names calls that take these codes; 64 tokens at a time are one of them."""
    g = torch.Generator().manual_seed(3)
    T, E, hidden, inter = 150, 5, 64, 32
    codes = [torch.randint(-100, 100, s, generator=g).to(I8).to(dev) for s in ((T, hidden), (E, 2 * inter, hidden), (E, hidden, inter))]
    if code == E4M3:
        codes = [c.float().to(E4M3) for c in codes]
    a, w13, w2 = codes
    sa, s13, s2 = (torch.rand(s, generator=g).to(dev) * 0.01 for s in ((T,), (E, 2 * inter), (E, hidden)))
    l = torch.randn(T, E, generator=g).to(dev)

    def call(t):
        return K().moe_few_tokens(a[t], sa[t], l[t], w13, s13, w2, s2, 2, out_dtype=torch.float32)

    with pytest.raises(ValueError, match="64 at a time") as refusal:
        call(slice(0, T))
    assert ("grouped_gemm_i8_dq" in str(refusal.value)) == (code == I8)
    got = torch.cat([call(slice(i, i + 64)) for i in range(0, T, 64)])
    want, slack = R.moe(*(t.cpu() for t in (a, sa, l, w13, s13, w2, s2)), 2)
    assert ((got.cpu().double() - want).abs() <= R.rounding(want, torch.float32) + slack * (1 + R.HALF[torch.float32])).all()
