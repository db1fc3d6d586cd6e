"""Residual addition, RMS norm and 8-bit codes against a 64-bit reference."""
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu
I8, E4M3 = torch.int8, torch.float8_e4m3fn


def K():
    from fms_mo_amd import kernels

    return kernels


def gen(seed):
    return torch.Generator().manual_seed(seed)


def check(x, w, res, got, code, eps, scale=None):
    q, s, h, n = (None if t is None else t.cpu() for t in got)
    eh, en = R.norm(x, w, res, eps)
    slack = (R.NORM_ERROR + 2.0 ** -24) * en.abs() + torch.finfo(torch.float32).tiny
    if res is not None:
        assert ((h.double() - eh).abs() <= R.rounding(eh, x.dtype) + 2.0 ** -23 * eh.abs()).all()
    if n is not None:
        assert ((n.double() - en).abs() <= R.rounding(en, x.dtype) + 2 * slack).all()
    if scale is None:
        es = en.abs().amax(-1).clamp(min=R.FLOOR[code]) / R.MOST[code]
        assert ((s.double() - es).abs() <= es * (R.NORM_ERROR + 4 * 2.0 ** -24)).all()
    else:
        assert s.numel() == 1
    by = s.double().reshape(-1, 1)
    v = (en / by).clamp(-R.MOST[code], R.MOST[code])
    off = (q.double() if code == I8 else q.float().double()) - v
    bound = R.code_half_step(v, code) + 2 * slack / by + 2.0 ** -22 * v.abs()
    assert (off.abs() <= bound * (1 + 2.0 ** -10)).all(), float((off.abs() / bound).max())


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("T,cols", [(1030, 264), (1100, 4096), (1025, 5120), (1024, 9000), (1, 8), (1, 4096), (3, 64), (5, 72), (7, 512), (4, 520), (9, 1024), (2, 1032), (6, 2048), (33, 4096), (3, 4104),
                                    (2, 8192), (3, 12800), (1, 16384), (2, 16392), (1, 40000)])
def test_rows(dev, dt, code, T, cols):
    g = gen(T * cols)
    x, res = torch.randn(T, cols, generator=g).to(dt), (3 * torch.randn(T, cols, generator=g)).to(dt)
    for w in (1 + 0.2 * torch.randn(cols, generator=g)).to(dt), torch.randn(cols, generator=g):
        got = K().add_rms_norm_quant(x.to(dev), w.to(dev), res.to(dev), eps=1e-5, dtype=code, want_normed=True)
        check(x, w, res, got, code, 1e-5)
        got = K().add_rms_norm_quant(x.to(dev), w.to(dev), dtype=code)
        assert got[2] is None and got[3] is None
        check(x, w, None, got, code, 1e-6)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("cols", [256, 4096, 20000])
def test_given_scale(dev, code, cols):
    g = gen(5)
    x, res, w = torch.randn(6, cols, generator=g).half(), torch.randn(6, cols, generator=g).half(), torch.randn(cols, generator=g).half()
    for value in (0.02, 0.005, 30.0):
        s = torch.tensor([value], device=dev)
        got = K().add_rms_norm_quant(x.to(dev), w.to(dev), res.to(dev), dtype=code, scale=s, want_normed=True)
        assert got[1].data_ptr() == s.data_ptr()
        check(x, w, res, got, code, 1e-6, s)
    got = K().add_rms_norm_quant(x.to(dev), w.to(dev), res.to(dev), dtype=code, scale=0.02)
    check(x, w, res, got, code, 1e-6, 0.02)


@pytest.mark.parametrize("cols", [512, 4096, 16392])
def test_in_place_and_strided_rows(dev, cols):
    g = gen(2)
    wide = torch.randn(5, 2 * cols + 8, generator=g).bfloat16()
    res, w = torch.randn(5, cols, generator=g).bfloat16(), torch.ones(cols).bfloat16()
    x = wide[:, cols:2 * cols]
    want = K().add_rms_norm_quant(x.to(dev).contiguous(), w.to(dev), res.to(dev))
    for mine in (True, False):
        d, r = wide.to(dev), res.to(dev)
        xs = d[:, cols:2 * cols]
        to = r if mine else xs
        got = K().add_rms_norm_quant(xs, w.to(dev), r, residual_out=to)
        assert got[2].data_ptr() == to.data_ptr()
        for i in range(3):
            assert torch.equal(got[i], want[i])
        assert torch.equal(d[:, :cols].cpu(), wide[:, :cols]) and torch.equal(d[:, 2 * cols:].cpu(), wide[:, 2 * cols:])
    # an address that is no multiple of 16 is copied, not refused
    odd = torch.empty(5 * cols + 4, dtype=torch.bfloat16, device=dev)[4:].view(5, cols).copy_(x.to(dev))
    for a, b in zip(K().add_rms_norm_quant(odd, w.to(dev), res.to(dev)), want):
        assert a is None and b is None or torch.equal(a, b)


def test_rows_of_zeros_and_of_no_numbers(dev):
    x = torch.zeros(4, 256).bfloat16()
    x[1, 3], x[2, 7], x[3] = float("inf"), float("nan"), 2.0
    w = torch.ones(256).bfloat16()
    for code in (I8, E4M3):
        q, s, _, n = K().add_rms_norm_quant(x.to(dev), w.to(dev), dtype=code, want_normed=True)
        assert not q[0].float().any() and s[0].item() == pytest.approx(R.FLOOR[code] / R.MOST[code]) and not n[0].any()
        assert s[1].isnan() and s[2].isnan() and n[2].isnan().all()
        check(x[3:], w, None, (q[3:], s[3:], None, n[3:]), code, 1e-6)
        if code == E4M3:
            assert q[1].float().isnan().all() and q[2].float().isnan().all()
    # rows whose squares leave fp32 are rows of zeros, as they are where every step is fp32
    q, s, _, _ = K().add_rms_norm_quant(torch.full((1, 64), 1e30).bfloat16().to(dev), torch.ones(64).bfloat16().to(dev))
    assert not q.any()


def test_codes_of_the_quantizer(dev):
    """The codes are those that the per-token e4m3 quantizer makes of an fp32 norm."""
    g = gen(9)
    x, w = torch.randn(40, 4096, generator=g).bfloat16().to(dev), torch.randn(4096, generator=g).to(dev)
    q, s, _, _ = K().add_rms_norm_quant(x, w, dtype=E4M3)
    n = x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6) * w
    q2, s2 = K().quant_act_fp8_pertoken(n)
    assert torch.allclose(s, s2, rtol=2e-6, atol=0)
    assert (q.view(torch.uint8) != q2.view(torch.uint8)).float().mean() < 1e-3


def test_no_rows(dev):
    q, s, h, n = K().add_rms_norm_quant(torch.empty(0, 64, device=dev).half(), torch.ones(64, device=dev).half(),
                                        torch.empty(0, 64, device=dev).half(), want_normed=True)
    assert q.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64) and n.shape == (0, 64)


def test_refusals(dev):
    k = K()
    x, w = torch.zeros(2, 64, device=dev).half(), torch.ones(64, device=dev).half()
    for bad, kind in [
        (lambda: k.add_rms_norm_quant(x.float(), w.float()), TypeError),
        (lambda: k.add_rms_norm_quant(x, w.bfloat16()), ValueError),
        (lambda: k.add_rms_norm_quant(x, w[:32]), ValueError),
        (lambda: k.add_rms_norm_quant(x[0], w), ValueError),
        (lambda: k.add_rms_norm_quant(x[:, :60], w[:60]), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, x[:1]), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, x.bfloat16()), TypeError),
        (lambda: k.add_rms_norm_quant(x, w, dtype=torch.float16), TypeError),
        (lambda: k.add_rms_norm_quant(x, w, residual_out=x), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, x, residual_out=x[:1]), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, x, residual_out=x.t().contiguous().t()), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, scale=torch.ones(2, device=dev)), ValueError),
        (lambda: k.add_rms_norm_quant(x, w, scale=torch.ones(1, device=dev).half()), ValueError),
        (lambda: k.add_rms_norm_quant(x, w.cpu()), RuntimeError),
        (lambda: k.add_rms_norm_quant(x.cpu(), w.cpu()), RuntimeError),
    ]:
        with pytest.raises(kind):
            bad()
