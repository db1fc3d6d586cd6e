"""The expert block of a few tokens against a 64-bit reference."""
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


def make(g, T, E, hidden, inter, code, dt=torch.bfloat16):
    def codes(*shape):
        x = torch.randn(*shape, generator=g)
        return (32 * x).round().clamp(-127, 127).to(I8) if code == I8 else (100 * x).clamp(-448, 448).to(E4M3)

    unit = 1 / 32 if code == I8 else 1 / 100
    a, sa = codes(T, hidden), unit * (0.5 + torch.rand(T, generator=g))
    w13, s13 = codes(E, 2 * inter, hidden), unit * hidden ** -0.5 * (0.5 + torch.rand(E, 2 * inter, generator=g))
    w2, s2 = codes(E, hidden, inter), unit * inter ** -0.5 * (0.5 + torch.rand(E, hidden, generator=g))
    return a, sa, torch.randn(T, E, generator=g).to(dt), w13, s13, w2, s2


def check(dev, args, top, renormalize=True, out_dtype=torch.float32, ref=None):
    d = [t.to(dev) for t in args]
    got = K().moe_few_tokens(*d, top, renormalize=renormalize, out_dtype=out_dtype)
    want, slack = ref or R.moe(*args, top, renormalize)
    off = (got.cpu().double() - want).abs()
    bound = R.rounding(want, out_dtype) + slack * (1 + R.HALF[out_dtype])
    assert (off <= bound).all(), float((off / bound).max())
    return got


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 33, 64])
@pytest.mark.parametrize("E,top,hidden,inter", [(4, 2, 64, 32), (1, 1, 16, 16), (9, 9, 144, 48), (64, 4, 128, 16), (70, 16, 32, 80),
                                                (3, 1, 272, 528), (2, 2, 1296, 144)])
def test_sizes(dev, code, T, E, top, hidden, inter):
    args = make(gen(T + E), T, E, hidden, inter, code)
    ref = R.moe(*args, top, True)
    check(dev, args, top, ref=ref)
    check(dev, args, top, out_dtype=torch.bfloat16, ref=ref)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("T,E,top,hidden,inter", [(1, 8, 2, 4096, 512), (3, 4, 2, 4112, 1040), (20, 300, 8, 256, 64), (8, 512, 4, 64, 32), (1, 6, 2, 512, 6160),
                                                  (2, 3, 2, 5120, 48)])
def test_larger(dev, code, T, E, top, hidden, inter):
    args = make(gen(T + E), T, E, hidden, inter, code, torch.float32)
    check(dev, args, top, out_dtype=torch.float16)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("T,E,top,hidden,inter", [
    (13, 32, 8, 528, 1040),   # waves with units of their own, rows that share lines, blocks that share outputs
    (9, 40, 2, 1024, 2048),   # the same with whole lines
    (33, 8, 4, 512, 1024),    # groups of 32, more than one an expert
    (64, 4, 2, 272, 1040),    # groups of 64
    (40, 3, 2, 640, 512),     # and blocks that share outputs
    (8, 4, 2, 4096, 128),     # four steps on their way
    (20, 64, 2, 4096, 16),    # the same behind a routing launch
    (17, 6, 2, 4112, 32),     # more blocks than units
    (2, 20, 8, 256, 1024),    # as many positions as the down kernel makes codes for
    (3, 20, 6, 256, 896),     # and more
    (1, 16, 16, 1008, 1008),
    (64, 200, 16, 48, 32),
    (20, 4, 2, 272, 2048),    # groups of 32, two products a unit
    (20, 8, 4, 144, 4096),    # the same, waves with units of their own
    (48, 2, 2, 272, 4096),    # groups of 64
])
def test_each_way_of_cutting(dev, code, T, E, top, hidden, inter):
    args = make(gen(T + E + hidden), T, E, hidden, inter, code, torch.float32)
    ref = R.moe(*args, top, True)
    first = check(dev, args, top, out_dtype=torch.float32, ref=ref)
    for _ in range(3):
        assert torch.equal(check(dev, args, top, out_dtype=torch.float32, ref=ref), first)


def test_two_products_a_unit_for_groups_of_16(dev):
    check(dev, make(gen(64), 64, 64, 2064, 512, E4M3), 5)


@pytest.mark.parametrize("hidden,inter", [(131056, 16), (16, 131056)])
def test_the_largest_sums_of_codes(dev, hidden, inter):
    """All codes the lowest: sums just below 2^31 (down: codes of h, all 127, times the lowest)."""
    a, w13, w2 = (torch.full(s, -128, dtype=I8) for s in ((2, hidden), (1, 2 * inter, hidden), (1, hidden, inter)))
    s13, s2 = torch.full((1, 2 * inter), 2.0 ** -30), torch.full((1, hidden), 2.0 ** -24)
    check(dev, (a, torch.ones(2), torch.zeros(2, 1), w13, s13, w2, s2), 1)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("renormalize", [True, False])
def test_types_of_logits_and_shares(dev, dt, renormalize):
    args = make(gen(2), 7, 12, 64, 48, I8, dt)
    check(dev, args, 3, renormalize)
    check(dev, args, 12, renormalize)


def test_equal_logits_go_to_the_lowest(dev):
    a, sa, l, *w = make(gen(4), 6, 130, 32, 16, I8, torch.float32)
    l.zero_()
    l[1, 100:] = 1.0
    l[2, ::7] = -1.0
    l[3, 64] = l[3, 63] = 2.0
    l[4], l[5] = -0.0, 0.0
    l[5, 3] = -0.0  # (the zeros are one number)
    ids, _ = R.route(l, 5, True)
    assert ids[0] == [0, 1, 2, 3, 4] and ids[1] == [100, 101, 102, 103, 104] and ids[3][:2] == [63, 64] and ids[5] == [0, 1, 2, 3, 4]
    check(dev, (a, sa, l, *w), 5)


def test_masked_experts(dev):
    """Experts with a logit of -infinity are not run; a token whose logits all are gets zero.  A type's lowest value is a number like others."""
    a, sa, l, *w = make(gen(5), 5, 8, 64, 32, E4M3, torch.float32)
    l[0, 1:] = float("-inf")
    l[1] = float("-inf")
    l[2, :7] = torch.finfo(torch.float32).min
    l[3] = torch.finfo(torch.float32).min
    w[2].view(torch.uint8)[l.shape[1] - 1] = w[2].view(torch.uint8)[0]
    got = check(dev, (a, sa, l, *w), 3)
    assert not got[1].any()
    # weights of no number in an expert that nobody runs change nothing
    l[:, 4] = float("-inf")
    clean = check(dev, (a, sa, l, *w), 3)
    for i in (0, 2):
        w[i].view(torch.uint8)[4] = 0x7f
    w[1][4], w[3][4] = float("nan"), float("inf")
    d = [t.to(dev) for t in (a, sa, l, *w)]
    assert torch.equal(K().moe_few_tokens(*d, 3, out_dtype=torch.float32), clean)


def test_no_numbers_stay_with_their_token(dev):
    a, sa, l, *w = make(gen(6), 4, 6, 64, 32, I8, torch.float32)
    clean = check(dev, (a, sa, l, *w), 2)
    for edit in (lambda: l[2].fill_(float("nan")), lambda: sa[2:3].fill_(float("nan"))):
        l0, s0 = l.clone(), sa.clone()
        edit()
        got = K().moe_few_tokens(*[t.to(dev) for t in (a, sa, l, *w)], 2, out_dtype=torch.float32)
        assert got[2].isnan().all() and torch.equal(got[[0, 1, 3]], clean[[0, 1, 3]])
        l.copy_(l0), sa.copy_(s0)


def test_silu_far_from_zero(dev):
    a, sa, l, *w = make(gen(7), 3, 4, 64, 48, I8, torch.float32)
    w[1] *= 60  # gates of about +-60
    check(dev, (a, sa, l, *w), 2)
    w[1] *= 1e-8  # h below the floor of the scale
    check(dev, (a, sa, l, *w), 2)


def test_one_scale_strided_rows_and_out(dev):
    a, sa, l, *w = make(gen(8), 6, 5, 128, 48, I8)
    sa = sa[:1]
    want = check(dev, (a, sa, l, *w), 2, out_dtype=torch.bfloat16)
    wide, lw, room = torch.zeros(6, 400, dtype=I8, device=dev), torch.zeros(6, 9, device=dev).bfloat16(), torch.full((8, 144), 3.0, device=dev).bfloat16()
    wide[:, 16:144], lw[:, 2:7] = a.to(dev), l.to(dev)
    d = [t.to(dev) for t in w]
    out = K().moe_few_tokens(wide[:, 16:144], sa.to(dev), lw[:, 2:7], *d, 2, out=room[1:7, 8:136])
    assert torch.equal(out, want) and (room[0] == 3).all() and (room[7] == 3).all() and (room[:, :8] == 3).all() and (room[:, 136:] == 3).all()
    assert torch.equal(K().moe_few_tokens(a.to(dev), float(sa), l.to(dev), *d, 2), want)


@pytest.mark.parametrize("code", [I8, E4M3])
def test_one_expert_takes_every_token(dev, code):
    a, sa, l, *w = make(gen(9), 64, 7, 160, 64, code)
    l[:, 3] = 20.0
    check(dev, (a, sa, l, *w), 1)
    check(dev, (a, sa, l, *w), 2)


def test_against_the_grouped_product(dev):
    """The gate and up products are those of grouped_gemm_i8_dq, bit for bit before the rounding: the whole against a chain of calls."""
    k = K()
    a, sa, l, w13, s13, w2, s2 = (t.to(dev) for t in make(gen(10), 24, 6, 256, 128, I8, torch.float32))
    p, ids = torch.topk(l.softmax(-1), 2)
    p = p / p.sum(-1, keepdim=True)
    order = ids.reshape(-1).argsort(stable=True)
    counts = torch.bincount(ids.reshape(-1), minlength=6)
    off = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    rows = order // 2
    up = k.grouped_gemm_i8_dq(a[rows], w13, off, sa[rows], s13, out_dtype=torch.float32, exact_ref=False)
    h = up[:, :128] / (1 + torch.exp(-up[:, :128])) * up[:, 128:]
    q, s = k.quant_act_i8_pertoken(h)
    down = k.grouped_gemm_i8_dq(q, w2, off, s, s2, out_dtype=torch.float32, exact_ref=False)
    y = torch.zeros(24, 256, device=dev).index_add_(0, rows, down * p.reshape(-1)[order][:, None])
    got = k.moe_few_tokens(a, sa, l, w13, s13, w2, s2, 2, out_dtype=torch.float32)
    assert ((got - y).norm() / y.norm()) < 2e-4  # (single codes at a border)


def test_no_tokens(dev):
    args = [t.to(dev) for t in make(gen(1), 1, 4, 32, 16, I8)]
    args[0], args[1], args[2] = args[0][:0], args[1][:0], args[2][:0]
    assert K().moe_few_tokens(*args, 2).shape == (0, 32)


def test_refusals(dev):
    k = K()
    a, sa, l, w13, s13, w2, s2 = (t.to(dev) for t in make(gen(1), 2, 4, 32, 16, I8))
    for bad, kind in [
        (lambda: k.moe_few_tokens(a.repeat(33, 1), sa.repeat(33), l.repeat(33, 1), w13, s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13, w2, s2, 0), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13, w2, s2, 5), ValueError),
        (lambda: k.moe_few_tokens(a.half(), sa, l, w13, s13, w2, s2, 2), TypeError),
        (lambda: k.moe_few_tokens(a, sa, l, w13.view(E4M3), s13, w2, s2, 2), TypeError),
        (lambda: k.moe_few_tokens(a, sa, l[:1], w13, s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l[:, :3], w13, s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l.int(), w13, s13, w2, s2, 2), TypeError),
        (lambda: k.moe_few_tokens(a, sa, l, w13[:, :, :16], s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13.transpose(1, 2).contiguous().transpose(1, 2), s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13[:, :16], w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13.half(), w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa.repeat(2), l, w13, s13, w2, s2, 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13, w2, s2, 2, out_dtype=torch.int8), TypeError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13, w2, s2, 2, out=torch.empty(2, 16, device=dev)), ValueError),
        (lambda: k.moe_few_tokens(a[:, :24].contiguous(), sa, l, w13[:, :, :24].contiguous(), s13, w2[:, :24].contiguous(), s2[:, :24].contiguous(), 2), ValueError),
        (lambda: k.moe_few_tokens(a, sa, l, w13, s13, w2.cpu(), s2, 2), RuntimeError),
    ]:
        with pytest.raises(kind):
            bad()
