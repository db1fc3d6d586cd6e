"""Calls of the operators around a layer's products at the ends of what they take."""
import pytest
import torch

import layer_reference as R
import test_gpu_lora as lora
from test_gpu_moe_few import check, gen, make

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


def test_rows_of_several_launches(dev):
    """2^26 rows and more, which no launch has threads for: the results of calls on pieces of them."""
    T, some = (1 << 26) + 5, 1 << 20
    g = torch.Generator(dev).manual_seed(5)
    x, w = torch.empty(T, 8, device=dev, dtype=torch.bfloat16).normal_(generator=g), torch.randn(8, device=dev).bfloat16()
    q, s, _, _ = K().add_rms_norm_quant(x, w, dtype=I8)
    q2, s2, _, _ = K().add_rms_norm_quant(x, w, dtype=E4M3, scale=0.01)
    for i in range(0, T, some):
        t = slice(i, min(i + some, T))
        a, b, _, _ = K().add_rms_norm_quant(x[t], w, dtype=I8)
        assert torch.equal(q[t], a) and torch.equal(s[t], b)
        assert torch.equal(q2[t].view(torch.uint8), K().add_rms_norm_quant(x[t], w, dtype=E4M3, scale=s2)[0].view(torch.uint8))


def test_residuals_of_several_launches(dev):
    """Rows on both sides of what one launch takes, with everything that a call can write, in place and apart."""
    T, some = (1 << 22) + 3, (1 << 21) - 7
    g = torch.Generator(dev).manual_seed(6)
    x, r = (torch.empty(T, 16, device=dev, dtype=torch.float16).normal_(generator=g) for _ in range(2))
    w = torch.randn(16, device=dev)
    got = K().add_rms_norm_quant(x, w, r, dtype=E4M3, want_normed=True)
    for i in range(0, T, some):
        t = slice(i, min(i + some, T))
        for a, b in zip(got, K().add_rms_norm_quant(x[t], w, r[t], dtype=E4M3, want_normed=True)):
            assert torch.equal(a[t].view(torch.uint8), b.view(torch.uint8))
    h = K().add_rms_norm_quant(x, w, r, dtype=E4M3, residual_out=r)
    assert h[2] is r and torch.equal(r, got[2]) and torch.equal(h[1], got[1])


@pytest.mark.parametrize("rank,T", [(128, 20001), (64, 40000)])
def test_one_row_requests_of_several_launches(dev, rank, T):
    g = torch.Generator().manual_seed(rank)
    x, y = torch.randn(T, 64, generator=g).bfloat16(), torch.randn(T, 64, generator=g).bfloat16()
    a, b = (0.125 * torch.randn(5, rank, 64, generator=g)).bfloat16(), torch.randn(5, 64, rank, generator=g).bfloat16()
    ids, scales = torch.randint(-1, 6, (T,), generator=g), 0.5 + torch.rand(5, generator=g)
    args = [t.to(dev) for t in (y, x, a, b, ids.to(torch.int32))]
    got = K().lora_add(*args, scales=scales.to(dev))
    # the rows of each adapter as one request of the reference
    order = ids.argsort(stable=True)
    start = [0] + torch.bincount(ids + 1, minlength=7).cumsum(0).tolist()
    want, slack = R.lora(y[order], x[order], a, b, list(range(-1, 6)), start, scales)
    bound = R.rounding(want, y.dtype) + slack * (1 + R.HALF[y.dtype]) + 2.0 ** -24 * want.abs()
    assert ((got.cpu()[order].double() - want).abs() <= bound).all()
    d = args[0].clone()
    assert K().lora_add(d, *args[1:], scales=scales.to(dev), out=d) is d and torch.equal(d, got)


def test_adapters_that_require_gradients(dev):
    """Refused where the native host call would take them; under no_grad parameters are operands like others."""
    g = torch.Generator().manual_seed(2)
    x, y = (torch.randn(3, 64, generator=g).half().to(dev) for _ in range(2))
    a, b = torch.randn(2, 8, 64, generator=g).half().to(dev), torch.randn(2, 64, 8, generator=g).half().to(dev)
    ids, scales = torch.tensor([1, -1, 0], dtype=torch.int32, device=dev), torch.rand(2, generator=g).to(dev)
    want = K().lora_add(y, x, a, b, ids, scales=scales)
    for i in range(5):
        d = [y, x, a, b, scales]
        d[i] = torch.nn.Parameter(d[i])

        def call(y, x, a, b, scales):
            return K().lora_add(y, x, a, b, ids, scales=scales)

        with pytest.raises(RuntimeError, match="no gradients"):
            call(*d)
        with torch.no_grad():
            assert torch.equal(call(*d), want) and torch.equal(torch.compile(call, backend="aot_eager", fullgraph=True)(*d), want)
        with torch.inference_mode():
            assert torch.equal(call(*d), want)


@pytest.mark.parametrize("code", [I8, E4M3])
@pytest.mark.parametrize("T,E,top,hidden,inter", [(16, 2, 2, 2048, 528), (12, 8, 6, 1040, 272), (64, 64, 6, 528, 144), (10, 4, 4, 2048, 80), (16, 2, 1, 1024, 512),
                                                  (48, 12, 1, 256, 1024)])
def test_experts_of_nine_tokens_and_more(dev, code, T, E, top, hidden, inter):
    args = make(gen(T + E), T, E, hidden, inter, code, torch.float32)
    first = check(dev, args, top)
    assert torch.equal(check(dev, args, top), first)


@pytest.mark.parametrize("rank,T", [(128, 2999), (128, 3000), (72, 3500), (72, 4095), (72, 4096), (16, 4096)])
def test_rows_about_the_larger_tiles(dev, rank, T):
    g = gen(rank + T)
    y, x, a, b, scales = lora.make(g, T, 136, 72, rank, 3, torch.float16)
    lora.check(dev, y, x, a, b, [2, -1, 0, 1], [3, 1500, 1501, 2000, T - 1], scales)


@pytest.mark.parametrize("T", [60, 4300])
@pytest.mark.parametrize("start,same", [([0, 0, 0, 0], None), ([60, 40, 20, 0], None), ([-9, 30, 2000000000, 60], [0, 30, 60, 60]), ([0, 50, 20, 60], False),
                                        ([2147483647, -2147483648, 5, 60], False), ([60, 0, 0, 60], False)])
def test_starts_of_any_values(dev, T, start, same):
    """Batches of 16-row and of 64-row tiles.  Rows that no request names are y's, starts outside of the rows end at them; where starts descend
    nothing but the rows of out is written."""
    k, g = K(), gen(T)
    y, x, a, b, scales = lora.make(g, T, 64, 72, 16, 2, torch.float16)
    by = T / 60
    given = [s if abs(s) > 100 else int(s * by) for s in start]
    if given[3] == int(60 * by):
        given[3] = T
    d = [t.to(dev) for t in (y, x, a, b, torch.tensor([0, 1, 0], dtype=torch.int32))]
    room = torch.full((T + 200, 72), 7.0, device=dev).half()
    out = k.lora_add(*d, torch.tensor(given, dtype=torch.int32, device=dev), scales=scales.to(dev), out=room[100:T + 100])
    torch.cuda.synchronize()
    assert (room[:100] == 7).all() and (room[T + 100:] == 7).all()
    if same is None:
        assert torch.equal(out, d[0])
    elif same:
        plain = [min(int(s * by), T) for s in same[:2]] + [T, T]
        assert torch.equal(out, k.lora_add(*d, torch.tensor(plain, dtype=torch.int32, device=dev), scales=scales.to(dev)))
        lora.check(dev, y, x, a, b, [0, 1, 0], plain, scales)


@pytest.mark.parametrize("T", [1, 4, 20, 64])
@pytest.mark.parametrize("which", [0, 3, 5])
def test_e4m3_codes_of_no_number_stay_with_their_tokens(dev, T, which):
    """In a token: its result alone; in an expert's weights: those of the tokens that it is run for."""
    args = list(make(gen(T), T, 4, 64, 32, E4M3, torch.float32))
    clean = check(dev, args, 2)
    args[which] = args[which].clone()
    if which == 0:
        args[0].view(torch.uint8)[T // 2, 3] = 0x7f
        odd = torch.arange(T) == T // 2
    else:
        args[which].view(torch.uint8)[1, 5, 7] = 0xff
        odd = torch.tensor([1 in row for row in R.route(args[2], 2, True)[0]])
    got = K().moe_few_tokens(*[t.to(dev) for t in args], 2, out_dtype=torch.float32).cpu()
    assert torch.equal(got[~odd], clean.cpu()[~odd]) and got[odd].isnan().any(1).all()


def test_several_launches_captured(dev):
    """Calls that are cut into several launches, replayed on new inputs with eager work and synchronizations between."""
    k, T, M = K(), 9000, (1 << 21) + 9
    g = torch.Generator(dev).manual_seed(4)

    def fresh():
        return (torch.empty(T, 64, device=dev, dtype=torch.float16).normal_(generator=g), torch.randint(-1, 3, (T,), device=dev, generator=g, dtype=torch.int32),
                torch.empty(M, 8, device=dev, dtype=torch.float16).normal_(generator=g))

    x, ids, rows = fresh()
    y = torch.empty(T, 72, device=dev, dtype=torch.float16).normal_(generator=g)
    a, b = (torch.empty(s, device=dev, dtype=torch.float16).normal_(generator=g) for s in ((3, 104, 64), (3, 72, 104)))
    w = torch.ones(8, device=dev).half()

    def call():
        return k.lora_add(y, x, a, b, ids), *k.add_rms_norm_quant(rows, w, dtype=I8)[:2]

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        for t, new in zip((x, ids, rows), fresh()):
            t.copy_(new)
        want = [t.clone() for t in call()]
        graph.replay()
        torch.empty(1 << 20, device=dev).normal_()
        if i % 2:
            torch.cuda.synchronize()
        for o, v in zip(out, want):
            assert torch.equal(o, v)
