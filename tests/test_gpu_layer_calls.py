"""The operators around a layer's products together and as a serving program calls them: one behind the other, captured, on other streams, compiled."""
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu


def K():
    from fms_mo_amd import kernels

    return kernels


class Layer:
    """residual + norm -> projection with adapters -> residual + norm -> experts; int8 or e4m3."""

    def __init__(self, dev, code, hidden=256, inter=96, experts=6, rank=16, seed=0):
        g = torch.Generator().manual_seed(seed)
        int8 = code == torch.int8

        def weights(*shape):
            x = torch.randn(*shape, generator=g)
            return ((32 * x).round().clamp(-127, 127).to(code) if int8 else (100 * x).clamp(-448, 448).to(code)).to(dev)

        unit = 1 / 32 if int8 else 1 / 100
        self.code, self.top = code, 2
        self.n1, self.n2 = ((1 + 0.2 * torch.randn(hidden, generator=g)).bfloat16().to(dev) for _ in range(2))
        self.w, self.ws = weights(hidden, hidden), torch.full((hidden,), unit * hidden ** -0.5, device=dev)
        self.a, self.b = ((torch.randn(*s, generator=g) * hidden ** -0.5).bfloat16().to(dev) for s in ((3, rank, hidden), (3, hidden, rank)))
        self.router = (torch.randn(experts, hidden, generator=g) * hidden ** -0.5).bfloat16().to(dev)
        self.w13, self.s13 = weights(experts, 2 * inter, hidden), torch.full((experts, 2 * inter), unit * hidden ** -0.5, device=dev)
        self.w2, self.s2 = weights(experts, hidden, inter), torch.full((experts, hidden), unit * inter ** -0.5, device=dev)

    def __call__(self, x, residual, ids, start=None):
        k = K()
        q, s, r, n = k.add_rms_norm_quant(x, self.n1, residual, dtype=self.code, want_normed=True)
        gemm = k.gemm_i8_dq if self.code == torch.int8 else k.gemm_fp8_dq
        y = gemm(q, self.w, s, self.ws, out_dtype=torch.bfloat16)
        y = k.lora_add(y, n, self.a, self.b, ids, start, out=y)
        q, s, r, n = k.add_rms_norm_quant(y, self.n2, r, dtype=self.code, want_normed=True)
        logits = n.float() @ self.router.float().t()
        return k.moe_few_tokens(q, s, logits, self.w13, self.s13, self.w2, self.s2, self.top), r, (y, n, logits)


def inputs(dev, T, hidden=256, seed=1, start=None):
    g = torch.Generator().manual_seed(seed)
    x, r = torch.randn(T, hidden, generator=g).bfloat16().to(dev), torch.randn(T, hidden, generator=g).bfloat16().to(dev)
    n = T if start is None else len(start) - 1
    return x, r, torch.randint(-1, 3, (n,), generator=g).to(torch.int32).to(dev), None if start is None else torch.tensor(start, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T,start", [(1, None), (13, None), (40, [0, 3, 40]), (64, [0, 0, 64])])
def test_a_run(dev, code, T, start):
    """Each step against its reference on what the step before gave."""
    k, layer = K(), Layer(dev, code)
    x, r, ids, st = inputs(dev, T, start=start)
    out, r2, (y, n, logits) = layer(x, r, ids, st)
    cpu = lambda *t: [None if v is None else v.cpu() for v in t]  # noqa: E731
    eh, en = R.norm(*cpu(x, layer.n1, r), 1e-6)
    q, s, r1, n1 = k.add_rms_norm_quant(x, layer.n1, r, dtype=code, want_normed=True)
    assert ((r1.cpu().double() - eh).abs() <= R.rounding(eh, torch.bfloat16) * 1.01).all()
    p = (k.gemm_i8_dq if code == torch.int8 else k.gemm_fp8_dq)(q, layer.w, s, layer.ws, out_dtype=torch.bfloat16)
    want, slack = R.lora(*cpu(p, n1, layer.a, layer.b, ids), start, None)
    assert ((y.cpu().double() - want).abs() <= R.rounding(want, torch.bfloat16) * 1.01 + slack).all()
    q, s, _, _ = k.add_rms_norm_quant(y, layer.n2, r1, dtype=code)
    want, slack = R.moe(*cpu(q, s, logits, layer.w13, layer.s13, layer.w2, layer.s2), 2)
    assert ((out.cpu().double() - want).abs() <= R.rounding(want, torch.bfloat16) * 1.01 + slack).all()


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T,start", [(1, None), (9, None), (64, [0, 30, 64])])
def test_graph_replays(dev, code, T, start):
    """Replays on new inputs, eager work and synchronizations between them, against eager calls."""
    layer = Layer(dev, code)
    x, r, ids, st = inputs(dev, T, start=start)
    layer(x, r, ids, st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, r, ids, st)
    for seed in range(4):
        x2, r2, i2, s2 = inputs(dev, T, seed=10 + seed, start=start)
        want = layer(x2, r2, i2, s2)
        x.copy_(x2), r.copy_(r2), ids.copy_(i2)
        graph.replay()
        torch.empty(1 << 20, device=dev).normal_()
        if seed % 2:
            torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_graphs_in_flight(dev):
    """Two captured calls replayed at once keep their workspaces apart."""
    layers = [Layer(dev, torch.int8, seed=s) for s in (1, 2)]
    data = [inputs(dev, 17, seed=s) for s in (3, 4)]
    want, graphs, outs, streams = [], [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for layer, d in zip(layers, data):
        want.append(layer(*d)[0].clone())
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(layer(*d)[0])
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert torch.equal(w, o)


def test_two_streams_at_once(dev):
    layer = Layer(dev, torch.float8_e4m3fn)
    data = [inputs(dev, T, seed=T) for T in (5, 64)]
    want = [layer(*d)[0] for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(layer(*data[i])[0])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, v) for v in g)


def test_same_bits_every_time(dev):
    layer = Layer(dev, torch.int8, hidden=512, inter=208)
    d = inputs(dev, 64, hidden=512)
    first = layer(*d)[0]
    for _ in range(10):
        assert torch.equal(layer(*d)[0], first)


def test_operators_and_general_path(dev):
    """The registered operators, and tensors that the native host calls hand on, give what plain calls give."""
    k, layer = K(), Layer(dev, torch.int8)
    x, r, ids, _ = inputs(dev, 6)
    q, s, h, n = k.add_rms_norm_quant(x, layer.n1, r, want_normed=True)
    q2, s2, h2, n2 = torch.empty_like(q), torch.empty_like(s), torch.empty_like(h), torch.empty_like(n)
    torch.ops.fms_mo_amd.add_rms_norm_quant(x, layer.n1, r, 1e-6, None, q2, s2, h2, n2)
    for a, b in ((q, q2), (s, s2), (h, h2), (n, n2)):
        assert torch.equal(a, b)
    y = k.lora_add(x, n, layer.a, layer.b, ids)
    out = torch.empty_like(y)
    torch.ops.fms_mo_amd.lora_add(x, n, layer.a, layer.b, ids, None, None, out)
    assert torch.equal(y, out)
    logits = n.float() @ layer.router.float().t()
    z = k.moe_few_tokens(q, s, logits, layer.w13, layer.s13, layer.w2, layer.s2, 2)
    out = torch.empty_like(z)
    torch.ops.fms_mo_amd.moe_few_tokens(q, s, logits, layer.w13, layer.s13, layer.w2, layer.s2, 2, True, out)
    assert torch.equal(z, out)
    odd = torch.empty(6 * 256 + 1, dtype=torch.int8, device=dev)[1:].view(6, 256).copy_(q)  # an address that is no multiple of 16
    assert torch.equal(k.moe_few_tokens(odd, s, logits, layer.w13, layer.s13, layer.w2, layer.s2, 2), z)
    p = torch.nn.Parameter(layer.n1)
    assert torch.equal(k.add_rms_norm_quant(x, p, r)[0], q)


def test_compiled(dev):
    layer = Layer(dev, torch.int8)
    x, r, ids, _ = inputs(dev, 6)

    def step(x, r, ids):
        out, r2, _ = layer(x, r, ids)
        return out, r2

    want = step(x, r, ids)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(x, r, ids)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_current_device_and_stream(dev):
    """Work goes to the stream that is current: a call behind a long copy there sees its result."""
    k, layer = K(), Layer(dev, torch.int8)
    x, r, ids, _ = inputs(dev, 8)
    want = k.add_rms_norm_quant(x, layer.n1, r)[0]
    side = torch.cuda.Stream()
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=dev)
        for _ in range(4):
            big = big @ big * 1e-2
        late.copy_(x)
        got = k.add_rms_norm_quant(late, layer.n1, r)[0]
    side.synchronize()
    assert torch.equal(got, want)
