"""Attention over a paged cache, calls around the kernels: parts of a window, workspaces, many shares of a row, batches of nonsense."""
import pytest
import torch

import paged_reference as R
from test_gpu_paged_attn import TYPES, compare, gen, i32, on

pytestmark = pytest.mark.gpu


def workspace_bytes(q, k, seqs, most_rows, most_keys):
    from fms_mo_amd import _lib as L

    return L.load().fmsmo_paged_attn_workspace_bytes(q.shape[1], k.shape[1], k.shape[3], L.KV_E4M3 if k.dtype == torch.float8_e4m3fn else L.F16, seqs,
                                                     q.shape[0], most_rows, most_keys)


@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(1500, 70), (1100, 0)])
def test_a_window_in_parts(dev, dt, e4m3, D, window, sinks):
    """Rows whose window several blocks share, as a prompt and as single tokens."""
    compare(dev, dt, e4m3, 4, 2, D, 32, [2500, 40, 1700, 0], [40, 3, 33, 0], window=window, sinks=sinks, seed=D, spare_rows=2)
    compare(dev, dt, e4m3, 4, 2, D, 32, [2500, 40, 1700, 0], window=window, sinks=sinks, seed=D)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("window,sinks", [(20, 3), (1000, 0), (1 << 40, 1 << 40), (5, 1 << 40)])
def test_a_window_through_the_registered_operator(dev, new, window, sinks):
    """Workspaces of calls with a window are as large as the entry point wants them, on either way to it."""
    from fms_mo_amd import kernels as K

    g = gen(21)
    lens, start = [1800, 77], None if new == 1 else i32([0, new, 2 * new], dev)
    table, pages = R.make_pages(g, lens, 16)
    k, v, _, _ = R.make_cache(g, pages, 2, 16, 64, torch.float16, False)
    q = torch.randn(2 * new, 4, 64, generator=g).half()
    qd, kd, vd, td = on(dev, q, k, v, table)
    want = K.paged_attention(qd, kd, vd, td, i32(lens, dev), start, window=window, sinks=sinks, max_query_len=new, max_seq_len=1800)
    y = torch.empty_like(qd)
    torch.ops.fms_mo_amd.paged_attention(qd, kd, vd, td, i32(lens, dev), start, 0.125, window, sinks, None, None, new, 1800, y, True)
    assert torch.equal(y, want)
    ref, bound = R.attention(q, k, v, table, lens, None if new == 1 else [0, new, 2 * new], None, window, sinks)
    assert R.worst(y, ref, bound) <= 1.0


def against(q, k, v, p, scale, up):
    """(out, bound, weights) of one sequence with one key head: q [rows, heads, D] at positions p, k and v [n, D] fp64; up: the probabilities' rounding."""
    n, D = k.shape
    u = R.eps_half(q.dtype)
    x = q.double().flatten(0, 1)
    s = (scale * x @ k.T).masked_fill(torch.arange(n) > p.repeat_interleave(q.shape[1])[:, None], -torch.inf)
    w = torch.softmax(s, -1)
    out, mean = w @ v, w @ v.abs()
    # scores: D products and sums, the scale, the exponent's argument of up to 64; sums of 32 keys at a time, then of the waves' and blocks' shares
    ds = abs(scale) * (x.abs() @ k.abs().T).amax(-1, keepdim=True) * (D + 8) * 2.0 ** -24 + 2.0 ** -18
    bound = u * out.abs() + (up + 2 * ds + (n / 32 + 64) * 2.0 ** -23) * (1 + u) * mean + 2.0 ** -24
    return out.view(q.shape), bound.view(q.shape), w


def paged(dev, k, v, size, ks=None, vs=None):
    """k and v [n, D] (and scales [n]) in shuffled pages of one key head: caches, scales, block table on the device."""
    n, D = k.shape
    pages = -(-n // size)
    order = torch.randperm(pages, generator=gen(n))
    out = []
    for t in (k, v, ks, vs):
        if t is None:
            out.append(None)
            continue
        room = torch.zeros(pages * size, *t.shape[1:], dtype=t.dtype)
        (room.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else room)[:n] = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        c = torch.zeros(pages, 1, size, *t.shape[1:], dtype=t.dtype)
        a, b = (x.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else x for x in (c, room))
        a[order, 0] = b.view(pages, size, *b.shape[1:])
        out.append(c.to(dev))
    return out, order.to(torch.int32)[None].to(dev)


@pytest.mark.parametrize("e4m3,rows,heads", [(False, 1, 8), (False, 3, 4), (True, 1, 8), (True, 3, 4), (True, 6, 5)])
def test_bf16_probabilities_of_few_rows_are_two_terms(dev, e4m3, rows, heads):
    """The rounded result is off by its own rounding and 2^-16 of the probabilities, not by the 2^-8 that one bf16 number would cost.  Values
    of both signs over 70 keys: many results lie near zero, where the result's own rounding does not hide the probabilities'."""
    from fms_mo_amd import kernels as K

    g = gen(rows)
    n, D = 70, 128
    k, v, ks, vs = (None if t is None else t.view(n, *t.shape[3:]) for t in R.make_cache(g, n, 1, 1, D, torch.bfloat16, e4m3))
    q = torch.randn(rows, heads, D, generator=g).bfloat16()
    kd, vd = (t.double() if s is None else t.double() * s.double()[:, None] for t, s in ((k, ks), (v, vs)))
    p = n - rows + torch.arange(rows)
    ref, bound, w = against(q, kd, vd, p, D ** -0.5, 2.0 ** -16)
    # one term: the bound sees it
    scales = torch.ones(n) if vs is None else vs
    top = w.amax(-1, keepdim=True)
    once = ((w / top).float() * scales).bfloat16().double() * top @ v.double()
    assert R.worst(once.bfloat16().view(q.shape), ref, bound) > 2.0
    (kc, vc, kc_s, vc_s), table = paged(dev, k, v, 16, ks, vs)
    y = K.paged_attention(q.to(dev), kc, vc, table, i32([n], dev), None if rows == 1 else i32([0, rows], dev), k_scale=kc_s, v_scale=vc_s)
    assert R.worst(y, ref, bound) <= 1.0


@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("n", [70001, 140000])
def test_one_row_in_hundreds_of_shares(dev, dt, e4m3, n):
    """One sequence with one key head: 273 and 512 blocks, all of them on the same rows."""
    from fms_mo_amd import kernels as K

    g = gen(n)
    D = 64
    k, v, ks, vs = (None if t is None else t.view(n, *t.shape[3:]) for t in R.make_cache(g, n, 1, 1, D, dt, e4m3))
    q = (2 * torch.randn(1, 4, D, generator=g)).to(dt)
    kd, vd = (t.double() if s is None else t.double() * s.double()[:, None] for t, s in ((k, ks), (v, vs)))
    ref, bound, _ = against(q, kd, vd, torch.tensor([n - 1]), D ** -0.5, R.eps_half(dt) if dt == torch.float16 and not e4m3 else 2.0 ** -16)
    (kc, vc, kc_s, vc_s), table = paged(dev, k, v, 32, ks, vs)
    cuts, share = 32, 16 * (D + 2) * 4
    assert workspace_bytes(q, kc, 1, 1, n) == {70001: 273, 140000: 512}[n] * (cuts + 2 * share)
    y = K.paged_attention(q.to(dev), kc, vc, table, i32([n], dev), k_scale=kc_s, v_scale=vc_s)
    assert R.worst(y, ref, bound) <= 1.0


@pytest.mark.parametrize("new,lens", [(1, [2600, 2000]), (40, [2600, 2000])])
def test_two_streams_and_a_graph_with_workspaces(dev, new, lens):
    """Calls in parts: on two streams at once, captured, replayed with eager calls between the replays."""
    from fms_mo_amd import kernels as K

    g = gen(8)
    table, pages = R.make_pages(g, lens, 32)
    k, v, _, _ = R.make_cache(g, pages, 2, 32, 64, torch.float16, False)
    T = 2 * new
    start = None if new == 1 else i32([0, new, T], dev)
    kd, vd, td, ld = k.to(dev), v.to(dev), table.to(dev), i32(lens, dev)
    q = [torch.randn(T, 4, 64, generator=g).half().to(dev) for _ in range(2)]
    assert workspace_bytes(q[0], kd, 2, new, lens[0]) > 0

    def call(x):
        return K.paged_attention(x, kd, vd, td, ld, start, max_query_len=new, max_seq_len=lens[0])
    want = [call(x) for x in q]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(side):
            with torch.cuda.stream(s):
                got[i].append(call(q[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(q[0])
    for i in range(4):
        now = [lens[0] - 370 * i, lens[1] - 100 * i]
        ld.copy_(i32(now, dev))
        q[0].normal_()
        graph.replay()
        want = call(q[0])
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    ref, bound = R.attention(q[0].cpu(), k, v, table, now, None if new == 1 else [0, new, T])
    assert R.worst(y, ref, bound) <= 1.0


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("lens,start,defined", [
    ([BIG, -5], [0, 20, 40], True), ([64, 64], [0, BIG, BIG], False), ([64, 64], [30, 10, 40], True), ([BIG, BIG], [-9, 5, -1], True), ([64, 0], [60, 70, 80], True)])
def test_nonsense_in_the_batch(dev, lens, start, defined):
    """Rows and lengths that the operands don't have, and descending starts: rows that a sequence names are computed from the keys that are
    there, all others stay, and nothing around the tensors changes."""
    from fms_mo_amd import kernels as K

    g = gen(14)
    table, pages = R.make_pages(g, [64, 64], 16)
    k, v, _, _ = R.make_cache(g, pages, 2, 16, 64, torch.float16, False)
    td = table.to(dev)
    caches = torch.full((2, pages + 2, 2, 16, 64), 5.0, dtype=torch.float16, device=dev)
    kd, vd = caches[0, 1:-1], caches[1, 1:-1]
    kd.copy_(k)
    vd.copy_(v)
    q = torch.randn(40, 4, 64, generator=g).half().to(dev)
    ld, sd = i32(lens, dev), i32(start, dev)
    rows = [r for r in R.rows_of(lens, start, 40) if start[r[1]] >= 0] if defined else []
    named = torch.zeros(40, dtype=torch.bool)
    named[[r[0] for r in rows]] = True
    for hint in (1, 8, 40):
        for w in (0, 5, BIG):
            room = torch.full((44, 4, 64), 3.0, dtype=torch.float16, device=dev)
            K.paged_attention(q, kd, vd, td, ld, sd, max_query_len=hint, out=room[2:42], window=w, sinks=2)
            assert (room[:2] == 3).all() and (room[42:] == 3).all()
            if defined:
                y = room[2:42].cpu()
                assert (y[~named] == 3).all()
                if rows:
                    ref, bound = R.attention(q.cpu(), k, v, table, lens, start, None, w, 2)
                    assert R.worst(y[named], ref[named], bound[named]) <= 1.0
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


@pytest.mark.parametrize("hint", [1, 4096])
def test_starts_that_go_up_and_down(dev, hint):
    """200 sequences that name the same 4096 rows, 2^24 units of work each: more rows than there are, of which nothing is computed by the kernel
    of few rows; the prompt kernel's blocks are as many as rows have tiles."""
    from fms_mo_amd import kernels as K

    g = gen(22)
    q = torch.randn(4096, 128, 64, generator=g).half().to(dev)
    k, v = (torch.randn(4, 8, 16, 64, generator=g).half().to(dev) for _ in range(2))
    seqs, P = 400, 4096
    table = torch.randint(0, 4, (1, P), generator=g).to(torch.int32).to(dev).expand(seqs, P)
    lens, start = i32([65536] * seqs, dev), i32([0, 4096] * (seqs // 2) + [0], dev)
    out = torch.full((4098, 128, 64), 3.0, dtype=torch.float16, device=dev)
    K.paged_attention(q, k, v, table, lens, start, max_query_len=hint, out=out[1:-1])
    assert (out[0] == 3).all() and (out[-1] == 3).all()
    if hint == 1:
        assert (out == 3).all()
    # what follows is as ever
    compare(dev, torch.float16, False, 4, 2, 64, 16, [100, 65, 1, 0, 333], [2, 1, 1, 0, 3], seed=3)


@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("new", [1, 3, 70])
def test_a_scale_that_is_no_number(dev, dt, e4m3, new):
    from fms_mo_amd import kernels as K

    g = gen(23)
    lens, start = [300, 77], None if new == 1 else i32([0, new, 2 * new], dev)
    table, pages = R.make_pages(g, lens, 16)
    kd, vd, ksd, vsd = on(dev, *R.make_cache(g, pages, 2, 16, 64, dt, e4m3))
    q = torch.randn(2 * new, 4, 64, generator=g).to(dt).to(dev)
    y = K.paged_attention(q, kd, vd, table.to(dev), i32(lens, dev), start, scale=float("nan"), k_scale=ksd, v_scale=vsd, max_query_len=new)
    assert y.isnan().all()


@pytest.mark.parametrize("rows,heads", [(1, 8), (3, 4)])
def test_fp16_probabilities_of_few_rows_are_two_terms(dev, rows, heads):
    """As for bf16: its own rounding and 2^-22 of the probabilities, not the 2^-11 of one fp16 number."""
    from fms_mo_amd import kernels as K

    g = gen(rows)
    n, D = 70, 128
    k, v = (t.view(n, D) for t in R.make_cache(g, n, 1, 1, D, torch.float16, False)[:2])
    q = (0.1 * torch.randn(rows, heads, D, generator=g)).half()
    ref, bound, w = against(q, k.double(), v.double(), n - rows + torch.arange(rows), D ** -0.5, 2.0 ** -22)
    top = w.amax(-1, keepdim=True)
    once = (w / top).half().double() * top @ v.double()
    assert R.worst(once.half().view(q.shape), ref, bound) > 1.5
    (kc, vc, _, _), table = paged(dev, k, v, 16)
    y = K.paged_attention(q.to(dev), kc, vc, table, i32([n], dev), None if rows == 1 else i32([0, rows], dev))
    assert R.worst(y, ref, bound) <= 1.0
