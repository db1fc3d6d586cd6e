"""Norm, rotation and store of new tokens into a paged cache against a 64-bit reference."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def K():
    from fms_mo_amd import kernels

    return kernels


def tables(n, half):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


def check(dev, dt, e4m3, heads, kv, D, size, lens, new=None, rotary=None, norm=True, interleaved=False, wdt=None, spare=0, seed=0, edit=None,
          layout="heads", in_place=False):
    g = gen(seed)
    start = None
    if new is not None:
        start = [0]
        for n in new:
            start.append(start[-1] + n)
    T = (len(lens) if new is None else start[-1]) + spare
    table, pages = R.make_pages(g, lens, size)
    if edit:
        table = edit(table)
    k, v, ks, vs = R.make_cache(g, pages, kv, size, D, dt, e4m3, layout)
    qkv = torch.randn(T, heads + 2 * kv, D, generator=g).to(dt)
    cos = sin = None
    if rotary:
        cos, sin = tables(max(lens + [1]), rotary // 2)
    qw, kw = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdt or dt) for _ in range(2)] if norm else (None, None)
    before = [None if t is None else t.clone() for t in (k, v, ks, vs)]
    d = [None if t is None else t.to(dev) for t in (k, v, table, cos, sin, qw, kw, ks, vs)]
    x = qkv.to(dev)
    q = x[:, :heads]
    out = K().qk_norm_rope_store(q, x[:, heads:heads + kv], x[:, heads + kv:], d[0], d[1], d[2],
                                 torch.tensor(lens, dtype=torch.int32, device=dev),
                                 None if start is None else torch.tensor(start, dtype=torch.int32, device=dev), cos=d[3], sin=d[4],
                                 interleaved=interleaved, q_weight=d[5], k_weight=d[6], eps=1e-5, k_scale=d[7], v_scale=d[8],
                                 out=q if in_place else None)
    torch.cuda.synchronize()
    u = R.eps_half(dt)
    got = [None if t is None else t.cpu() for t in (d[0], d[1], d[7], d[8])]
    y = out.cpu().double()
    touched = torch.zeros(pages, size, dtype=torch.bool)
    mine = torch.zeros(T, dtype=torch.bool)
    for r, b, p in R.rows_of(lens, start, T):
        mine[r] = True
        if p < 0:
            assert (y[r] == 0).all()
            continue
        want, off = R.turned(qkv[r, :heads], qw, 1e-5, cos, sin, p, interleaved)
        assert ((y[r] - want).abs() <= u * want.abs() * (1 + 1e-3) + off + 2.0 ** -25).all()
        page = R.page_of(table, b, p, size, pages)
        if page is None:
            continue
        touched[page, p % size] = True
        for i, (xr, w, tables_) in enumerate(((qkv[r, heads:heads + kv], kw, (cos, sin)), (qkv[r, heads + kv:], None, (None, None)))):
            want, off = R.turned(xr, w, 1e-5, tables_[0], tables_[1], p, interleaved)
            have = got[i][page, :, p % size].double()
            if not e4m3:
                assert ((have - want).abs() <= u * want.abs() * (1 + 1e-3) + off + 2.0 ** -25).all()
                continue
            s = got[2 + i][page, :, p % size].double()
            ref = want.abs().amax(-1) / 448
            assert ((s - ref).abs() <= off.amax(-1) / 448 + ref * 2.0 ** -22).all()
            # half a step of e4m3 (2^-4 of the value, 2^-10 under its normals) of the quotient by the scale that was stored
            t = want / s[:, None]
            assert ((have - t).abs() <= 2.0 ** -4 * t.abs() * (1 + 1e-3) + 2.0 ** -10 + off / s[:, None]).all()
            assert (have.abs().amax(-1) == 448).all()
    for i, t in enumerate(before):  # nothing else was written
        if t is None:
            continue
        now = got[i].view(torch.uint8) if t.dtype == torch.float8_e4m3fn else got[i]
        was = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
        keep = ~touched[:, None].expand(pages, kv, size)
        assert torch.equal(now[keep], was[keep])
    if not in_place:
        assert (y[~mine] == 0).all()
    else:
        assert torch.equal(out.cpu()[~mine], qkv[:, :heads][~mine])
    return d, out


TYPES = [(torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)]


@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("heads,kv,D", [(8, 2, 128), (3, 3, 64), (5, 1, 256), (64, 8, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_one_token(dev, dt, e4m3, heads, kv, D, interleaved):
    check(dev, dt, e4m3, heads, kv, D, 16, [1, 17, 40, 0, 300], rotary=D, interleaved=interleaved, seed=D)


@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("rotary,norm", [(0, True), (0, False), (64, False), (32, True), (16, True), (128, False)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_prompts(dev, dt, e4m3, rotary, norm, interleaved):
    check(dev, dt, e4m3, 4, 2, 128, 32, [70, 33, 0, 5, 200], [70, 2, 0, 0, 63], rotary=rotary, norm=norm, interleaved=interleaved, spare=5,
          seed=rotary, wdt=torch.float32 if rotary == 32 else None)


@pytest.mark.parametrize("dt,e4m3", TYPES)
def test_pages_that_are_not_there_and_more_tokens_than_keys(dev, dt, e4m3):
    def edit(t):
        t = t.clone()
        t[0, 1] = -5
        t[1, 0] = 1 << 30
        return t
    check(dev, dt, e4m3, 4, 2, 64, 16, [40, 20, 3], [40, 20, 7], rotary=64, edit=edit)
    check(dev, dt, e4m3, 4, 2, 64, 16, [60, 20], [60, 20], rotary=64, edit=lambda t: t[:, :2].contiguous())


@pytest.mark.parametrize("dt,e4m3", TYPES)
def test_in_place_layouts_and_many_sequences(dev, dt, e4m3):
    check(dev, dt, e4m3, 4, 2, 128, 16, [70, 33], [70, 2], rotary=128, in_place=True, spare=4)
    check(dev, dt, e4m3, 4, 2, 128, 16, [70, 33], [70, 2], rotary=64, layout="keys", in_place=True)
    check(dev, dt, e4m3, 2, 1, 64, 16, [1 + i % 7 for i in range(200)], [i % 3 for i in range(200)], rotary=64)


def test_values_e4m3_has_no_room_for(dev):
    """Rows of zeros, of tiny values, with infinities and NaN: the recipe's floor of the scale, NaN codes, nothing silently finite."""
    D, kv, size = 64, 1, 16
    x = torch.zeros(6, 3, D, dtype=torch.bfloat16)
    x[1] = 1e-15
    x[2, :, 3] = float("inf")
    x[3, :, 4] = float("nan")
    x[4] = -0.0
    x[5, :, 0] = -3e38
    table = torch.zeros(6, 1, dtype=torch.int32)
    k, v = (torch.zeros(1, kv, size, D, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(1, kv, size, device=dev) for _ in range(2))
    xd = x.to(dev)
    K().qk_norm_rope_store(xd[:, :1], xd[:, 1:2], xd[:, 2:], k, v, table.to(dev), torch.arange(1, 7, dtype=torch.int32, device=dev), k_scale=ks, v_scale=vs)
    f, s = v[0, 0, :6].float().cpu(), vs[0, 0, :6].cpu()
    floor = torch.tensor(1e-12)
    assert s[0] == floor and s[1] == floor and s[4] == floor and s[2] == float("inf") and s[3].isnan()
    assert (f[0] == 0).all() and (f[4] == 0).all()
    assert torch.equal(f[1], (x[1, 0].float() / floor).to(torch.float8_e4m3fn).float())
    assert f[2, 3].isnan() and f[3].isnan().all()
    assert f[5, 0] == -448 and (f[5, 1:] == 0).all()
    assert torch.equal(k.view(torch.uint8), v.view(torch.uint8))


def test_positions_behind_the_tables_are_not_numbers(dev):
    D = 64
    x = torch.randn(2, 3, D, generator=gen(0)).half().to(dev)
    k, v = (torch.zeros(4, 1, 16, D, dtype=torch.float16, device=dev) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
    cos, sin = (t.to(dev) for t in tables(20, 32))
    q = K().qk_norm_rope_store(x[:, :1], x[:, 1:2], x[:, 2:], k, v, table, torch.tensor([20, 21], dtype=torch.int32, device=dev), cos=cos, sin=sin)
    assert torch.isfinite(q[0]).all() and q[1].isnan().all() and k[3, 0, 4].isnan().all() and torch.equal(v[3, 0, 4], x[1, 2])


def test_store_then_attend_as_a_model_does(dev):
    """A prompt in two chunks, then tokens one by one, through PagedKVCache, against attention over all of them at once in 64 bits."""
    from fms_mo_amd.modules.attention import PagedKVCache

    g = gen(11)
    heads, kv, D, L = 8, 2, 128, 140
    cos, sin = tables(L, D // 2)
    for dt, cdt in ((torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn)):
        cache = PagedKVCache(16, 16, kv, D, cdt, device=dev)
        x = torch.randn(L, heads + 2 * kv, D, generator=g).to(dt)
        w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dt) for _ in range(2)]
        table = torch.randperm(16, generator=g).to(torch.int32)[None]
        parts, at = [], 0
        for n in (100, 32, 1, 1, 3, 1, 2):
            xd = x[at:at + n].to(dev)
            at += n
            lens = torch.tensor([at], dtype=torch.int32, device=dev)
            start = None if n == 1 else torch.tensor([0, n], dtype=torch.int32, device=dev)
            q = cache.store(xd[:, :heads], xd[:, heads:heads + kv], xd[:, heads + kv:], table.to(dev), lens, start, cos=cos.to(dev),
                            sin=sin.to(dev), q_weight=w[0].to(dev), k_weight=w[1].to(dev))
            parts.append((q, cache.attend(q, table.to(dev), lens, start, window=90, sinks=3)))
        q, y = (torch.cat([p[i] for p in parts]).cpu() for i in range(2))
        ks, vs = (None if t is None else t.cpu() for t in (cache.k_scale, cache.v_scale))
        ref, bound = R.attention(q, cache.k.cpu(), cache.v.cpu(), table, [L], [0, L], None, 90, 3, ks, vs)
        assert at == L and R.worst(y, ref, bound) <= 1.0
        want = torch.stack([R.turned(x[p, :heads], w[0], 1e-6, cos, sin, p, False)[0] for p in range(L)])
        assert ((q.double() - want).abs() <= R.eps_half(dt) * want.abs() * 1.01 + 2.0 ** -14).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_codes_are_those_of_a_division(dev, dt, D):
    """Scale and codes bit for bit those of max / 448 and x / scale divided in fp32, over the types' whole range of scales (the values,
    which neither norm nor rotation changes)."""
    g = gen(D)
    T, kv, size = 900, 2, 64
    x = torch.randn(T, 3 * kv, D, generator=g)
    top = 120 if dt == torch.bfloat16 else 12
    x = (x * 2.0 ** torch.randint(-top, top, (T, 3 * kv, 1), generator=g)).to(dt)
    x[::7] = x[::7].abs().clamp(max=1.0)
    pages = -(-T // size)
    k, v = (torch.zeros(pages, kv, size, D, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(pages, kv, size, device=dev) for _ in range(2))
    xd = x.to(dev)
    K().qk_norm_rope_store(xd[:, :kv], xd[:, kv:2 * kv], xd[:, 2 * kv:], k, v, torch.arange(pages, dtype=torch.int32, device=dev)[None],
                           torch.tensor([T], dtype=torch.int32, device=dev), torch.tensor([0, T], dtype=torch.int32, device=dev), k_scale=ks, v_scale=vs)
    for part, codes, scales in ((x[:, kv:2 * kv], k, ks), (x[:, 2 * kv:], v, vs)):
        f = part.float()
        s = (f.abs().amax(-1) / 448).clamp(min=1e-12)
        want = (f / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        have = codes.cpu().view(torch.uint8).transpose(1, 2).reshape(-1, kv, D)[:T]
        assert torch.equal(scales.cpu().transpose(1, 2).reshape(-1, kv)[:T], s)
        assert torch.equal(have, want.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_captured_step_replays(dev, dtype):
    """Store and attention of single tokens in one graph, replayed as the sequences grow, with eager steps on a second cache between."""
    from fms_mo_amd.modules.attention import PagedKVCache

    g = gen(5)
    heads, kv, D, size, B = 8, 2, 128, 16, 3
    caches = [PagedKVCache(40, size, kv, D, dtype, dev) for _ in range(2)]
    table = torch.randperm(40, generator=g)[:36].reshape(B, 12).to(torch.int32).to(dev)
    cos, sin = (t.to(dev) for t in tables(200, D // 2))
    w = (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().to(dev)
    x = torch.zeros(B, heads + 2 * kv, D, dtype=torch.bfloat16, device=dev)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)

    def step(cache):
        q = cache.store(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], table, lens, cos=cos, sin=sin, q_weight=w, k_weight=w)
        return cache.attend(q, table, lens, max_seq_len=192)
    lens.copy_(torch.tensor([1, 15, 100], dtype=torch.int32))
    for cache in caches:
        step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(caches[0])
    for i in range(20):
        lens += 1
        x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        graph.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
