"""Norm, rotation and store of so many tokens that a block goes through several groups of heads (768 and more), against 64 bits and against
the same tokens in calls of fewer."""
import pytest
import torch

import paged_reference as R
from test_gpu_kv_store import K, TYPES, gen, tables

pytestmark = pytest.mark.gpu

EPS = 1e-5


def turned(x, w, cos, sin, p, interleaved):
    """(y, how far fp32 may be from it) of rows [T, H, D] at positions p; see paged_reference.turned."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    y, off = x.clone(), x.abs()
    if cos is not None:
        half = cos.shape[1]
        c, s = cos[p].double()[:, None], sin[p].double()[:, None]
        one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
        a, b = x[..., one], x[..., two]
        y[..., one], y[..., two] = a * c - b * s, b * c + a * s
        off[..., one] = off[..., two] = a.abs() + b.abs()
    return y, off * 32 * 2.0 ** -24


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


# heads + key heads and their width: groups of 2048 elements 2 (the last one not full), 2, 3, 5, and 10 (two blocks, of 8 and of 2)
@pytest.mark.parametrize("heads,kv,D", [(9, 3, 256), (40, 4, 64), (32, 8, 128), (24, 8, 256), (64, 8, 256)])
@pytest.mark.parametrize("dt,e4m3", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_many_tokens(dev, dt, e4m3, heads, kv, D, interleaved, in_place):
    g = gen(heads + D)
    size, spare = 32, 6
    lens, new = [330, 40, 450, 900, 5, 9], [330, 0, 400, 100, 5, 12]  # (more new tokens than keys in the last one)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    T = start[-1] + spare
    assert start[-1] >= 768
    table, pages = R.make_pages(g, lens, size)
    table[2, 3], table[3, -3] = -7, pages
    k, v, ks, vs = R.make_cache(g, pages, kv, size, D, dt, e4m3)
    qkv = torch.randn(T, heads + 2 * kv, D, generator=g).to(dt)
    rotary = D if heads != 32 else D // 2
    cos, sin = tables(max(lens), rotary // 2)
    wdt = torch.float32 if heads == 24 else dt
    qw, kw = [(1 + 0.3 * torch.randn(D, generator=g)).to(wdt) for _ in range(2)]
    d = [None if t is None else t.to(dev) for t in (table, cos, sin, qw, kw)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    def call(x, cache, lens, start, table):
        q = x[:, :heads]
        return K().qk_norm_rope_store(q, x[:, heads:heads + kv], x[:, heads + kv:], cache[0], cache[1], table, i32(lens), i32(start), cos=d[1], sin=d[2],
                                      interleaved=interleaved, q_weight=d[3], k_weight=d[4], eps=EPS, k_scale=cache[2], v_scale=cache[3],
                                      out=q if in_place else None)
    cache = [None if t is None else t.to(dev) for t in (k, v, ks, vs)]
    small = [None if t is None else t.clone() for t in cache]
    x = qkv.to(dev)
    out = call(x, cache, lens, start, d[0])
    assert not in_place or out.data_ptr() == x.data_ptr()
    # sequence by sequence: calls of fewer tokens, whose blocks take one group of heads
    for b, n in enumerate(new):
        y = call(qkv[start[b]:start[b] + n].to(dev), small, lens[b:b + 1], [0, n], d[0][b:b + 1])
        assert torch.equal(out[start[b]:start[b] + n], y)
    for a, b in zip(cache, small):
        assert a is None or torch.equal(raw(a), raw(b))
    torch.cuda.synchronize()

    y = out.cpu()
    assert torch.equal(y[start[-1]:], qkv[start[-1]:, :heads] if in_place else torch.zeros_like(y[start[-1]:]))
    if in_place:
        assert torch.equal(x[:, heads:].cpu(), qkv[:, heads:])
    rows = R.rows_of(lens, start, T)
    seq, p = torch.tensor([r[1] for r in rows]), torch.tensor([r[2] for r in rows])
    assert (y[:len(rows)][p < 0] == 0).all()
    page = torch.tensor([-1 if (n := R.page_of(table, b, int(j), size, pages)) is None else n for b, j in zip(seq, p)])
    assert (page < 0).any()
    u = R.eps_half(dt)
    at = p.clamp(min=0)
    want, off = turned(qkv[:len(rows), :heads], qw, cos, sin, at, interleaved)
    assert (((y[:len(rows)].double() - want).abs() <= u * want.abs() * (1 + 1e-3) + off + 2.0 ** -25) | (p < 0)[:, None, None]).all()
    got = [None if t is None else t.cpu() for t in cache]
    there = page >= 0
    for i, (z, w, turn) in enumerate(((qkv[:, heads:heads + kv], kw, True), (qkv[:, heads + kv:], None, False))):
        want, off = turned(z[:len(rows)][there], w, cos if turn else None, sin, at[there], interleaved)
        have = got[i][page[there], :, at[there] % size].double()
        if not e4m3:
            assert ((have - want).abs() <= u * want.abs() * (1 + 1e-3) + off + 2.0 ** -25).all()
            continue
        s = got[2 + i][page[there], :, at[there] % size].double()
        top = want.abs().amax(-1) / 448
        assert ((s - top).abs() <= off.amax(-1) / 448 + top * 2.0 ** -22).all()
        t = want / s[..., None]
        assert ((have - t).abs() <= 2.0 ** -4 * t.abs() * (1 + 1e-3) + 2.0 ** -10 + off / s[..., None]).all()
        assert (have.abs().amax(-1) == 448).all()
    touched = torch.zeros(pages, size, dtype=torch.bool)
    touched[page[there], at[there] % size] = True
    keep = ~touched[:, None].expand(pages, kv, size)
    for was, now in zip((k, v, ks, vs), got):
        assert was is None or torch.equal(raw(was)[keep], raw(now)[keep])


@pytest.mark.parametrize("rotary,norm", [(0, True), (64, False), (16, True)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens_without_norm_or_rotation(dev, rotary, norm, interleaved):
    """The forms without a norm, without a rotation and with a part of it, and one token per sequence: as calls of fewer tokens have them."""
    g = gen(7)
    heads, kv, D, size, B = 32, 8, 128, 16, 800
    qkv = torch.randn(B, heads + 2 * kv, D, generator=g).bfloat16().to(dev)
    table = torch.randperm(B, generator=g).to(torch.int32)[:, None].to(dev)
    lens = torch.randint(1, 17, (B,), generator=g).to(torch.int32).to(dev)
    cos, sin = (t.to(dev) for t in tables(16, rotary // 2)) if rotary else (None, None)
    w = (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().to(dev) if norm else None
    caches = [[torch.zeros(B, kv, size, D, dtype=torch.float8_e4m3fn, device=dev) for _ in range(2)] + [torch.zeros(B, kv, size, device=dev) for _ in range(2)]
              for _ in range(2)]

    def call(x, c, table, lens):
        return K().qk_norm_rope_store(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], c[0], c[1], table, lens, cos=cos, sin=sin,
                                      interleaved=interleaved, q_weight=w, k_weight=w, k_scale=c[2], v_scale=c[3])
    whole = call(qkv, caches[0], table, lens)
    parts = torch.cat([call(qkv[i:i + 200], caches[1], table[i:i + 200], lens[i:i + 200]) for i in range(0, B, 200)])
    assert torch.equal(whole, parts)
    for a, b in zip(*caches):
        assert torch.equal(raw(a), raw(b))


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("lens,start,last", [
    ([BIG, -5], [0, 20, 40], 0), ([64, 64], [0, BIG, BIG], 0), ([64, 64], [30, 10, 40], 1), ([BIG, BIG], [-9, 5, -1], -1), ([64, 0], [60, 70, 80], -1),
    ([64, 64], [50, 0, 40], 1), ([64, 64], [0, 40, 20], 0)])
def test_nonsense_in_the_batch(dev, lens, start, last):
    """Rows and lengths that the operands don't have, and descending starts: nothing around the tensors changes, rows that no sequence names
    are zero, and a sequence's keys are written by its own rows only (`last`: the one sequence with rows)."""
    g = gen(14)
    table, pages = R.make_pages(g, [64, 64], 16)
    caches = torch.full((2, pages + 2, 2, 16, 64), 5.0, dtype=torch.float16, device=dev)
    kd, vd = caches[0, 1:-1], caches[1, 1:-1]
    x = torch.randn(40, 8, 64, generator=g).half().to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for in_place in (False, True):
        q = x[:, :4].clone() if in_place else x[:, :4]
        room = torch.full((44, 4, 64), 3.0, dtype=torch.float16, device=dev)
        out = K().qk_norm_rope_store(q, x[:, 4:6], x[:, 6:], kd, vd, table.to(dev), i32(lens), i32(start), out=room[2:42] if in_place else None)
        torch.cuda.synchronize()
        assert (room[:2] == 3).all() and (room[42:] == 3).all()
        assert (caches[:, 0] == 5).all() and (caches[:, -1] == 5).all()
        if last < 0:
            assert (out == (3 if in_place else 0)).all()
        theirs = [int(n) for n in table[1 - last] if 0 <= n < pages] if last >= 0 else range(pages)
        for n in theirs:
            assert (kd[n] == 5).all() and (vd[n] == 5).all()
