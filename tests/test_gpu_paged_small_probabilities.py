"""Attention over a paged cache where one key stands out over very many small ones, and where probabilities enter as two terms: bounds
that follow the numbers the probabilities are held in, not the length of the cache."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu


def starts(n, rows):
    return None if rows == 1 else [i * rows for i in range(n + 1)]


def outstanding(dt, D, n, rows, heads, gap, at, seed):
    """q, k, v of one sequence and one key head: key `at` has a score of `gap` and a value of zero, all others scores of about zero and
    values of about one."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(rows, heads, D, generator=g)
    k = 0.05 * torch.randn(n, D, generator=g)
    v = 1.0 + 0.5 * torch.randn(n, D, generator=g)
    k[:, 0] = 0.0
    k[at] = 0.0
    k[at, 0] = 8.0
    v[at] = 0.0
    q[:, :, 0] = gap * D ** 0.5 / 8.0
    return q.to(dt), k.to(dt), v.to(dt)


def expected(q, k, v, at, held):
    """(out, bound).  held: what is lost of a probability at most, relative to the sequence's largest one, because its 16 bits end."""
    rows, heads, D = q.shape
    n = k.shape[0]
    scale = D ** -0.5
    u = R.eps_half(q.dtype)
    x, kd, vd = q.double().flatten(0, 1), k.double(), v.double()
    s = scale * x @ kd.T
    p = n - rows + torch.arange(rows).repeat_interleave(heads)
    s.masked_fill_(torch.arange(n) > p[:, None], -torch.inf)
    w = torch.softmax(s, -1)
    out = w @ vd
    mean = w @ vd.abs()
    # scores: D products and sums (the outstanding key: one product, the others are zero), the scale, the exponent's argument of up to 64
    size = scale * x.abs() @ kd.abs().T
    roundings = torch.full((n,), D + 8.0, dtype=torch.float64)
    roundings[at] = 9.0
    ds = (size * roundings).amax(-1, keepdim=True) * 2.0 ** -24 + 2.0 ** -18
    # sums: a matrix instruction takes 16 keys; l takes a tile of 64 at a time, of which a lane has added up 32
    adds = (n / 16 + n / 64 + 64) * 2.0 ** -23
    bound = u * out.abs() + (u + 2 * ds + adds) * (1 + u) * mean + n * held * vd.abs().max() + R.eps_half(q.dtype) * 2.0 ** -14
    return out.view(rows, heads, D), bound.view(rows, heads, D)


def run(dev, q, k, v, size, **kw):
    from fms_mo_amd import kernels as K

    rows, n, D = q.shape[0], k.shape[0], q.shape[2]
    pages = -(-n // size)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n))
    kc, vc = torch.zeros(2, pages, 1, size, D, dtype=q.dtype)
    for c, x in ((kc, k), (vc, v)):
        c[order, 0] = torch.cat([x, torch.zeros(pages * size - n, D, dtype=q.dtype)]).view(pages, size, D)
    start = None if rows == 1 else torch.tensor([0, rows], dtype=torch.int32, device=dev)
    y = K.paged_attention(q.to(dev), kc.to(dev), vc.to(dev), order.to(torch.int32)[None].to(dev), torch.tensor([n], dtype=torch.int32, device=dev),
                          start, **kw)
    torch.cuda.synchronize()
    return y


# fp16 ends 2^-25 below one; the split kernel holds powers up to 2^14, the prompt kernel at least 2^11 times the probability
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("gap", [10.0, 14.0, 18.0, 22.0])
@pytest.mark.parametrize("kind,rows,heads,hints", [
    ("one token", 1, 4, {}), ("one launch", 1, 4, dict(max_seq_len=64)), ("a few tokens", 3, 2, dict(max_query_len=3)),
    ("a prompt", 70, 2, dict(max_seq_len=64)), ("a prompt in parts", 70, 2, {})])
def test_small_probabilities_beside_a_large_one_fp16(dev, kind, rows, heads, hints, gap, D):
    n, at = 32768 + 100, 0
    q, k, v = outstanding(torch.float16, D, n, rows, heads, gap, at, D)
    ref, bound = expected(q, k, v, at, 2.0 ** -36 if rows == 70 else 2.0 ** -39)
    assert R.worst(run(dev, q, k, v, 32, **hints), ref, bound) <= 1.0


@pytest.mark.parametrize("rows,heads,hints", [(1, 4, {}), (70, 2, dict(max_seq_len=64)), (70, 2, {})])
@pytest.mark.parametrize("at", [777, 20001])
def test_a_large_one_met_later_fp16(dev, rows, heads, hints, at):
    n = 32768
    q, k, v = outstanding(torch.float16, 128, n, rows, heads, 17.0, at, at)
    ref, bound = expected(q, k, v, at, 2.0 ** -36 if rows == 70 else 2.0 ** -39)
    assert R.worst(run(dev, q, k, v, 64, **hints), ref, bound) <= 1.0


@pytest.mark.parametrize("rows", [1, 70])
def test_very_many_small_ones_fp16(dev, rows):
    n = 131072
    q, k, v = outstanding(torch.float16, 64, n, rows, 2, 16.0, 0, 5)
    ref, bound = expected(q, k, v, 0, 2.0 ** -36 if rows == 70 else 2.0 ** -39)
    assert R.worst(run(dev, q, k, v, 128), ref, bound) <= 1.0
