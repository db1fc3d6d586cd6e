"""Adapters of many requests against a 64-bit reference."""
import pytest
import torch

import layer_reference as R

pytestmark = pytest.mark.gpu


def K():
    from fms_mo_amd import kernels

    return kernels


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(g, T, cols, rows, rank, slots, dt, big=1.0):
    x, y = torch.randn(T, cols, generator=g).to(dt), torch.randn(T, rows, generator=g).to(dt)
    a, b = (big * cols ** -0.5 * torch.randn(slots, rank, cols, generator=g)).to(dt), torch.randn(slots, rows, rank, generator=g).to(dt)
    return y, x, a, b, 0.5 + torch.rand(slots, generator=g)


def check(dev, y, x, a, b, ids, start, scales, **kw):
    d = [t.to(dev) for t in (y, x, a, b)]
    got = K().lora_add(*d, torch.tensor(ids, dtype=torch.int32, device=dev),
                       None if start is None else torch.tensor(start, dtype=torch.int32, device=dev),
                       scales=None if scales is None else scales.to(dev), **kw)
    want, slack = R.lora(y, x, a, b, ids, start, scales)
    off = (got.cpu().double() - want).abs()
    bound = R.rounding(want, y.dtype) + slack * (1 + R.HALF[y.dtype]) + 2.0 ** -24 * want.abs()
    assert (off <= bound).all(), float((off / bound).max())
    return got


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 48, 64, 104, 128])
@pytest.mark.parametrize("cols,rows", [(64, 64), (8, 8), (200, 328), (1032, 1096)])
def test_one_row_per_request(dev, dt, rank, cols, rows):
    g = gen(rank + cols)
    for T, slots in ((1, 1), (5, 3), (40, 2)):
        ids = torch.randint(-1, slots + 1, (T,), generator=g).tolist()  # (none, and one too many, among them)
        check(dev, *make(g, T, cols, rows, rank, slots, dt)[:4], ids, None, None)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank", [8, 16, 40, 64, 128])
@pytest.mark.parametrize("cols,rows", [(64, 64), (136, 264), (1096, 520)])
@pytest.mark.parametrize("new", [[1], [3, 0, 5], [64], [65, 1, 130], [0, 0, 0], [15, 16, 17, 63], [200]])
def test_requests_of_several_rows(dev, dt, rank, cols, rows, new):
    g = gen(rank + cols + len(new))
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    T = max(start[-1], 1)
    y, x, a, b, scales = make(g, T, cols, rows, rank, 3, dt)
    ids = torch.randint(-1, 3, (len(new),), generator=g).tolist()
    check(dev, y, x, a, b, ids, start, scales)


def test_rows_of_no_request(dev):
    """Rows before the first request and behind the last one are y's, and are left as they are in place."""
    g = gen(3)
    y, x, a, b, scales = make(g, 230, 72, 136, 16, 2, torch.bfloat16)
    start = [7, 20, 150]
    want = check(dev, y, x, a, b, [1, 0], start, scales)
    for rows in (slice(0, 7), slice(150, 230)):
        assert torch.equal(want[rows].cpu().view(torch.int16), y[rows].view(torch.int16))
    d = y.to(dev)
    got = K().lora_add(d, x.to(dev), a.to(dev), b.to(dev), torch.tensor([1, 0], dtype=torch.int32, device=dev),
                       torch.tensor(start, dtype=torch.int32, device=dev), scales=scales.to(dev), out=d)
    assert got.data_ptr() == d.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
def test_rows_of_no_request_are_copied_whole(dev, dt, rank):
    """Many outputs of few rows without a request, again and again: each store leaves with the data that it was given."""
    g = gen(rank)
    y, x, a, b, scales = (t.to(dev) for t in make(g, 426, 72, 4104, rank, 2, dt))
    ids, start = torch.tensor([0, 1], dtype=torch.int32, device=dev), torch.tensor([0, 90, 423], dtype=torch.int32, device=dev)
    first = K().lora_add(y, x, a, b, ids, start, scales=scales)
    for _ in range(20):
        got = K().lora_add(y, x, a, b, ids, start, scales=scales)
        assert torch.equal(got[423:], y[423:]) and torch.equal(got, first)
    alone = torch.full((426,), -1, dtype=torch.int32, device=dev)
    for _ in range(5):
        assert torch.equal(K().lora_add(y, x, a, b, alone), y)


def test_no_adapter_keeps_the_bits(dev):
    y = torch.tensor([[-0.0, float("nan"), float("inf"), 1.0] * 4], device=dev).half()
    x = torch.full((1, 16), float("nan"), device=dev).half()
    a, b = torch.ones(1, 8, 16, device=dev).half(), torch.ones(1, 16, 8, device=dev).half()
    got = K().lora_add(y, x, a, b, torch.tensor([-1], dtype=torch.int32, device=dev))
    assert torch.equal(got.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("start", [[0, 50, 20, 60], [60, 40, 20, 0], [-9, 30, 2000000000, 60], [2147483647, -2147483648, 5, 60], [0, 0, 0, 0]])
def test_starts_that_mean_nothing(dev, start):
    """Nothing outside of the operands is touched, whatever the arrays say; rows that one request alone names are right."""
    g = gen(4)
    y, x, a, b, scales = (t.to(dev) for t in make(g, 60, 64, 72, 16, 2, torch.float16))
    room = torch.full((64, 72), 7.0, device=dev).half()
    K().lora_add(y, x, a, b, torch.tensor([0, 1, 0], dtype=torch.int32, device=dev), torch.tensor(start, dtype=torch.int32, device=dev),
                 scales=scales, out=room[2:62])
    torch.cuda.synchronize()
    assert (room[:2] == 7).all() and (room[62:] == 7).all()


def test_strided_operands(dev):
    """x and y inside wider rows, the pool a view of one with higher ranks."""
    g = gen(6)
    y, x, a, b, scales = make(g, 37, 128, 192, 32, 3, torch.bfloat16)
    ids = [2, 0, 1]
    start = [0, 4, 30, 37]
    want = check(dev, y, x, a[:, :16].contiguous(), b[:, :, :16].contiguous(), ids, start, scales)
    wx, wy = torch.zeros(37, 400, device=dev).bfloat16(), torch.zeros(37, 392, device=dev).bfloat16()
    wx[:, 136:264], wy[:, 192:384] = x.to(dev), y.to(dev)
    pool_a, pool_b = a.to(dev), b.to(dev)
    args = (torch.tensor(ids, dtype=torch.int32, device=dev), torch.tensor(start, dtype=torch.int32, device=dev))
    got = K().lora_add(wy[:, 192:384], wx[:, 136:264], pool_a[:, :16], pool_b[:, :, :16], *args, scales=scales.to(dev), out=wy[:, 192:384])
    assert torch.equal(got, want) and not wy[:, :192].any() and not wy[:, 384:].any()
    with pytest.raises(ValueError):  # a pool is not copied
        K().lora_add(wy[:, 192:384], wx[:, 136:264], pool_a[:, ::2, ].transpose(1, 2).contiguous().transpose(1, 2), pool_b[:, :, :16], *args)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_large_and_small_numbers(dev, dt):
    """a x beyond fp16's range, and far below its smallest numbers."""
    g = gen(8)
    for big, back in ((3000.0, 2.0 ** -14), (2.0 ** -13, 2.0 ** 10)):
        y, x, a, b, _ = make(g, 20, 512, 64, 16, 2, dt, big)
        x, scales = x * 64, torch.tensor([back, back])
        check(dev, y, x, a, b, [0, 1], [0, 3, 20], scales)


def test_no_numbers_stay_in_their_row(dev):
    g = gen(1)
    for start in (None, [0, 3, 70]):
        T = 2 if start is None else 70
        y, x, a, b, scales = make(g, T, 64, 64, 24, 2, torch.float16)
        clean = check(dev, y, x, a, b, [0, 0], start, scales)
        x[1, 5] = float("nan")
        got = K().lora_add(y.to(dev), x.to(dev), a.to(dev), b.to(dev), torch.tensor([0, 0], dtype=torch.int32, device=dev),
                           None if start is None else torch.tensor(start, dtype=torch.int32, device=dev), scales=scales.to(dev))
        assert got[1].isnan().all()
        keep = [t for t in range(T) if t != 1]
        assert torch.equal(got[keep], clean[keep])


def test_many_requests(dev):
    g = gen(11)
    y, x, a, b, scales = make(g, 700, 64, 64, 8, 5, torch.bfloat16)
    check(dev, y, x, a, b, torch.randint(-1, 5, (700,), generator=g).tolist(), None, scales)
    start = sorted(torch.randint(0, 701, (299,), generator=g).tolist())
    check(dev, y, x, a, b, torch.randint(-1, 5, (300,), generator=g).tolist(), [0] + start + [700], scales)


def test_rows_far_apart(dev):
    """One-row requests whose rows lie over more than 2 GB: what 32 bits reach at a time; an adapter's rows among both pieces."""
    g = gen(13)
    T, far = 300, 1 << 22
    y, x, a, b, scales = make(g, T, 64, 72, 8, 3, torch.float16)
    ids = torch.randint(-1, 3, (T,), generator=g).tolist()
    want = check(dev, y, x, a, b, ids, None, scales)
    room = torch.empty(T * far, dtype=torch.float16, device=dev)
    apart = room.as_strided((T, 64), (far, 1))
    apart.copy_(x)
    args = (a.to(dev), b.to(dev), torch.tensor(ids, dtype=torch.int32, device=dev))
    assert torch.equal(K().lora_add(y.to(dev), apart, *args, scales=scales.to(dev)), want)
    out = room.as_strided((T, 72), (far, 1), 128)
    assert K().lora_add(y.to(dev), x.to(dev), *args, scales=scales.to(dev), out=out) is out and torch.equal(out, want)
    start = torch.arange(0, T + 1, 2, dtype=torch.int32, device=dev)
    two = K().lora_add(y.to(dev), x.to(dev), *args[:2], args[2][:150], start, scales=scales.to(dev))
    assert torch.equal(K().lora_add(y.to(dev), apart, *args[:2], args[2][:150], start, scales=scales.to(dev)), two)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank,cols,rows,new", [(128, 4104, 264, [700]), (24, 72, 4104, [90, 333]), (64, 2056, 1032, [64, 128, 1, 500]), (16, 9000, 136, [1030]),
                                                (32, 264, 2056, [2000])])
def test_longer_requests(dev, dt, rank, cols, rows, new):
    g = gen(rank + cols)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    y, x, a, b, scales = make(g, start[-1] + 3, cols, rows, rank, 4, dt)
    ids = torch.randint(0, 4, (len(new),), generator=g).tolist()
    first = check(dev, y, x, a, b, ids, start, scales)
    assert torch.equal(check(dev, y, x, a, b, ids, start, scales), first)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rank,cols,rows", [(8, 136, 72), (16, 1032, 136), (24, 72, 1096), (64, 200, 264), (104, 264, 136), (128, 2056, 64)])
def test_tiles_of_64_rows(dev, dt, rank, cols, rows):
    """Enough rows, requests that end beside tiles and empty ones among them, rows of no request in front and behind; in place; a row of NaN, and
    infinities in one without an adapter, which is y's."""
    g = gen(rank + cols)
    start = [5]
    for n in (1200, 0, 63, 64, 65, 1, 128, 0, 2600):
        start.append(start[-1] + n)
    y, x, a, b, scales = make(g, start[-1] + 70, cols, rows, rank, 4, dt)
    ids = [3, 0, 1, -1, 2, 0, 4, 1, 0]
    x[40] = float("nan")
    x[1300] = float("inf")
    args = [t.to(dev) for t in (a, b)] + [torch.tensor(ids, dtype=torch.int32, device=dev), torch.tensor(start, dtype=torch.int32, device=dev)]
    got = K().lora_add(y.to(dev), x.to(dev), *args, scales=scales.to(dev))
    assert got[40].isnan().all() and torch.equal(got[1300].cpu(), y[1300])
    d = y.to(dev)
    K().lora_add(d, x.to(dev), *args, scales=scales.to(dev), out=d)
    assert torch.equal(d.view(torch.int16), got.view(torch.int16))
    x[40] = x[1300] = 0
    clean = check(dev, y, x, a, b, ids, start, scales)
    keep = [t for t in range(y.shape[0]) if t not in (40, 1300)]
    assert torch.equal(got[keep], clean[keep])
    for part in (slice(0, 5), slice(start[-1], None), slice(start[3], start[4])):
        assert torch.equal(got[part].cpu().view(torch.int16), y[part].view(torch.int16))


def test_nothing_to_do(dev):
    k = K()
    z = torch.empty(0, 64, device=dev).half()
    a, b, none = torch.zeros(2, 8, 64, device=dev).half(), torch.zeros(2, 64, 8, device=dev).half(), torch.empty(0, dtype=torch.int32, device=dev)
    assert k.lora_add(z, z, a, b, none).shape == (0, 64)
    y = torch.randn(3, 64, device=dev).half()
    start = torch.zeros(1, dtype=torch.int32, device=dev)
    assert torch.equal(k.lora_add(y, y, a, b, none, start), y)  # no requests: every row is y's
    one = torch.zeros(3, dtype=torch.int32, device=dev)
    assert torch.equal(k.lora_add(y, y, a[:0], b[:0], one), y)  # no slots: no adapter


def test_refusals(dev):
    k = K()
    x, y = torch.zeros(4, 64, device=dev).half(), torch.zeros(4, 32, device=dev).half()
    a, b = torch.zeros(2, 16, 64, device=dev).half(), torch.zeros(2, 32, 16, device=dev).half()
    ids = torch.zeros(4, dtype=torch.int32, device=dev)
    for bad, kind in [
        (lambda: k.lora_add(y.float(), x.float(), a.float(), b.float(), ids), TypeError),
        (lambda: k.lora_add(y, x.bfloat16(), a, b, ids), (TypeError, ValueError)),
        (lambda: k.lora_add(y.bfloat16(), x, a, b, ids), TypeError),
        (lambda: k.lora_add(y, x, a[:, :12], b[:, :, :12], ids), ValueError),
        (lambda: k.lora_add(y, x, a.repeat(1, 9, 1), b.repeat(1, 1, 9), ids), ValueError),
        (lambda: k.lora_add(y, x[:, :60], a[:, :, :60], b, ids), ValueError),
        (lambda: k.lora_add(y, x, a, b[:1], ids), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids[:3]), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids.long()), TypeError),
        (lambda: k.lora_add(y, x, a, b, ids, ids), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids, scales=torch.ones(3, device=dev)), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids, scales=torch.ones(2, device=dev).half()), ValueError),
        (lambda: k.lora_add(y[:3], x, a, b, ids), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids, out=y[:, :16]), ValueError),
        (lambda: k.lora_add(y, x, a, b, ids, out=y[:1].expand(4, 32)), ValueError),
        (lambda: k.lora_add(y, x, a, b.cpu(), ids), RuntimeError),
        (lambda: k.lora_add(y, x, a, b, ids.cpu()), RuntimeError),
    ]:
        with pytest.raises(kind):
            bad()
