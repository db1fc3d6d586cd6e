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
