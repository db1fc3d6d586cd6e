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
