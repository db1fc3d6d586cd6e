"""How attention over a paged cache is divided, as its workspace shows it, without a GPU: every call below is refused before a launch."""
import random

import test_paged_rules as rules
from test_paged_rules import ALIGN, SCRATCH, p  # noqa: F401


def query(*args):
    from fms_mo_amd import _lib as L

    return L.load().fmsmo_paged_attn_workspace_bytes(*args)


def test_a_window_is_planned_for(p):  # noqa: F811
    """A call with a window needs the workspace of what a tile of rows goes through, not that of the whole cache: with so many bytes it gets as
    far as their alignment, with one less it does not.  40 rows behind 65536 keys, 4 + 2 heads of 64."""
    from fms_mo_amd import _lib as L

    big = rules.batch_struct(p, table_width=4096, query_start=p, seqs=1)
    for window, sinks, keys in ((1024, 4, 1068), (4000, 500, 4540), (100, 0, 140), (1, 0, 41), (1 << 40, 0, 65536), (70000, 1 << 50, 65536), (0, 5, 65536)):
        need = query(4, 2, 64, L.F16, 1, 40, 40, min(keys, 65536))
        call = lambda n: rules.attend(p, batch=big, rows=40, max_rows=40, max_keys=65536, window=window, sinks=sinks, ws=p + 8, nbytes=n)  # noqa: E731
        assert call(need) == ALIGN
        if need:
            assert call(need - 1) == SCRATCH
    assert query(4, 2, 64, L.F16, 1, 40, 40, 1068) < query(4, 2, 64, L.F16, 1, 40, 40, 65536) / 10


def test_fewer_keys_never_need_more():
    from fms_mo_amd import _lib as L

    rng = random.Random(0)
    for _ in range(2000):
        kv = rng.choice([1, 2, 8])
        heads = kv * rng.choice([1, 4, 8, 20])
        seqs = rng.choice([1, 3, 64, 300])
        rows = seqs * rng.choice([1, 2, 5, 40, 500])
        most = min(rows, rng.choice([1, 2, 5, 40, 500]))
        keys = sorted(int(2 ** rng.uniform(0, 21)) for _ in range(2))
        args = (heads, kv, rng.choice([64, 128, 256]), rng.choice([L.F16, L.KV_E4M3]), seqs, rows, most)
        assert query(*args, keys[0]) <= query(*args, keys[1]) <= 270 << 20
