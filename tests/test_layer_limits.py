"""Sizes at which calls of the operators around a layer's products are cut or refused: no GPU is needed."""
import random

import pytest
import torch

from test_layer_rules import SCRATCH, UNSUPPORTED, lib, p  # noqa: F401


@pytest.mark.parametrize("rank", [8, 32, 64, 128])
def test_sums_of_one_row_requests_fit_64_mb(lib, rank):  # noqa: F811
    for seqs in (1, 100, 8192, 8193, 70000, 1 << 20, (1 << 29) - 1):
        for K in (64, 14336):
            assert 0 < lib.fmsmo_lora_workspace_bytes(seqs, seqs, 0, 1 << 30, rank, K) <= 64 << 20


def test_adapters_of_more_tiles_than_a_launch_has_threads_for(lib, p):  # noqa: F811
    def call(rows, seqs):
        return lib.fmsmo_lora_add(0, p, 64, p, 32, p, 32, p, 1024, 64, p, 512, 16, 2, 16, p, p, seqs, None, rows, 32, 64, p, 16, None)

    assert call(4, (1 << 24) - 3) == SCRATCH and call(4, (1 << 24) - 2) == UNSUPPORTED and call(4, 1 << 28) == UNSUPPORTED
    assert call((1 << 28) - 64, 1 << 23) == UNSUPPORTED and call(1 << 28, 2) == SCRATCH and call((1 << 30) - 64, 1) == UNSUPPORTED


def test_adapters_have_no_gradients():
    """Where a gradient would be expected the call is refused (and goes on to the next check where none is)."""
    from fms_mo_amd import kernels as k

    h, ids = torch.zeros(2, 64).half(), torch.zeros(2, dtype=torch.int32)
    given = dict(y=h, x=h, a=torch.zeros(1, 8, 64).half(), b=torch.zeros(1, 64, 8).half(), scales=torch.ones(1), out=torch.zeros(2, 64).half())
    for name in given:
        d = dict(given)
        d[name] = torch.nn.Parameter(d[name])
        with pytest.raises(RuntimeError, match="no gradients"):
            k.lora_add(adapters=ids, **d)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            k.lora_add(adapters=ids, **d)
    with pytest.raises(RuntimeError, match="no CPU path"):
        k.lora_add(adapters=ids, **given)


@pytest.mark.parametrize("T,E,top,K,I,blocks", [(16, 2, 2, 2048, 16384, 2), (16, 8, 8, 2048, 7168, 2), (12, 8, 6, 2048, 5632, 2), (64, 64, 6, 2048, 1408, 2),
                                                (10, 4, 4, 2048, 5632, 2), (64, 128, 8, 2048, 768, 1), (32, 32, 4, 2048, 2048, 1), (8, 4, 4, 2048, 5632, 1)])
def test_experts_of_more_than_eight_tokens(lib, T, E, top, K, I, blocks):  # noqa: F811
    """The down product's blocks of eight outputs read an expert's weights for every eight of its tokens.  Where that is more than once for most
    experts, blocks of sixteen go two for the same outputs, whose sums need room in the workspace."""
    rest = 5 * T * top * I + T * top * I // 2 + 24 * T * top + 8192  # codes, h, its maxima, numbers of a choice, groups
    n = lib.fmsmo_moe_few_workspace_bytes(T, E, top, K, I)
    assert (n > rest) == (blocks > 1) and (blocks == 1 or n >= 4 * blocks * T * K + 5 * T * top * I)


def few(rows, seqs, ragged, rank):
    return not ragged or rows < 32 * seqs or rows < (3000 if rank >= 120 else 4096)


@pytest.mark.parametrize("rank", [8, 24, 40, 72, 128])
@pytest.mark.parametrize("K", [8, 64, 1000, 14336])
def test_lora_workspace_holds_the_tiles_of_any_starts(lib, rank, K):  # noqa: F811
    """The sums of every tile of ascending starts, rows in front of the first request and behind the last among them, for tiles of 16 rows and
    of 64; with one step of K they are all that there is."""
    r, padded = random.Random(rank), 16 if rank <= 16 else 32 if rank <= 32 else 64 if rank <= 64 else 128
    seen = set()
    for rows, seqs in ((1, 1), (1, 3), (5, 700), (100, 2), (2047, 1), (2999, 2), (3000, 2), (4095, 1), (4096, 1), (4096, 128), (4096, 129), (8192, 1),
                       (8192, 256), (8192, 257), (50000, 3)):
        tile = 16 if few(rows, seqs, True, rank) else 64
        seen.add(tile)
        n = lib.fmsmo_lora_workspace_bytes(rows, seqs, 1, 3, rank, K)
        assert n % 16 == 0
        if K <= 64:
            assert n == 4 * padded * tile * (rows // tile + seqs + 2)
        for _ in range(20):
            at = sorted(r.randint(0, rows) for _ in range(seqs + 1))
            tiles = sum(-(-(b - a) // tile) for a, b in zip([0] + at, at + [rows]))
            assert n >= 4 * padded * tile * tiles
    assert seen == {16, 64}


@pytest.mark.parametrize("rank", [8, 24, 40, 128])
def test_lora_workspace_of_one_row_requests(lib, rank):  # noqa: F811
    padded = 16 if rank <= 16 else 32 if rank <= 32 else 64 if rank <= 64 else 128
    for rows in (1, 7, 100, 8192):
        assert lib.fmsmo_lora_workspace_bytes(rows, rows, 0, 3, rank, 64) == 4 * padded * 16 * rows
