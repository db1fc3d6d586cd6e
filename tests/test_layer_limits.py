"""Sizes at which calls of the operators around a layer's products are cut or refused: no GPU is needed."""
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
