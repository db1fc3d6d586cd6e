"""Sizes at which calls of the operators around a layer's products are cut or refused: no GPU is needed."""
import pytest

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
