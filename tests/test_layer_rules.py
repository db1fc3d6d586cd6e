"""Argument checks and workspace sizes of the operators around a layer's products: rejected before any launch, so no GPU is needed."""
import ctypes
import random

import pytest
import torch

NULL, SHAPE, ALIGN, UNSUPPORTED, SCRATCH = 1, 2, 3, 4, 6


@pytest.fixture(scope="module")
def lib():
    from fms_mo_amd import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 65536)()
    at = (ctypes.addressof(buf) + 63) // 64 * 64
    lib_keeps = buf  # noqa: F841
    yield at


def test_norm(lib, p):
    def call(**k):
        d = dict(x=p, dtype=1, ldx=64, residual=p, ldr=64, weight=p, wdt=1, eps=1e-6, codes=0, static=0, q=p, ldq=64, scale=p, ro=p, ldo=64, n=None,
                 ldn=0, M=2, K=64, stream=None)
        d.update(k)
        return lib.fmsmo_add_rms_norm_quant(*d.values())

    assert call(M=0) == 0 and call(K=0) == 0
    for name in ("x", "weight", "q", "scale"):
        assert call(**{name: None}) == NULL
    assert call(residual=None) == NULL  # residual_out without a residual
    assert call(M=-1) == SHAPE and call(K=-8) == SHAPE
    for ld in ("ldx", "ldr", "ldo", "ldq"):
        assert call(**{ld: 56}) == SHAPE and call(**{ld: 68}) == ALIGN
    assert call(n=p, ldn=56) == SHAPE
    assert call(K=60) == ALIGN
    for at in ("x", "residual", "weight", "ro"):
        assert call(**{at: p + 8}) == ALIGN
    assert call(q=p + 4) == ALIGN and call(scale=p + 2) == ALIGN
    assert call(dtype=2) == UNSUPPORTED and call(wdt=0) == UNSUPPORTED and call(codes=2) == UNSUPPORTED
    assert call(M=1 << 31) == UNSUPPORTED


def test_lora(lib, p):
    size = lib.fmsmo_lora_workspace_bytes(4, 4, 0, 2, 16, 64)
    assert 0 < size < 65536

    def call(**k):
        d = dict(dtype=0, x=p, ldx=64, y=p, ldy=32, out=p, ldo=32, a=p, a_slot=1024, a_row=64, b=p, b_slot=512, b_row=16, slots=2, rank=16, ids=p,
                 start=None, seqs=4, scales=None, rows=4, N=32, K=64, ws=p, bytes=size, stream=None)
        d.update(k)
        return lib.fmsmo_lora_add(*d.values())

    assert call(rows=0) == 0 and call(N=0) == 0
    for name in ("x", "y", "out", "a", "b", "ids", "ws"):
        assert call(**{name: None}) == NULL
    assert call(seqs=3) == SHAPE and call(rows=-1) == SHAPE and call(slots=-1) == SHAPE
    for ld in (dict(ldx=56), dict(ldy=24), dict(ldo=24), dict(a_row=56), dict(b_row=8), dict(a_slot=-8)):
        assert call(**ld) == SHAPE
    for ld in (dict(ldx=68), dict(ldy=36), dict(ldo=36), dict(a_row=68), dict(b_row=20), dict(a_slot=1028), dict(K=60), dict(N=28), dict(x=p + 8), dict(ws=p + 8)):
        assert call(**ld) == ALIGN
    for bad in (dict(rank=4), dict(rank=12), dict(rank=136), dict(dtype=2), dict(rows=1 << 30, seqs=1 << 30)):
        assert call(**bad) == UNSUPPORTED
    assert call(bytes=size - 1) == SCRATCH


@pytest.mark.parametrize("rank", [8, 24, 40, 128])
@pytest.mark.parametrize("K", [8, 64, 1000, 14336])
def test_lora_workspace_holds_every_tile(lib, rank, K):
    for rows, seqs in ((1, 1), (1, 3), (7, 7), (100, 2), (8192, 1), (8192, 256), (5, 700)):
        for ragged in (0, 1):
            if not ragged:
                seqs = rows
            n = lib.fmsmo_lora_workspace_bytes(rows, seqs, ragged, 3, rank, K)
            # a tile per 64 rows (16 where requests are short), one more per request and for the rows of none; fp32
            tile = 64 if ragged and rows >= 32 * seqs else 16
            tiles = rows // tile + seqs + 2 if ragged else seqs
            assert n % 16 == 0 and n >= 4 * tiles * tile * rank
    assert lib.fmsmo_lora_workspace_bytes(0, 4, 1, 3, rank, K) == 0 and lib.fmsmo_lora_workspace_bytes(4, 4, 0, 3, 12, K) == 0


def test_lora_workspace_of_any_sizes(lib):
    """No sizes, a caller's mistakes among them, end in anything but a number."""
    r = random.Random(1)
    for _ in range(50000):
        rows = int(2 ** r.uniform(0, 30))
        seqs = r.choice([0, 1, 2, rows // 64, rows // 33, rows, int(2 ** r.uniform(0, 29))])
        n = lib.fmsmo_lora_workspace_bytes(rows, seqs, r.randint(0, 1), int(2 ** r.uniform(0, 40)) - 1, 8 * r.randint(1, 16), 8 * int(2 ** r.uniform(0, 19)))
        assert n >= 0 and n % 16 == 0
    assert lib.fmsmo_lora_workspace_bytes(3, 0, 1, 2, 16, 64) > 0 and lib.fmsmo_lora_workspace_bytes(3, 0, 0, 2, 16, 64) == 0


def test_moe(lib, p):
    size = lib.fmsmo_moe_few_workspace_bytes(2, 4, 2, 32, 16)
    assert 0 < size < 65536

    def call(**k):
        d = dict(codes=0, a=p, lda=32, sa=p, sn=2, l=p, ldt=1, ldl=4, w13=p, s13=p, w2=p, s2=p, T=2, E=4, top=2, renorm=1, y=p, ydt=1, ldy=32, K=32,
                 I=16, ws=p, bytes=size, stream=None)
        d.update(k)
        return lib.fmsmo_moe_few_tokens(*d.values())

    assert call(T=0) == 0
    for name in ("a", "sa", "l", "w13", "s13", "w2", "s2", "y", "ws"):
        assert call(**{name: None}) == NULL
    assert call(T=-1) == SHAPE and call(sn=3) == SHAPE and call(lda=16) == SHAPE and call(ldl=3) == SHAPE and call(ldy=16) == SHAPE
    for bad in (dict(T=65), dict(E=513), dict(E=0), dict(top=0), dict(top=5), dict(top=17, E=32), dict(K=24), dict(I=24), dict(K=0), dict(codes=2),
                dict(ldt=3), dict(ydt=7), dict(K=1 << 20),
                dict(K=1 << 17, lda=1 << 17, ldy=1 << 17), dict(I=1 << 17)):
        assert call(**bad) == UNSUPPORTED
    for bad in (dict(a=p + 8), dict(w13=p + 1), dict(w2=p + 1), dict(s2=p + 4), dict(ws=p + 4), dict(lda=40)):
        assert call(**bad) == ALIGN
    assert call(bytes=size - 1) == SCRATCH


def test_moe_workspace(lib):
    for T, E, top, K, I in ((1, 1, 1, 16, 16), (64, 512, 16, 4096, 1024), (3, 7, 5, 2048, 768)):
        n = lib.fmsmo_moe_few_workspace_bytes(T, E, top, K, I)
        assert n >= T * top * I * 5 + 16 * E + 12 * T * top  # h in fp32 and as codes, an entry per expert, three numbers per choice
    assert lib.fmsmo_moe_few_workspace_bytes(65, 8, 2, 64, 64) == 0


def test_no_cpu_path():
    from fms_mo_amd import kernels as k

    h, i8 = torch.zeros(2, 64).half(), torch.zeros(2, 64, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        k.add_rms_norm_quant(h, h[0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        k.lora_add(h, h, h.view(1, 2, 64), h.view(1, 64, 2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        k.moe_few_tokens(i8, torch.ones(2), h, i8.view(1, 2, 64), torch.ones(1, 2), i8.view(1, 64, 2), torch.ones(1, 64), 1)
