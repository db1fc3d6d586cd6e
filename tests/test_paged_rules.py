"""What the paged cache's entry points refuse, without a GPU: every call below is rejected before a launch, or has nothing to do."""
import ctypes

import pytest
import torch


def cache_struct(p, **kw):
    from fms_mo_amd import _lib as L

    c = L.KvCache(k=p, v=p, k_scale=p, v_scale=p, pages=4, page_size=16, heads=2, dim=64, dtype=L.F16)
    c.k_strides[:] = c.v_strides[:] = (2048, 1024, 64)
    c.k_scale_strides[:] = c.v_scale_strides[:] = (32, 16)
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


def batch_struct(p, **kw):
    from fms_mo_amd import _lib as L

    b = L.KvBatch(block_table=p, table_stride=8, table_width=8, seq_lens=p, query_start=None, seqs=3)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.fixture()
def p():
    buf = (ctypes.c_char * 4096)()
    keep.append(buf)
    return (ctypes.addressof(buf) + 15) // 16 * 16


keep = []
NULL, SHAPE, ALIGN, UNSUPPORTED, SCRATCH = 1, 2, 3, 4, 6


def attend(p, cache=None, batch=None, dtype=0, rows=3, heads=4, q=0, q_row=256, q_head=64, out=0, o_row=256, o_head=64, window=0, sinks=0, max_rows=1,
           max_keys=128, ws=0, nbytes=0):
    from fms_mo_amd import _lib as L

    c, b = cache or cache_struct(p), batch or batch_struct(p)
    return L.load().fmsmo_paged_attn(ctypes.byref(c), ctypes.byref(b), dtype, rows, heads, p if q == 0 else q, q_row, q_head, p if out == 0 else out, o_row,
                                     o_head, 1.0, window, sinks, max_rows, max_keys, 0, p if ws == 0 else ws, nbytes, None)


def store(p, cache=None, batch=None, dtype=0, rows=3, heads=4, k=0, k_row=128, cos=0, table_rows=9, rotary=64, w=0, wdt=0):
    from fms_mo_amd import _lib as L

    c, b = cache or cache_struct(p), batch or batch_struct(p)
    z = lambda x: p if x == 0 else x  # noqa: E731
    return L.load().fmsmo_kv_store(ctypes.byref(c), ctypes.byref(b), dtype, rows, heads, p, 256, 64, z(k), k_row, 64, p, 128, 64, p, 256, 64, z(w), z(w), wdt,
                                   1e-6, z(cos), z(cos), table_rows, rotary, 0, 0, None)


@pytest.mark.parametrize("call", [attend, store])
def test_c_entries_refuse(p, call):
    from fms_mo_amd import _lib as L

    C, B = (lambda **k: call(p, cache=cache_struct(p, **k))), (lambda **k: call(p, batch=batch_struct(p, **k)))
    assert C(k=None) == NULL and C(v=None) == NULL and B(block_table=None) == NULL and B(seq_lens=None) == NULL
    assert C(dtype=L.KV_E4M3, k_scale=None) == NULL
    assert C(dtype=L.F32) == UNSUPPORTED and C(dtype=L.BF16) == UNSUPPORTED and call(p, dtype=2) == UNSUPPORTED
    assert C(dim=96) == UNSUPPORTED and C(dim=32) == UNSUPPORTED
    assert C(page_size=8) == UNSUPPORTED and C(page_size=48) == UNSUPPORTED and C(page_size=1 << 17) == UNSUPPORTED and C(page_size=0) == UNSUPPORTED
    assert C(pages=0) == SHAPE and C(heads=0) == SHAPE and C(heads=3) == SHAPE and call(p, heads=0) == SHAPE and call(p, heads=3) == SHAPE
    assert B(table_width=0) == SHAPE and B(seqs=2) == SHAPE and B(seqs=-1) == SHAPE and call(p, rows=-1) == SHAPE and call(p, rows=1 << 40) == SHAPE
    assert C(k_strides=(2048, 1024, 32)) == SHAPE and C(v_strides=(-8, 1024, 64)) == SHAPE
    assert C(k_strides=(2047, 1024, 64)) == ALIGN and C(k_strides=(2048, 1024, 68)) == ALIGN and C(k=p + 8) == ALIGN and B(seq_lens=p + 2) == ALIGN
    assert C(k_strides=(2048, 1024, 1 << 30)) == UNSUPPORTED
    e = dict(dtype=L.KV_E4M3)
    assert C(k_strides=(2048, 1024, 72), **e) == ALIGN and C(k_scale_strides=(32, 15), **e) == ALIGN and C(v_scale=p + 4, **e) == ALIGN
    assert B(table_width=1 << 30) == UNSUPPORTED and C(pages=1 << 31) == UNSUPPORTED


def test_attention_refuses(p):
    assert attend(p, q=None) == NULL and attend(p, out=None) == NULL
    assert attend(p, q_row=250) == ALIGN and attend(p, o_head=4) == ALIGN and attend(p, q=p + 2) == ALIGN and attend(p, o_row=-8) == SHAPE
    assert attend(p, window=-1) == SHAPE and attend(p, sinks=-1) == SHAPE and attend(p, nbytes=-1) == SHAPE
    big = batch_struct(p, table_width=4096)
    assert attend(p, batch=big, max_keys=0) == SCRATCH and attend(p, batch=big, max_keys=65536, ws=None, nbytes=1 << 30) == SCRATCH
    assert attend(p, batch=big, max_keys=65536, ws=p + 8, nbytes=1 << 30) == ALIGN
    assert attend(p, rows=0, batch=batch_struct(p, seqs=0)) == 0


def test_store_refuses(p):
    assert store(p, k=None) == NULL and store(p, cos=None) == NULL
    assert store(p, rotary=72) == SHAPE and store(p, rotary=-16) == SHAPE and store(p, rotary=8) == UNSUPPORTED and store(p, table_rows=0) == SHAPE
    assert store(p, k_row=100) == ALIGN and store(p, k_row=-8) == SHAPE and store(p, k=p + 8) == ALIGN and store(p, cos=p + 4) == ALIGN
    assert store(p, w=p + 4) == ALIGN and store(p, wdt=1) == UNSUPPORTED
    assert store(p, rows=0, batch=batch_struct(p, seqs=0)) == 0


def test_workspace_grows_with_what_is_split():
    from fms_mo_amd import _lib as L

    f = L.load().fmsmo_paged_attn_workspace_bytes
    F16, E4M3 = L.F16, L.KV_E4M3
    assert f(4, 2, 128, F16, 3, 3, 1, 64) == 0              # one launch
    n = f(4, 2, 128, F16, 3, 3, 1, 100000)
    assert n > 0 and n % 16 == 0 and n > f(4, 2, 64, F16, 3, 3, 1, 100000) > 0 and n == f(4, 2, 128, F16, 3, 3, 1, 200000)
    assert f(4, 2, 128, F16, 1, 20000, 20000, 20000) == 0   # prompts: tiles of rows enough for the chip
    m = f(4, 2, 128, F16, 1, 100, 100, 100000)              # a few tokens behind many: several blocks for a tile of rows
    assert m > 0 and m % 16 == 0 and m < 1 << 28
    assert f(64, 8, 256, E4M3, 300, 400, 200, 1 << 20) < 1 << 30
    assert f(3, 2, 128, F16, 3, 3, 1, 100) == 0 and f(0, 0, 128, F16, 0, 0, 0, 0) == 0


def meta(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_wrappers_refuse_before_a_launch(monkeypatch):
    from fms_mo_amd import kernels as K

    with pytest.raises(RuntimeError, match="no CPU path"):
        K.paged_attention(meta(1, 4, 64), meta(2, 2, 16, 64), meta(2, 2, 16, 64), meta(1, 2, dtype=torch.int32), meta(1, dtype=torch.int32))
    # the checks themselves, with the one for the device set aside and nothing launched
    monkeypatch.setattr(K, "_need_gpu", lambda *t: None)
    monkeypatch.setattr(K, "_stream", lambda t: None)
    monkeypatch.setattr(K, "_dev", lambda t: K._NO_SWITCH)

    def launched(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(K.L, "call", launched)
    i32 = torch.int32

    def attend(q=None, k=None, v=None, table=None, lens=None, **kw):
        z = lambda x, *s, **d: x if x is not None else meta(*s, **d)  # noqa: E731
        K.paged_attention(z(q, 2, 4, 64), z(k, 3, 2, 16, 64), z(v, 3, 2, 16, 64), z(table, 2, 2, dtype=i32), z(lens, 2, dtype=i32), **kw)
    bad = [
        dict(q=meta(2, 256)), dict(q=meta(2, 3, 64)), dict(q=meta(2, 4, 128)), dict(q=meta(2, 4, 64, dtype=torch.float32)), dict(q=meta(2, 4, 64, dtype=torch.bfloat16)),
        dict(q=meta(3, 4, 64)), dict(k=meta(3, 2, 16, 128)), dict(k=meta(3, 2, 24, 64), v=meta(3, 2, 24, 64)), dict(k=meta(3, 16, 128)),
        dict(k=meta(3, 2, 8, 64), v=meta(3, 2, 8, 64)), dict(k=meta(3, 2, 64, 16).transpose(2, 3)), dict(k=meta(3, 2, 16, 96), v=meta(3, 2, 16, 96), q=meta(2, 4, 96)),
        dict(k=meta(3, 2, 16, 68)[..., 4:]), dict(table=meta(2, 2, dtype=torch.int64)), dict(table=meta(3, 2, dtype=i32)), dict(table=meta(2, 0, dtype=i32)),
        dict(lens=meta(2, dtype=torch.int64)), dict(query_start=meta(2, dtype=i32)), dict(query_start=meta(3, dtype=torch.int64)),
        dict(window=-1), dict(sinks=-2), dict(max_query_len=-1), dict(max_seq_len=-1), dict(k_scale=meta(3, 2, 16, dtype=torch.float32)),
        dict(k=meta(3, 2, 16, 64, dtype=torch.float8_e4m3fn), v=meta(3, 2, 16, 64, dtype=torch.float8_e4m3fn)),
        dict(k=meta(3, 2, 16, 64, dtype=torch.int8), v=meta(3, 2, 16, 64, dtype=torch.int8)),
        dict(out=meta(2, 4, 32)), dict(out=meta(2, 4, 64, dtype=torch.bfloat16)), dict(out=meta(1, 4, 64).expand(2, 4, 64)),
        dict(k=meta(3, 2, 16, 64, dtype=torch.float8_e4m3fn), v=meta(3, 2, 16, 64, dtype=torch.float8_e4m3fn), k_scale=meta(3, 2, 16), v_scale=meta(3, 2, 16)),
    ]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            attend(**kw)

    def store(q=None, k=None, v=None, kc=None, **kw):
        z = lambda x, *s, **d: x if x is not None else meta(*s, **d)  # noqa: E731
        K.qk_norm_rope_store(z(q, 2, 4, 64), z(k, 2, 2, 64), z(v, 2, 2, 64), z(kc, 3, 2, 16, 64), meta(3, 2, 16, 64), meta(2, 2, dtype=i32), meta(2, dtype=i32), **kw)
    f32 = torch.float32
    bad = [
        dict(k=meta(2, 4, 64)), dict(v=meta(3, 2, 64)), dict(k=meta(2, 2, 64, dtype=torch.bfloat16)), dict(kc=meta(1, 2, 16, 64).expand(3, 2, 16, 64)),
        dict(cos=meta(9, 32, dtype=f32)), dict(cos=meta(9, 32), sin=meta(9, 32)), dict(cos=meta(9, 64, dtype=f32), sin=meta(9, 64, dtype=f32)),
        dict(cos=meta(9, 4, dtype=f32), sin=meta(9, 4, dtype=f32)), dict(cos=meta(0, 32, dtype=f32), sin=meta(0, 32, dtype=f32)),
        dict(cos=meta(9, 32, dtype=f32), sin=meta(8, 32, dtype=f32)), dict(q_weight=meta(32)), dict(q_weight=meta(64, dtype=torch.bfloat16)),
        dict(q_weight=meta(64), k_weight=meta(64, dtype=f32)),
    ]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            store(**kw)
    with pytest.raises(AssertionError, match="launched"):  # (what is right gets as far as the launch)
        store()


def test_cache_refuses_other_types():
    from fms_mo_amd.modules.attention import PagedKVCache

    with pytest.raises(TypeError):
        PagedKVCache(4, 16, 2, 64, torch.int8, device="cpu")
    c = PagedKVCache(4, 16, 2, 64, torch.float8_e4m3fn, device="cpu")
    assert c.k_scale.shape == (4, 2, 16) and PagedKVCache(4, 16, 2, 64, device="cpu").k_scale is None
