"""Paged cache operators: what they refuse before any device work (no GPU
needed: the pointers are never followed), and the host-side rotation table."""
import ctypes as C

import numpy as np
import pytest

P = 1 << 20  # a 16-byte aligned address that is never read


def desc(tirlib, **kw):
    """A cache description that passes every check, changed by kw."""
    f = dict(k=P, v=P, k_scale=P, v_scale=P, table=P, table_rows=4, table_stride=8, n_pages=32, page_stride=16 * 4 * 64,
             pos_stride=4 * 64, head_stride=64, max_pages=8, page_size=16, kv_heads=4, dim=64, dtype=0)
    f.update(kw)
    return tirlib.KVPagesDesc(**f)


def norm(tirlib, **kw):
    f = dict(q_weight=P, k_weight=P, rope=P, rope_positions=128, rope_dim=64, pairs=0, eps=1e-5)
    f.update(kw)
    return tirlib.QKNorm(**f)


def attention(tirlib, d, q=P, q_stride=8 * 64, lens=P, out=P, out_stride=8 * 64, rows=4, q_heads=8, dtype=0, scale=0.0,
              max_len=0, window=0, ws=P, ws_bytes=1 << 30):
    tirlib.check(tirlib.lib().tir_paged_attention(q, q_stride, C.addressof(d) if d else None, lens, out, out_stride, rows,
                                                  q_heads, dtype, scale, max_len, window, ws, ws_bytes, None))


def append(tirlib, d, k=P, k_stride=256, v=P, v_stride=256, seqs=P, pos=P, tokens=4, dtype=0):
    tirlib.check(tirlib.lib().tir_kv_append(C.addressof(d) if d else None, k, k_stride, v, v_stride, seqs, pos, tokens,
                                            dtype, None))


def gather(tirlib, d, k=P, k_stride=256, v=P, v_stride=256, seqs=P, pos=P, tokens=4, dtype=0):
    tirlib.check(tirlib.lib().tir_kv_gather(C.addressof(d) if d else None, k, k_stride, v, v_stride, seqs, pos, tokens,
                                            dtype, None))


def fused(tirlib, d, n, q=P, q_stride=512, k=P, v=P, kv_stride=256, q_out=P, seqs=P, pos=P, tokens=4, q_heads=8, dtype=0):
    tirlib.check(tirlib.lib().tir_qk_norm_rope_append(q, q_stride, k, kv_stride, v, kv_stride, q_out, q_stride,
                                                      C.addressof(d), seqs, pos, tokens, q_heads, dtype,
                                                      C.addressof(n) if n else None, None))


def norm_rope(tirlib, n, q=P, q_stride=512, k=P, k_stride=256, q_out=P, k_out=P, pos=P, tokens=4, q_heads=8, kv_heads=4,
              dim=64, dtype=0):
    tirlib.check(tirlib.lib().tir_qk_norm_rope(q, q_stride, k, k_stride, q_out, q_stride, k_out, k_stride, pos, tokens,
                                               q_heads, kv_heads, dim, dtype, C.addressof(n) if n else None, None))


def refused(tirlib, name, fn, *a, **kw):
    with pytest.raises(tirlib.TirError) as e:
        fn(tirlib, *a, **kw)
    assert e.value.name == name, str(e.value)
    assert "tir_" in e.value.message  # names the entry point


CACHES = [("INVALID_ARG", dict(k=None)), ("INVALID_ARG", dict(v=None)), ("INVALID_ARG", dict(table=None)),
          ("INVALID_ARG", dict(dtype=8, k_scale=None)), ("INVALID_ARG", dict(dtype=8, v_scale=None)),
          ("UNSUPPORTED_DTYPE", dict(dtype=2)), ("UNSUPPORTED_SHAPE", dict(dim=96)), ("UNSUPPORTED_SHAPE", dict(dim=0)),
          ("INVALID_ARG", dict(kv_heads=0)), ("INVALID_ARG", dict(page_size=0)), ("INVALID_ARG", dict(max_pages=0)),
          ("INVALID_ARG", dict(table_stride=7)), ("INVALID_ARG", dict(n_pages=0)), ("INVALID_ARG", dict(n_pages=1 << 31)),
          ("UNSUPPORTED_SHAPE", dict(max_pages=1 << 20, table_stride=1 << 20, page_size=1 << 12)),
          ("INVALID_ARG", dict(pos_stride=258)), ("INVALID_ARG", dict(head_stride=-64)),
          ("INVALID_ARG", dict(dtype=1, head_stride=68)), ("INVALID_ARG", dict(dtype=8, pos_stride=4 * 64 + 32)),
          ("INVALID_ARG", dict(k=P + 4)), ("INVALID_ARG", dict(dtype=8, v_scale=P + 2))]


@pytest.mark.parametrize("name,kw", CACHES, ids=[str(i) for i in range(len(CACHES))])
def test_bad_caches_are_refused_by_every_entry(tirlib, name, kw):
    d = desc(tirlib, **kw)
    refused(tirlib, name, attention, d)
    refused(tirlib, name, append, d)
    refused(tirlib, name, gather, d)
    refused(tirlib, name, fused, d, norm(tirlib))
    assert tirlib.lib().tir_paged_attention_workspace(C.addressof(d), 4, 8, 0, 0) == -1


def test_attention_refusals(tirlib):
    d = desc(tirlib)
    refused(tirlib, "INVALID_ARG", attention, None)
    refused(tirlib, "INVALID_ARG", attention, d, q=None)
    refused(tirlib, "INVALID_ARG", attention, d, out=None)
    refused(tirlib, "INVALID_ARG", attention, d, lens=None)
    refused(tirlib, "INVALID_ARG", attention, d, rows=5)          # the table has four
    refused(tirlib, "INVALID_ARG", attention, d, rows=-1)
    refused(tirlib, "INVALID_ARG", attention, d, q_heads=6)       # not a multiple of four
    refused(tirlib, "INVALID_ARG", attention, d, q_heads=0)
    refused(tirlib, "INVALID_ARG", attention, d, q_stride=8 * 64 - 4)
    refused(tirlib, "INVALID_ARG", attention, d, q_stride=8 * 64 + 2)
    refused(tirlib, "INVALID_ARG", attention, d, q=P + 8)
    refused(tirlib, "INVALID_ARG", attention, d, window=-1)
    refused(tirlib, "INVALID_ARG", attention, d, max_len=-1)
    refused(tirlib, "INVALID_ARG", attention, d, scale=float("nan"))
    refused(tirlib, "INVALID_ARG", attention, d, scale=-1.0)
    refused(tirlib, "INVALID_ARG", attention, d, scale=float("inf"))
    refused(tirlib, "UNSUPPORTED_DTYPE", attention, d, dtype=8)
    refused(tirlib, "UNSUPPORTED_DTYPE", attention, d, dtype=1)   # f16 queries, f32 cache
    refused(tirlib, "UNSUPPORTED_DTYPE", attention, desc(tirlib, dtype=30), dtype=1)
    attention(tirlib, d, rows=0, q=None, out=None, lens=None)     # nothing to do is no error


def test_row_operator_refusals(tirlib):
    d, n = desc(tirlib), norm(tirlib)
    for fn in (append, gather):
        refused(tirlib, "INVALID_ARG", fn, None)
        refused(tirlib, "INVALID_ARG", fn, d, k=None)
        refused(tirlib, "INVALID_ARG", fn, d, v=None)
        refused(tirlib, "INVALID_ARG", fn, d, pos=None)
        refused(tirlib, "INVALID_ARG", fn, d, tokens=-1)
        refused(tirlib, "INVALID_ARG", fn, d, seqs=None, tokens=5)
        refused(tirlib, "INVALID_ARG", fn, d, k_stride=252)
        refused(tirlib, "INVALID_ARG", fn, d, v=P + 4)
        refused(tirlib, "UNSUPPORTED_DTYPE", fn, d, dtype=8)
        fn(tirlib, d, tokens=0, k=None, v=None, pos=None)
    refused(tirlib, "INVALID_ARG", fused, d, None)
    refused(tirlib, "INVALID_ARG", fused, d, n, q=None)
    refused(tirlib, "INVALID_ARG", fused, d, n, q_out=None)
    refused(tirlib, "INVALID_ARG", fused, d, n, q_heads=-1)
    refused(tirlib, "INVALID_ARG", fused, d, norm(tirlib, pairs=2))
    refused(tirlib, "UNSUPPORTED_SHAPE", norm_rope, n, dim=80)
    refused(tirlib, "UNSUPPORTED_DTYPE", norm_rope, n, dtype=3)
    refused(tirlib, "INVALID_ARG", norm_rope, None)
    refused(tirlib, "INVALID_ARG", norm_rope, n, pos=None)
    refused(tirlib, "INVALID_ARG", norm_rope, n, k_out=None)
    refused(tirlib, "INVALID_ARG", norm_rope, n, tokens=-3)
    refused(tirlib, "UNSUPPORTED_SHAPE", norm_rope, norm(tirlib, rope_dim=24))
    refused(tirlib, "UNSUPPORTED_SHAPE", norm_rope, norm(tirlib, rope_dim=128))
    refused(tirlib, "INVALID_ARG", norm_rope, norm(tirlib, rope_positions=0))
    refused(tirlib, "INVALID_ARG", norm_rope, norm(tirlib, eps=-1.0))
    refused(tirlib, "INVALID_ARG", norm_rope, norm(tirlib, eps=float("nan")))
    norm_rope(tirlib, n, tokens=0, q=None, k=None, q_out=None, k_out=None, pos=None)


@pytest.mark.parametrize("base,dim,n", [(10000.0, 64, 40), (500000.0, 128, 3), (10000.0, 2, 1), (10000.0, 64, 0)])
def test_rope_table_is_cos_and_sin_of_rope_angles(tirlib, base, dim, n):
    """Bit-equal to cosf / sinf of rope_angles: both are the same libm calls, so
    the angles are compared exactly and the table within half a step of f32
    (2^-24 relative) plus libm's own error (below one step)."""
    t = tirlib.rope_table(base, dim, n)
    assert t.shape == (n, dim // 2, 2)
    for pos in range(n):
        a = tirlib.rope_angles(base, pos, dim).astype(np.float64)
        np.testing.assert_allclose(t[pos, :, 0], np.cos(a), rtol=0, atol=1.5 * 2.0 ** -24)
        np.testing.assert_allclose(t[pos, :, 1], np.sin(a), rtol=0, atol=1.5 * 2.0 ** -24)


def test_rope_table_refusals(tirlib):
    for base, dim, n in [(1e4, 63, 4), (1e4, 0, 4), (1e4, 64, -1)]:
        assert tirlib.lib().tir_rope_table(base, dim, n, None) == 23
    assert tirlib.lib().tir_rope_table(1e4, 64, 4, None) == 23


def test_bindings_refuse_what_the_library_cannot_see(tirlib):
    torch = pytest.importorskip("torch")
    pool = torch.zeros(4, 16, 2, 64)
    table = torch.zeros(2, 2, dtype=torch.int32)
    for bad in [dict(k=pool, v=pool[:2], table=table), dict(k=pool, v=pool.half(), table=table),
                dict(k=pool.transpose(2, 3), v=pool.transpose(2, 3), table=table),
                dict(k=pool, v=pool, table=table.long()), dict(k=pool, v=pool, table=table[0]),
                dict(k=pool.to(torch.int8), v=pool.to(torch.int8), table=table),
                dict(k=pool, v=pool, table=table, k_scale=pool.half(), v_scale=pool.half()),
                dict(k=pool, v=pool, table=table)]:  # on the CPU
        with pytest.raises(tirlib.TirError) as e:
            tirlib.KVPages(**bad)
        assert e.value.name == "INVALID_ARG"
    with pytest.raises(tirlib.TirError) as e:
        tirlib.KVPages(pool.double(), pool.double(), table)
    assert e.value.name == "UNSUPPORTED_DTYPE"
    with pytest.raises(tirlib.TirError):
        tirlib.qk_norm_rope(pool[0], pool[0], pool[0], pool[0], table[0])
