"""CPU tests of the paged 8-bit cache: the C entry points refuse bad arguments
before any CUDA call, and the tests' own model keeps its invariants."""
import ctypes

import numpy as np
import pytest

from tests.kv8_ref import RefCache, quantise_block


def fake(**kw):
    from stealcode_b200.kv8 import _Cache

    buf = np.zeros(4096, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    c = _Cache(p, p, p, p, p, p, p, p, 1, 4, 2, 4, 2, 64, 32, 16)
    for k, v in kw.items():
        setattr(c, k, v)
    c._keep = buf
    return c, p


def call(c, p, **kw):
    from stealcode_b200._lib import lib
    from stealcode_b200.kv8 import _Batch

    b = _Batch(None, None, kw.pop("m", 2), kw.pop("n", 1), kw.pop("total", 2))
    if "cu" in kw:
        b.cu = kw.pop("cu")
    a = dict(layer=0, q=p, heads=4, window=0, sinks=0, out=p, dtype=0, lse=None)
    a.update(kw)
    return lib.sc_kv8_attend(ctypes.byref(c), a["layer"], ctypes.byref(b), a["q"], 256, 64, a["heads"], 0.125,
                             a["window"], a["sinks"], 0, a["out"], 256, 64, a["lse"], a["dtype"], None, 0, None)


@pytest.mark.parametrize("kw", [dict(k=None), dict(status=None), dict(k=8), dict(table=2), dict(n_layers=0),
                                dict(n_pages=0), dict(n_seqs=-1), dict(max_pages=1 << 40), dict(n_kv_heads=0),
                                dict(n_pages=1 << 33), dict(n_seqs=1 << 30, max_pages=1 << 20)])
def test_caches_are_refused(kw):
    from stealcode_b200 import _lib

    c, p = fake()
    for k, v in kw.items():
        setattr(c, k, p + v if k in ("k", "table") and v is not None else v)
    assert call(c, p) == _lib.SC_ERR_INVALID
    assert _lib.lib.sc_kv8_compact(ctypes.byref(c), None, 0, None) == _lib.SC_ERR_INVALID
    assert "kv8" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(head_dim=32), dict(head_dim=80), dict(head_dim=256), dict(block=8), dict(block=48),
                                dict(page=24), dict(page=8), dict(page=2048), dict(page=0)])
def test_shapes_outside_the_kernels_are_unsupported(kw):
    from stealcode_b200 import _lib

    c, p = fake(**kw)
    assert call(c, p) == _lib.SC_ERR_UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(layer=1), dict(layer=-1), dict(q=None), dict(out=None), dict(heads=3),
                                dict(heads=0), dict(window=-1), dict(sinks=-2), dict(dtype=7), dict(m=-1), dict(n=-1),
                                dict(total=3), dict(m=3, total=3), dict(m=2, n=1 << 30, total=1 << 31)])
def test_calls_are_refused(kw):
    from stealcode_b200 import _lib

    c, p = fake()
    assert call(c, p, **kw) == _lib.SC_ERR_INVALID


def test_other_entries_refuse_and_empty_calls_pass():
    from stealcode_b200 import _lib
    from stealcode_b200._lib import lib
    from stealcode_b200.kv8 import _Batch

    c, p = fake()
    r = ctypes.byref(c)
    b = _Batch(None, None, 2, 1, 2)
    assert lib.sc_kv8_append(r, 0, ctypes.byref(b), None, 128, 64, p, 128, 64, 0, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_append(r, 0, ctypes.byref(b), p, 128, 64, p, 128, 64, 9, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_append(r, 0, None, p, 128, 64, p, 128, 64, 0, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_append(None, 0, ctypes.byref(b), p, 128, 64, p, 128, 64, 0, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_rows(r, 2, ctypes.byref(b), p, p, 0, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_rows(r, 0, ctypes.byref(b), p + 4, p, 0, None) == _lib.SC_ERR_INVALID
    need = lib.sc_kv8_page_workspace_bytes(r)
    assert need > 0 and lib.sc_kv8_page_workspace_bytes(None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_reserve(r, None, p, 2, p, need - 1, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_reserve(r, None, p, 2, p + 16, need, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_reserve(r, None, None, 2, p, need, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_reserve(r, None, p, 3, p, need, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_fork(r, p, None, 1, p, need, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_release(r, None, -1, None) == _lib.SC_ERR_INVALID
    assert lib.sc_kv8_slide(r, None, 2, 0, 0, None) == _lib.SC_ERR_INVALID
    empty = _Batch(None, None, 0, 0, 0)
    assert lib.sc_kv8_append(r, 0, ctypes.byref(empty), None, 0, 0, None, 0, 0, 0, None) == _lib.SC_OK
    assert lib.sc_kv8_rows(r, 0, ctypes.byref(empty), None, None, 0, None) == _lib.SC_OK
    assert lib.sc_kv8_release(r, None, 0, None) == _lib.SC_OK
    assert lib.sc_kv8_reserve(r, None, None, 0, p, need, None) == _lib.SC_OK


def test_block_quantiser_error():
    """Fresh values are within half a step (and f32 rounding) of what they stand for; a value that was
    rounded again because its block grew, within one more half step of the new scale."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, 64)).astype(np.float32)
    c, s = quantise_block(np.zeros((0, 64), np.int8), 0.0, x[:9])
    assert np.abs(c * np.float64(s) - x[:9]).max() <= s * (0.5 + 1e-4)
    c, s2 = quantise_block(c, s, x[9:] * 3)
    assert s2 > s
    assert np.abs(c[:9] * np.float64(s2) - x[:9]).max() <= s2 * (0.5 + 1e-4) + s * (0.5 + 1e-4)


def test_model_counts_follow_its_tables():
    rng = np.random.default_rng(2)
    r = RefCache(1, 20, 1, 64, 5, 6, 16, 16)
    for _ in range(200):
        op, m = rng.integers(0, 5), int(rng.integers(1, 4))
        seqs = rng.permutation(5)[:m].tolist()
        if op == 0:
            r.reserve(seqs, rng.integers(0, 40, m).tolist())
        elif op == 1:
            r.fork(rng.integers(0, 5, m).tolist(), seqs)
        elif op == 2:
            r.release(seqs[:1])
        elif op == 3:
            r.slide(int(rng.integers(1, 40)), int(rng.integers(0, 40)), seqs)
        else:
            r.compact()
            assert not r.refs[int((r.refs > 0).sum()):].any()
        assert np.array_equal(np.bincount(r.table[r.table >= 0], minlength=20), r.refs)
