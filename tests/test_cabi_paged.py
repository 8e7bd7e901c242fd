"""Host-side contract of the C entry points for positions and the paged cache: struct layouts, workspaces, refusals.  Nothing
here reaches a GPU: every refusal comes before one is looked for."""

import ctypes

import pytest

from flashbob_b200 import _lib

FAKE = 0x10000                                       # an aligned address that is never read


def _cache(bits=16, D=128, pages=100, heads=8, page=64):
    c = _lib.Cache(pages=pages, heads=heads, page_size=page, D=D, dtype=_lib.BF16, bits=bits, device=0)
    row = D * bits // 8
    for w in range(2):
        c.data[w] = FAKE
        c.strides[w][:] = (heads * page * row, page * row, row)
        if bits == 4:
            c.scales[w] = FAKE
            c.scale_strides[w][:] = (heads * page * 8, page * 8, 8)
    return c


def _sequences(B=4, max_pages=64):
    return _lib.Sequences(B=B, max_pages=max_pages, table=FAKE, table_stride=max_pages, lengths=FAKE)


def _paged(N=1, Hq=32, **kw):
    seq = {k: kw.pop(k) for k in ("B", "max_pages") if k in kw}
    a = _lib.PagedArgs(cache=_cache(**kw), seq=_sequences(**seq), Hq=Hq, N=N, is_causal=1, q=FAKE, out=FAKE, scale=0.1)
    a.rotary.pairs, a.rotary.factor = a.cache.D // 2, 1.0
    a.q_strides[:] = (Hq * N * a.cache.D, N * a.cache.D, a.cache.D)
    return a


def test_struct_layouts():
    assert ctypes.sizeof(_lib.Rotary) == 8 + 8 + 64 * 8
    assert ctypes.sizeof(_lib.Cache) == 32 + 16 + 48 + 16 + 48
    assert ctypes.sizeof(_lib.Sequences) == 8 + 8 + 8 + 8 + 8
    assert ctypes.sizeof(_lib.PagedArgs) == 160 + 40 + 528 + 16 + 8 + 24 + 8 + 8
    assert ctypes.sizeof(_lib.RotateArgs) == 32 + 16 + 48 + 16 + 8 + 16 + 8 + 8 + 528


@pytest.mark.parametrize("kw", [dict(), dict(bits=4), dict(N=4), dict(N=1024), dict(N=131072, max_pages=2048, B=1), dict(N=131072, max_pages=2048, B=1, bits=4),
                                dict(N=8192, max_pages=4096, B=16, bits=4), dict(D=32, Hq=8), dict(N=100, bits=4)])
def test_workspaces_of_valid_calls(kw):
    lib = _lib.load()
    a = _paged(**kw)
    n = lib.bob_sm100_paged_workspace_bytes(ctypes.byref(a))
    assert 256 <= n < 8 << 30
    a.seq.lengths = FAKE + 4                         # (not a matter of lengths)
    assert lib.bob_sm100_paged_workspace_bytes(ctypes.byref(a)) == n


def _set(path, value):
    def change(a):
        *owners, last = path.split(".")
        for o in owners:
            a = getattr(a, o)
        if "[" in last:
            last, *at = last.replace("]", "").split("[")
            a = getattr(a, last)
            for i in at[:-1]:
                a = a[int(i)]
            a[int(at[-1])] = value
        else:
            setattr(a, last, value)
    return change


@pytest.mark.parametrize("path,value,code", [
    ("cache.dtype", 2, -3), ("cache.D", 48, -4), ("cache.pages", 0, -2), ("cache.heads", 0, -2), ("cache.page_size", 24, -2), ("cache.page_size", 8, -2),
    ("cache.page_size", 8192, -2), ("cache.bits", 8, -2), ("cache.data[0]", None, -1), ("cache.data[1]", FAKE + 8, -10), ("cache.strides[0][2]", 24, -5),
    ("cache.strides[1][0]", -256, -5), ("seq.B", 0, -2), ("seq.max_pages", 0, -2), ("seq.max_pages", 1 << 27, -2), ("seq.table", None, -1),
    ("seq.lengths", None, -1), ("seq.table_stride", -1, -2), ("rotary.pairs", 65, -2), ("rotary.pairs", -1, -2), ("rotary.factor", float("nan"), -2),
    ("Hq", 0, -2), ("Hq", 12, -2), ("N", 0, -2), ("window", -1, -2), ("scale", 0.0, -2), ("scale", float("inf"), -2), ("q", None, -1), ("q", FAKE + 2, -10),
    ("q_strides[1]", 4, -5), ("out", None, -1), ("out", FAKE + 8, -10),
])
def test_refusals(path, value, code):
    lib = _lib.load()
    a = _paged()
    _set(path, value)(a)
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE, None) == code
    assert lib.bob_sm100_paged_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.bob_sm100_error_string(code)
    if path.split(".")[0] in ("cache", "seq", "rotary"):
        strides = (ctypes.c_int64 * 3)(1024, 128, 128)
        args = (ctypes.byref(a.cache), ctypes.byref(a.seq))
        assert lib.bob_sm100_cache_append(*args, ctypes.byref(a.rotary), 1, FAKE, strides, FAKE, strides, None) == code
        if not path.startswith("rotary"):
            assert lib.bob_sm100_cache_read(*args, 4, FAKE, FAKE, None) == code


def test_more_refusals():
    lib = _lib.load()
    a = _paged(bits=4)
    a.cache.scales[0] = None
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE, None) == -1
    a = _paged(bits=4)
    a.cache.scale_strides[1][2] = 4
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE, None) == -5
    a = _paged()
    assert lib.bob_sm100_paged_fwd(None, FAKE, None) == -1
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), None, None) == -6
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE + 16, None) == -6
    a.is_causal, a.window = 0, 5
    assert lib.bob_sm100_paged_fwd(ctypes.byref(a), FAKE, None) == -2
    r = _lib.RotateArgs(B=1, N=4, D=64, dtype=_lib.FP16, position_bits=0)
    r.heads[0], r.in_[0], r.out[0] = 2, FAKE, FAKE
    r.rotary.pairs, r.rotary.factor = 32, 1.0
    for path, value, code in [("B", 0, -2), ("N", 0, -2), ("D", 40, -4), ("dtype", 7, -3), ("heads[0]", 0, -2), ("heads[1]", -1, -2), ("heads[0]", 70000, -2),
                              ("in_[0]", None, -1), ("in_[0]", FAKE + 4, -10), ("in_strides[0][0]", 3, -5), ("out[0]", None, -1), ("out[0]", FAKE + 4, -10),
                              ("positions", FAKE, -2), ("rotary.pairs", 33, -2), ("heads[1]", 1, -1)]:
        b = _lib.RotateArgs.from_buffer_copy(r)
        _set(path, value)(b)
        assert lib.bob_sm100_rotate(ctypes.byref(b), None) == code, path
    assert lib.bob_sm100_rotate(None, None) == -1
