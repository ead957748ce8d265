"""Refusals of the rotary and paged-chunk operators, through the C ABI: a status and nothing
launched (no GPU needed)."""

from __future__ import annotations

import ctypes as C

import pytest

OK, NULL, MODE, SHAPE, DTYPE, ALIGN, CUDA, CAPACITY = range(8)
I8, I32, F32, F16, BF16 = 0, 2, 4, 5, 6
SIZE = {I8: 1, I32: 4, F32: 4, F16: 2, BF16: 2}


@pytest.fixture(scope="module")
def L(q3):
    return q3._lib


def view(L, rows, cols, dt=F32, at=0x100000, rb=None, cb=None):
    es = SIZE[dt]
    return L.View(at, cols * es if rb is None else rb, es if cb is None else cb, rows, cols, dt)


def ref(x):
    return None if x is None else C.byref(x)


# ------------------------------------------------------------------ tables
def tables(L, spec=None, cos=None, sin=None, **kw):
    d = dict(theta=1e6, factor=2.0, original_max=4096.0, beta_fast=32.0, beta_slow=1.0,
             attn_factor=0.0, scaling=0)
    d.update(kw)
    s = L.RopeSpec(**d) if spec is None else spec
    cos = view(L, 0, 64) if cos is None else cos
    return L.lib().q3_rope_tables(C.byref(s), 0, ref(cos), ref(sin or view(L, cos.rows, cos.cols)),
                                  None)


def test_rope_tables_refuses(L):
    inf, nan = float("inf"), float("nan")
    assert tables(L) == OK                                     # no rows: nothing to do
    assert L.lib().q3_rope_tables(None, 0, None, None, None) == NULL
    assert tables(L, cos=view(L, 4, 64, at=None)) == NULL
    assert tables(L, scaling=3) == MODE and tables(L, scaling=-1) == MODE
    for bad in (dict(theta=1.0), dict(theta=inf), dict(theta=nan), dict(scaling=1, factor=0.5),
                dict(scaling=2, factor=nan), dict(scaling=2, original_max=0.0),
                dict(scaling=2, beta_slow=0.0), dict(scaling=2, beta_slow=33.0),
                dict(attn_factor=inf), dict(attn_factor=nan)):
        assert tables(L, **bad) == SHAPE, bad
    for cos in (view(L, 4, 0, rb=512), view(L, 4, 129)):
        assert tables(L, cos=cos, sin=cos) == SHAPE
    assert tables(L, cos=view(L, 4, 64), sin=view(L, 4, 32)) == SHAPE
    assert tables(L, cos=view(L, 4, 64), sin=view(L, 5, 64)) == SHAPE
    assert tables(L, cos=view(L, 4, 64, F16)) == DTYPE
    assert tables(L, cos=view(L, 4, 64, cb=8)) == SHAPE
    assert tables(L, cos=view(L, 4, 64, rb=0)) == ALIGN        # a broadcast row is no output


# -------------------------------------------------------------------- rows
def rows_call(L, **kw):
    a = dict(x=view(L, 0, 512), nw=None, pos=0x100, cos=view(L, 100, 64), sin=view(L, 100, 64),
             out=view(L, 8, 512, at=0x900000), scale=None, heads=4, hd=128)
    a.update(kw)
    return L.lib().q3_rope_rows(ref(a["x"]), ref(a["nw"]), a["pos"], ref(a["cos"]), ref(a["sin"]),
                                ref(a["out"]), ref(a["scale"]), a["heads"], a["hd"], 0,
                                0.01, None)


def test_rope_rows_refuses(L):
    v = lambda *a, **k: view(L, *a, **k)                       # noqa: E731
    assert rows_call(L) == OK
    assert rows_call(L, pos=None) == NULL and rows_call(L, cos=None) == NULL
    assert rows_call(L, sin=None) == NULL and rows_call(L, x=v(2, 512, at=None)) == NULL
    assert rows_call(L, out=None) == NULL
    for hd in (32, 96, 0, 512):
        assert rows_call(L, hd=hd, x=v(0, 4096), out=v(1, 4096)) == SHAPE
    assert rows_call(L, heads=0) == SHAPE and rows_call(L, heads=5) == SHAPE
    for half in (0, 4, 12, 72):                                # rot: not a multiple of 16; over hd
        assert rows_call(L, cos=v(100, half, rb=512), sin=v(100, half, rb=512)) == SHAPE, half
    assert rows_call(L, sin=v(99, 64)) == SHAPE
    assert rows_call(L, cos=v(100, 64, F16)) == DTYPE
    assert rows_call(L, cos=v(100, 64, at=0x100004)) == ALIGN
    assert rows_call(L, cos=v(100, 64, rb=260)) == ALIGN
    assert rows_call(L, x=v(2, 512, I8)) == DTYPE and rows_call(L, out=v(2, 512, I32)) == DTYPE
    assert rows_call(L, x=v(2, 512, at=0x100008)) == ALIGN
    assert rows_call(L, x=v(2, 512, F16, rb=1032)) == ALIGN
    assert rows_call(L, x=v(2, 512, cb=8)) == SHAPE
    assert rows_call(L, x=v(9, 512)) == SHAPE                  # more rows than out has
    assert rows_call(L, out=v(8, 512, I8)) == NULL             # codes without their scales
    assert rows_call(L, x=v(2, 512), out=v(8, 512, I8), scale=v(2, 3)) == SHAPE
    assert rows_call(L, x=v(2, 512), out=v(8, 512, I8), scale=v(1, 4)) == SHAPE
    assert rows_call(L, nw=v(1, 127)) == SHAPE and rows_call(L, nw=v(2, 64)) == SHAPE
    assert rows_call(L, nw=v(128, 1, rb=8)) == SHAPE and rows_call(L, nw=v(1, 128, F16)) == DTYPE
    x = v(2, 512, F16)
    assert rows_call(L, x=x, out=v(2, 512, BF16)) == SHAPE     # in place changes no type
    assert rows_call(L, x=x, out=v(2, 512, F16, rb=2048)) == SHAPE


# ------------------------------------------------------------------- append
def pool(L, **kw):
    d = dict(k=0x10000000, v=0x20000000, ks=0x30000000, vs=0x40000000, table=0, page_tokens=32,
             page_bytes=32 * 256, row_bytes=256, scale_page_bytes=32 * 8, scale_row_bytes=8)
    d.update(kw)
    return L.PagedKV(**d)


BAD_POOLS = [
    (dict(k=None), NULL), (dict(vs=None), NULL), (dict(page_tokens=0), SHAPE),
    (dict(page_tokens=65536), SHAPE), (dict(row_bytes=240), SHAPE),
    (dict(scale_row_bytes=4), SHAPE), (dict(page_bytes=31 * 256), SHAPE),
    (dict(scale_page_bytes=100), SHAPE), (dict(k=0x10000008), ALIGN), (dict(v=0x20000004), ALIGN),
    (dict(row_bytes=264, page_bytes=32 * 264), ALIGN), (dict(page_bytes=32 * 256 + 8), ALIGN),
    (dict(ks=0x30000002), ALIGN), (dict(scale_row_bytes=10, scale_page_bytes=320), ALIGN)]


def append_call(L, **kw):
    a = dict(k=view(L, 0, 256), v=view(L, 0, 256), nw=None, cos=None, sin=None, kv=pool(L),
             pages=100, tables=0x100, max_pages=4, row0=0x100, kv_len=0x100, seqs=2, kvh=2, hd=128)
    a.update(kw)
    return L.lib().q3_paged_kv_append_batch(
        ref(a["k"]), ref(a["v"]), ref(a["nw"]), 1.0 / 128, ref(a["cos"]), ref(a["sin"]), 0,
        ref(a["kv"]), a["pages"], a["tables"], a["max_pages"], a["row0"], a["kv_len"], a["seqs"],
        a["kvh"], a["hd"], None)


def test_append_refuses(L):
    v = lambda *a, **k: view(L, *a, **k)                       # noqa: E731
    assert append_call(L) == OK                                # no rows
    assert append_call(L, seqs=0, k=v(3, 256), v=v(3, 256)) == OK
    for name in ("tables", "row0", "kv_len", "kv", "k", "v"):
        assert append_call(L, **{name: None}) == NULL, name
    for bad, code in BAD_POOLS:
        assert append_call(L, kv=pool(L, **bad)) == code, bad
    assert append_call(L, pages=0) == SHAPE and append_call(L, pages=65537) == SHAPE
    assert append_call(L, max_pages=0) == SHAPE and append_call(L, max_pages=1 << 27) == SHAPE
    assert append_call(L, kvh=0) == SHAPE and append_call(L, kvh=3) == SHAPE
    assert append_call(L, hd=32) == SHAPE
    assert append_call(L, v=v(0, 256, F16)) == DTYPE and append_call(L, v=v(1, 256)) == SHAPE
    assert append_call(L, k=v(0, 256, I8), v=v(0, 256, I8)) == DTYPE
    assert append_call(L, k=v(0, 255)) == SHAPE
    assert append_call(L, cos=v(9, 64)) == NULL                # cos without sin
    assert append_call(L, cos=v(9, 65), sin=v(9, 65)) in (SHAPE, ALIGN)


# ---------------------------------------------------------------- attention
def attn_call(L, **kw):
    a = dict(q=view(L, 0, 512, F16), qs=None, kv=pool(L), pages=100, tables=0x100, max_pages=4,
             row0=0x100, kv_len=0x100, seqs=2, max_rows=1, o=view(L, 9, 512, F16), os=None, heads=4,
             kvh=2, hd=128, causal=1, window=0, scale=0.1, ws=None, ws_bytes=0)
    a.update(kw)
    return L.lib().q3_attention_chunk_batch(
        ref(a["q"]), ref(a["qs"]), ref(a["kv"]), a["pages"], a["tables"], a["max_pages"], a["row0"],
        a["kv_len"], a["seqs"], a["max_rows"], ref(a["o"]), ref(a["os"]), a["heads"], a["kvh"],
        a["hd"], a["causal"], a["window"], a["scale"], a["ws"], a["ws_bytes"], None)


def test_attention_refuses(L):
    v = lambda *a, **k: view(L, *a, **k)                       # noqa: E731
    assert attn_call(L) == OK and attn_call(L, seqs=0, q=v(1, 512, F16)) == OK
    for name in ("tables", "row0", "kv_len", "kv", "q", "o"):
        assert attn_call(L, **{name: None}) == NULL, name
    for bad, code in BAD_POOLS:
        assert attn_call(L, kv=pool(L, **bad)) == code, bad
    for hd in (32, 96, 256):
        assert attn_call(L, hd=hd) == SHAPE
    assert attn_call(L, heads=3) == SHAPE and attn_call(L, heads=0) == SHAPE
    assert attn_call(L, heads=34, kvh=2, q=v(0, 34 * 128, F16), o=v(0, 34 * 128, F16)) == SHAPE
    assert attn_call(L, causal=2) == MODE
    assert attn_call(L, causal=0, window=5) == SHAPE and attn_call(L, window=1 << 31) == SHAPE
    for s in (0.0, -1.0, float("nan"), float("inf")):
        assert attn_call(L, scale=s) == SHAPE
    assert attn_call(L, q=v(0, 512)) == DTYPE and attn_call(L, o=v(9, 512)) == DTYPE
    assert attn_call(L, q=v(0, 512, I8)) == NULL               # codes without scales
    assert attn_call(L, q=v(2, 512, I8), qs=v(2, 3)) == SHAPE
    assert attn_call(L, q=v(2, 512, I8), qs=v(1, 4)) == SHAPE
    assert attn_call(L, o=v(9, 512, I8)) == NULL
    assert attn_call(L, q=v(2, 512, F16), o=v(2, 512, I8), os=v(1, 4)) == SHAPE
    assert attn_call(L, q=v(10, 512, F16)) == SHAPE            # more rows than o
    assert attn_call(L, q=v(2, 500, F16, rb=1024)) == SHAPE
    assert attn_call(L, q=v(2, 512, F16, at=0x100008)) == ALIGN
    assert attn_call(L, q=v(2, 512, F16), max_rows=0) == SHAPE
    # a call whose keys are split needs its workspace
    n = L.lib().q3_attention_chunk_workspace_bytes(1, 1, 1, 4096 * 32, 4, 2, 128)
    assert n > 0
    big = dict(q=v(1, 512, F16), seqs=1, pages=5000, max_pages=4096)
    assert attn_call(L, **big) == NULL
    assert attn_call(L, **big, ws=0x1000, ws_bytes=n - 1) == CAPACITY
    assert attn_call(L, **big, ws=0x1008, ws_bytes=n) == ALIGN


def test_longest_tables(L):
    """Positions rounded up to a tile of keys stay below 2^31."""
    long = pool(L, page_tokens=32767, page_bytes=32767 * 256, scale_page_bytes=32767 * 8)
    assert append_call(L, kv=long, max_pages=65537) == OK
    assert append_call(L, kv=long, max_pages=65538) == SHAPE   # 2^31 - 2 tokens
    assert attn_call(L, kv=long, max_pages=65537) == OK
    assert attn_call(L, kv=long, max_pages=65538) == SHAPE


def test_attention_workspace_bytes(L):
    f = L.lib().q3_attention_chunk_workspace_bytes
    assert f(0, 1, 1, 4096, 4, 2, 128) == 0 and f(4, 0, 1, 4096, 4, 2, 128) == 0
    assert f(4, 1, 4, 4096, 5, 2, 128) == 0                    # such a call is refused


def test_wrappers_refuse(q3):
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 256)
    with pytest.raises(ValueError):
        q3.ops.rope_rows(x, x, x, x, x, 2)
    with pytest.raises(ValueError):
        q3.ops.rope_tables(x, x, 1e6)


def test_attention_workspace_of_padded_rows(L):
    """Parts of split keys are those of the rows that sequences can have: rows that belong to nobody
    take none, and a card's worth of 256-row parts is the most."""
    f = L.lib().q3_attention_chunk_workspace_bytes
    for hd in (64, 128):
        for n_seqs, max_rows, max_kv in ((1, 256, 8192), (3, 200, 30000), (1, 100, 100000)):
            own = f(n_seqs * max_rows, n_seqs, max_rows, max_kv, 8, 8, hd)
            assert own > 0
            for rows in (4096, 8192, 100000):
                assert f(rows, n_seqs, max_rows, max_kv, 8, 8, hd) == own
    for rows in (64, 200, 8192, 1 << 20):
        for n_seqs in (1, 2, 7, 30, 200):
            for max_rows in (49, 256, 1000, 1 << 20):
                for kvh in (1, 2, 8):
                    parts = 148 * 256 * 130 * 4        # of the tensor-core kernel: a CTA an SM
                    few = 2 * 148 * 3 * 4 * 16 * 130 * 4
                    assert f(rows, n_seqs, max_rows, 8192, 4 * kvh, kvh, 128) <= parts + few
                    # float32 sums of long key ranges where keys are not split
                    sums = rows * 4 * kvh * 128 * 4
                    got = f(rows, n_seqs, max_rows, 50000, 4 * kvh, kvh, 128)
                    assert got <= few + max(parts, sums)


def test_attention_workspace_of_loose_bounds(L):
    """A sequence has no more new rows than its table holds tokens: a looser max_rows changes
    nothing."""
    f = L.lib().q3_attention_chunk_workspace_bytes
    for rows, n_seqs, max_kv, kvh in ((4096, 1, 1000, 1), (4096, 2, 16, 8), (2000, 3, 24, 2),
                                      (500, 1, 40, 4), (4096, 64, 256, 8)):
        for hd in (64, 128):
            tight = f(rows, n_seqs, max_kv, max_kv, 2 * kvh, kvh, hd)
            for loose in (2 * max_kv, 1 << 20, (1 << 32) - 1):
                assert f(rows, n_seqs, loose, max_kv, 2 * kvh, kvh, hd) == tight


def test_wrapper_refuses_other_workspaces(q3):
    """A workspace that is no tensor is named, before anything is done with it."""
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 256)
    for ws in (bytearray(64), 0x1000, [1], "ws"):
        with pytest.raises(ValueError, match="workspace: a"):
            q3.ops.attention_chunk_batch(x, None, pool(q3._lib), 9, x, 1, x, x, 1, 1, x, None, 4, 2, 64,
                                         True, 0, 0.1, workspace=ws)


def test_attention_workspace_bytes_of_refused_groups(L):
    f = L.lib().q3_attention_chunk_workspace_bytes
    assert f(64, 2, 32, 4096, 32, 2, 128) > 0                  # 16 query heads a KV head
    for rows in (1, 64, 4096):
        assert f(rows, 2, 2000, 4096, 34, 2, 128) == 0 and f(rows, 2, 1, 4096, 68, 4, 64) == 0


def test_attention_refuses_rows_past_32_bits(L):
    """Packed rows, rounded up to a tile, stay below 2^31."""
    big = lambda n, dt: view(L, n, 16 * 64, dt)                # noqa: E731
    call = lambda n: attn_call(L, q=big(n, F16), o=big(n, F16), heads=16, kvh=1, hd=64,  # noqa: E731
                               max_rows=1)
    assert call(2 ** 27 - 1) == SHAPE and call(2 ** 27 - 15) == SHAPE
    assert call(2 ** 27 - 16) == NULL                          # 2^31 - 256: on to the workspace


def test_factors_past_float32(L):
    """Finite in the type that they are given in, not in the one that is used."""
    assert tables(L, attn_factor=1e39) == SHAPE and tables(L, attn_factor=3e38) == OK
    assert attn_call(L, scale=3e38) == SHAPE and attn_call(L, scale=2e38) == OK
