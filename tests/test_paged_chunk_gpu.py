"""Rotary tables and rows, the append of K/V rows to the int8 pages, and the attention of a ragged
batch over them, on the GPU against float64 formulas (float32 steps where the codes are defined by
them).

Roundings: a result rounded to type t is off by at most eps(t)/2 of its value.  The attention
rounds its weights to f16 (2^-11 of each, and 2^-25 of the row's largest weight below f16's normal
range); everything else is float32, allowed for as 2^-20 of the largest logit's terms."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F = np.float32


@pytest.fixture(scope="module")
def ops(q3):
    assert torch.cuda.is_available(), "GPU tests need CUDA"
    return q3.ops


@pytest.fixture(autouse=True)
def clean_status(request, q3):
    q3._lib.lib().q3_device_status()
    yield
    if "status" not in request.node.keywords:
        assert q3._lib.lib().q3_device_status() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------ tables
def ref_freq(rot, theta, scaling, factor, orig, fast=32.0, slow=1.0):
    f = np.array([theta ** (-2.0 * i / rot) for i in range(rot // 2)])
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        per = rot / (2 * math.log(theta))
        lo = max(0, math.floor(per * math.log(orig / (fast * 2 * math.pi))))
        hi = min(rot - 1, math.ceil(per * math.log(orig / (slow * 2 * math.pi))))
        t = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 1e-3), 0, 1)
        return f * (1 - t) + f / factor * t
    return f


@pytest.mark.parametrize("rot,theta,scaling,factor,orig", [
    (128, 1e6, "none", 1.0, 0), (64, 1e4, "linear", 2.5, 0), (128, 1e6, "yarn", 4.0, 32768),
    (256, 5e5, "yarn", 8.0, 4096), (2, 10.0, "none", 1.0, 0), (34, 1e4, "yarn", 1.0, 64)])
@pytest.mark.parametrize("n,pos0", [(1, 0), (1, 2 ** 31 + 12345), (77, 131071), (3000, 0)])
def test_rope_tables(ops, rot, theta, scaling, factor, orig, n, pos0):
    cos = torch.full((n, rot // 2), 9.0, device="cuda")
    sin = torch.full((n, rot // 2 + 3), 9.0, device="cuda")[:, :rot // 2]   # a strided view
    ops.rope_tables(cos, sin, theta, pos0, scaling, factor, orig)
    a = 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0
    ang = np.outer(np.arange(pos0, pos0 + n, dtype=np.float64), ref_freq(rot, theta, scaling,
                                                                         factor, orig))
    # float32: the functions' last bit, the scaling by a; the oracle's angle: 2^-52 of itself
    tol = a * (4 * 2.0 ** -24 + 2 * ang.max() * 2.0 ** -52)
    assert np.abs(cos.cpu().numpy() - a * np.cos(ang)).max() <= tol
    assert np.abs(sin.cpu().numpy() - a * np.sin(ang)).max() <= tol


# -------------------------------------------------------------------- rows
def tables_f32(span, rot, theta=1e6):
    ang = torch.outer(torch.arange(span, dtype=torch.float64, device="cuda"),
                      torch.tensor(ref_freq(rot, theta, "none", 1, 0), device="cuda"))
    return torch.cos(ang).float(), torch.sin(ang).float()


def ref_norm(x, w):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w


def ref_rotate(x, cos, sin, inter):
    """x [rows][heads][hd]; cos, sin [rows][half], all float64."""
    half = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    y = x.clone()
    a = slice(0, 2 * half, 2) if inter else slice(0, half)
    b = slice(1, 2 * half, 2) if inter else slice(half, 2 * half)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows,heads,hd,rot", [(1, 1, 64, 64), (7, 3, 128, 128), (33, 16, 128, 64),
                                               (5, 6, 256, 256), (130, 5, 64, 16), (3, 9, 256, 80),
                                               (2, 4, 128, 112)])
@pytest.mark.parametrize("xt,ot,norm", [("f32", "f32", True), ("f32", "f16", False),
                                        ("bf16", "bf16", False), ("f16", "bf16", True),
                                        ("f16", "f32", False)])
def test_rope_rows(ops, rows, heads, hd, rot, inter, xt, ot, norm):
    g = gen(rows * hd + rot)
    wide = torch.randn(rows, heads * hd + 16, device="cuda", generator=g).to(TYPES[xt])
    x = wide[:, 8:8 + heads * hd] if xt != "f32" else wide[:, 4:4 + heads * hd]
    pos = torch.randint(0, 999, (rows,), device="cuda", generator=g, dtype=torch.int32)
    cos, sin = tables_f32(999, rot)
    nw = torch.rand(hd, device="cuda", generator=g) + 0.5 if norm else None
    out = torch.full((rows + 2, heads * hd), 7.0, device="cuda", dtype=TYPES[ot])
    ops.rope_rows(x, pos, cos, sin, out, heads, hd, nw=nw, interleaved=inter)
    want = x.double().reshape(rows, heads, hd)
    if norm:
        want = ref_norm(want, nw.double())
    p = pos.long()
    want = ref_rotate(want, cos.double()[p], sin.double()[p], inter).reshape(rows, -1)
    # float32 steps: two products and a sum (3), the norm (sum of hd squares: 2 + 5 + 8, root,
    # quotient, two products), each 2^-24 of at most sqrt(2) of the largest value
    tol = half_step(TYPES[ot]) * want.abs() + 20 * 2.0 ** -24 * want.abs().max() * 1.5
    assert ((out[:rows].double() - want).abs() <= tol).all()
    assert (out[rows:] == 7.0).all()


@pytest.mark.parametrize("hd,rot,inter", [(64, 64, False), (64, 32, True), (128, 128, False),
                                          (256, 128, False), (256, 256, True)])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_rows_codes(ops, hd, rot, inter, xt, norm):
    """int8 output: the bits of the float32 steps, through MatrixViews, heads left over in a warp."""
    rows, heads, V = 11, 13, ops.MatrixView
    g = gen(hd + rot)
    x = torch.randn(rows, heads * hd, device="cuda", generator=g).to(TYPES[xt])
    pos = torch.randint(0, 70, (rows,), device="cuda", generator=g, dtype=torch.int32)
    cos, sin = tables_f32(70, rot)
    nw = torch.rand(1, hd, device="cuda", generator=g) + 0.5 if norm else None
    out = torch.full((rows, (heads + 2) * hd), 5, device="cuda", dtype=torch.int8)
    scale = torch.full((rows, heads + 1), 5.0, device="cuda")
    ops.rope_rows(V.of(x), pos, V.of(cos), sin, V.of(out).cols_of(hd, heads * hd), heads, hd,
                  nw=nw, scale=V.of(scale), interleaved=inter)
    p = pos.long()
    host = lambda y: y.float().cpu().numpy()          # noqa: E731
    y = norm_rope_f32(host(x).reshape(rows, heads, hd), host(nw)[0] if norm else None, host(cos[p]),
                      host(sin[p]), inter)
    q, sc = int8_f32(y)
    got = out.cpu().numpy()
    assert np.array_equal(got[:, hd:-hd], q.reshape(rows, -1))
    assert (got[:, :hd] == 5).all() and (got[:, -hd:] == 5).all()
    assert np.array_equal(scale.cpu().numpy()[:, :heads], sc) and (scale[:, heads] == 5.0).all()


def test_rope_rows_in_place_and_bad_positions(ops, q3, request):
    request.node.keywords["status"] = True
    g = gen(3)
    x = torch.randn(6, 2 * 128, device="cuda", generator=g)
    cos, sin = tables_f32(50, 128)
    pos = torch.tensor([0, 49, 50, -1, 2 ** 31 - 1, 7], dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    ops.rope_rows(x, pos.clamp(0, 49), cos, sin, out, 2)
    before = x.clone()
    assert q3._lib.lib().q3_device_status() == 0
    ops.rope_rows(x, pos, cos, sin, x, 2)
    assert q3._lib.lib().q3_device_status() == 1 << 4
    ok = [0, 1, 5]
    assert torch.equal(x[ok], out[ok]) and torch.equal(x[2:5], before[2:5])


# ------------------------------------------------------------------ the pool
class Pool:
    """A page pool and the ragged batch over it: lens = (new rows, tokens with them) a sequence."""

    def __init__(self, ops, lens, kvh, hd, page=32, seed=0, pad_heads=0, spare=0):
        g = gen(seed)
        self.lens, self.kvh, self.hd, self.page = lens, kvh, hd, page
        self.mp = max(1, max(-(-kv // page) for _, kv in lens)) + spare
        n = self.n_pages = len(lens) * self.mp + 3
        w = kvh + pad_heads
        self.k = (torch.randn(n, page, w * hd, device="cuda", generator=g) * 42).round() \
            .clamp(-127, 127).to(torch.int8)
        self.v = (torch.randn(n, page, w * hd, device="cuda", generator=g) * 42).round() \
            .clamp(-127, 127).to(torch.int8)
        self.ks = torch.rand(n, page, w, device="cuda", generator=g) * 0.03 + 0.005
        self.vs = torch.rand(n, page, w, device="cuda", generator=g) * 0.03 + 0.005
        self.tables = torch.randperm(n, generator=torch.Generator().manual_seed(seed))[
            :len(lens) * self.mp].to(torch.int16).cuda().view(len(lens), self.mp)
        row0 = np.cumsum([0] + [a for a, _ in lens]).astype(np.int32)
        self.rows = int(row0[-1])
        self.row0 = torch.from_numpy(row0).cuda()
        self.kv_len = torch.tensor([b for _, b in lens], dtype=torch.int32, device="cuda")
        self.max_rows = max(a for a, _ in lens)
        self.kv = ops.paged_kv(self.k, self.v, self.ks, self.vs, self.tables, w, hd, page)

    def cached(self, s, kvlen=None):
        """K and V of sequence s: float64 [tokens][kvh][hd]."""
        n = self.lens[s][1] if kvlen is None else kvlen
        pages = self.tables[s, :-(-n // self.page)].long() & 0xFFFF
        return [(c[pages].reshape(-1, c.shape[-1] // self.hd, self.hd)[:n, :self.kvh].double(),
                 sc[pages].reshape(-1, sc.shape[-1])[:n, :self.kvh].double())
                for c, sc in ((self.k, self.ks), (self.v, self.vs))]


# ------------------------------------------------------------------- append
def int8_f32(x):
    """Codes and scales by the float32 steps of the cache's other writers."""
    x = x.astype(F)
    scale = (np.abs(x).max(-1) * F(1.0 / 127.0)).astype(F)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.rint((x / scale[..., None]).astype(F))
    return np.clip(np.nan_to_num(q), -127, 127).astype(np.int8), scale


def norm_rope_f32(x, nw, cos, sin, inter):
    """x [rows][heads][hd] float32 through the path's float32 steps."""
    from oracle import q3_oracle as O
    if nw is not None:
        r, h, d = x.shape
        x = O.rmsnorm(x.reshape(r * h, d), nw, F(1.0 / d)).reshape(r, h, d)
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos[:, None].astype(F), sin[:, None].astype(F)
    a = slice(0, 2 * half, 2) if inter else slice(0, half)
    b = slice(1, 2 * half, 2) if inter else slice(half, 2 * half)
    y = x.copy()
    y[..., a] = (x[..., a] * c).astype(F) - (x[..., b] * s).astype(F)
    y[..., b] = (x[..., a] * s).astype(F) + (x[..., b] * c).astype(F)
    return y


@pytest.mark.parametrize("kvh,hd,page,rot,inter,norm,t,lens", [
    (8, 128, 32, 128, False, True, "f32", [(1, 1), (1, 32), (1, 33), (0, 5), (1, 64)]),
    (2, 64, 16, 32, True, False, "bf16", [(40, 40), (0, 0), (3, 100), (17, 31)]),
    (1, 128, 32, 0, False, False, "f16", [(5, 70)]),
    (5, 256, 8, 256, False, True, "f16", [(9, 20), (1, 8), (30, 30)]),
    (4, 64, 7, 64, False, True, "bf16", [(13, 29), (8, 9)]),
    (3, 128, 32, 64, True, True, "f32", [(1, 1 + s % 40) for s in range(70)])])
def test_append(ops, kvh, hd, page, rot, inter, norm, t, lens):
    P = Pool(ops, lens, kvh, hd, page, seed=kvh + hd, pad_heads=1)
    g = gen(11)
    x = [(torch.randn(P.rows + 3, kvh * hd + 8, device="cuda", generator=g)).to(TYPES[t])
         for _ in range(2)]
    k, v = (y[:, :kvh * hd] for y in x)
    k[0, :hd] = 0.0                                   # an all-zero head: scale 0, codes 0
    nw = torch.rand(hd, device="cuda", generator=g) + 0.5 if norm else None
    cos, sin = tables_f32(P.mp * page, rot) if rot else (None, None)
    want = [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
    ops.paged_kv_append_batch(k, v, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, len(lens),
                              kvh, hd, nw=nw, cos=cos, sin=sin, interleaved=inter)
    host = lambda y: y.float().cpu().numpy()          # noqa: E731
    for s, (n, kv) in enumerate(lens):
        if not n:
            continue
        r = slice(int(P.row0[s]), int(P.row0[s]) + n)
        p = torch.arange(kv - n, kv, device="cuda")
        at = ((P.tables[s].long() & 0xFFFF)[p // page], p % page)
        kx = norm_rope_f32(host(k[r]).reshape(n, kvh, hd), host(nw) if norm else None,
                           host(cos[p]) if rot else None, host(sin[p]) if rot else None, inter)
        for y, codes, scales in ((kx, want[0], want[2]),
                                 (host(v[r]).reshape(n, kvh, hd), want[1], want[3])):
            q, sc = int8_f32(y)
            new = codes[at]
            new[:, :kvh * hd] = torch.from_numpy(q.reshape(n, -1)).cuda()
            codes[at] = new
            new = scales[at]
            new[:, :kvh] = torch.from_numpy(sc).cuda()
            scales[at] = new
    for got, exp in zip((P.k, P.v, P.ks, P.vs), want):
        assert torch.equal(got, exp)                  # everything else as it was, too


def test_append_refuses_on_the_device(ops, q3, request):
    """Rows that do not fit are skipped, the others written."""
    request.node.keywords["status"] = True
    P = Pool(ops, [(2, 40), (2, 10), (2, 64), (2, 33)], 2, 64, seed=4)
    P.kv_len.copy_(torch.tensor([1, 10, 65, 33]))      # fewer tokens than rows; beyond the table
    P.tables[3, 0] = -1                                # page 65535: beyond the pool
    k = torch.randn(P.rows, 128, device="cuda", generator=gen(1))
    before = [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
    cos, sin = tables_f32(64, 64)
    ops.paged_kv_append_batch(k, k, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 4, 2, 64,
                              cos=cos, sin=sin)
    assert q3._lib.lib().q3_device_status() == (1 << 5) | (1 << 2) | (1 << 1)
    changed = {(int(a), int(b)) for a, b in (P.ks != before[2]).any(-1).nonzero()}
    tab = (P.tables.long() & 0xFFFF).tolist()
    # sequence 0: position 0 of its second row; 1: both; 2: position 63; 3: position 32
    assert changed == {(tab[0][0], 0), (tab[1][0], 8), (tab[1][0], 9), (tab[2][1], 31),
                       (tab[3][1], 0)}


# ---------------------------------------------------------------- attention
def ref_attention(P, q, heads, causal, window, scale):
    """q float64 [rows][heads][hd] -> o, and what bounds its error: sum of weight |v|, the largest
    logit's sum of |terms| (base 2) and the part of weights below f16's normal range."""
    grp = heads // P.kvh
    o = torch.zeros(P.rows, heads, P.hd, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for s, (n, kv) in enumerate(P.lens):
        if not n:
            continue
        r = int(P.row0[s])
        (k8, ks), (v8, vs) = P.cached(s)
        k, v = k8 * ks[..., None], v8 * vs[..., None]
        qq = q[r:r + n].reshape(n, P.kvh, grp, P.hd)
        t = torch.einsum("nkgd,jkd->nkgj", qq, k) * scale
        big = torch.einsum("nkgd,jkd->nkgj", qq.abs(), k.abs()).amax(-1, keepdim=True) * scale
        j, p = torch.arange(kv, device="cuda"), torch.arange(kv - n, kv, device="cuda")[:, None]
        see = (j <= p) if causal else torch.ones(n, kv, dtype=torch.bool, device="cuda")
        if window:
            see = see & (j > p - window)
        t.masked_fill_(~see[:, None, None], -math.inf)
        w = torch.softmax(t, -1)
        o[r:r + n] = torch.einsum("nkgj,jkd->nkgd", w, v).reshape(n, heads, P.hd)
        a = torch.einsum("nkgj,jkd->nkgd", w, v.abs())
        rel = 2.0 ** -11 + 2 * 2.0 ** -20 * (big * 1.4427 + 8)
        low = 2.0 ** -25 * (w * vs.T[None, :, None]).amax(-1, keepdim=True) * \
            (v8.abs().sum(0)[None, :, None])
        tol[r:r + n] = (rel * a + low).reshape(n, heads, P.hd)
    return o, tol


def make_q(P, heads, qtype, seed, rows=None, spread=1.5):
    g = gen(seed)
    rows = P.rows if rows is None else rows
    x = torch.randn(rows, heads, P.hd, device="cuda", generator=g) * spread
    if qtype == "i8":
        qs = x.abs().amax(-1) / 127
        c = (x / qs[..., None]).round().clamp(-127, 127).to(torch.int8)
        return c.reshape(rows, -1), qs.contiguous(), c.double() * qs.double()[..., None]
    x = x.to(TYPES[qtype])
    return x.reshape(rows, -1), None, x.double()


def check_rows(got, os, want, tol, heads, hd, rows):
    if got.dtype == torch.int8:
        assert got.shape[1] >= heads * hd
        c = got[:rows, :heads * hd].reshape(rows, heads, hd).double()
        sc = os[:rows, :heads].double()
        top = want.abs().amax(-1)
        assert ((sc * 127 - top).abs() <= tol.amax(-1) + 3 * 2.0 ** -24 * top).all()
        assert c.abs().max() <= 127
        lim = tol + sc[..., None] * (0.5 + 2.0 ** -15)
        assert ((c * sc[..., None] - want).abs() <= lim).all()
    else:
        o = got[:rows].reshape(rows, heads, hd).double()
        lim = tol + half_step(got.dtype) * (want.abs() + tol) + \
            torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        assert ((o - want).abs() <= lim).all(), float(((o - want).abs() / lim).max())


def run_attention(ops, P, heads, qtype, otype, causal=True, window=0, seed=1, scale=None,
                  workspace=None, stream=None, spread=1.5):
    scale = P.hd ** -0.5 if scale is None else scale
    q, qs, q64 = make_q(P, heads, qtype, seed, spread=spread)
    dt = torch.int8 if otype == "i8" else TYPES[otype]
    o = torch.full((P.rows + 2, heads * P.hd), 7, device="cuda", dtype=dt)
    os = torch.full((P.rows + 2, heads), 7.0, device="cuda") if otype == "i8" else None
    ops.attention_chunk_batch(q, qs, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len,
                              len(P.lens), P.max_rows, o, os, heads, P.kvh, P.hd, causal, window,
                              scale, workspace=workspace, stream=stream)
    want, tol = ref_attention(P, q64, heads, causal, window, scale)
    check_rows(o, os, want, tol, heads, P.hd, P.rows)
    assert (o[P.rows:] == 7).all() and (os is None or (os[P.rows:] == 7).all())
    return o


SHAPES = [
    # heads, kv heads, head_dim, page, (new rows, tokens) per sequence
    (16, 8, 128, 32, [(1, 1), (1, 33), (1, 64), (0, 7), (1, 200), (1, 129)]),
    (16, 8, 128, 32, [(5, 5), (3, 300), (0, 0), (8, 41)]),
    (8, 1, 128, 32, [(1, 77), (2, 160)]),
    (12, 4, 64, 32, [(5, 1000), (1, 3), (4, 4)]),
    (5, 1, 64, 16, [(3, 50), (7, 100)]),
    (16, 1, 128, 7, [(1, 30), (3, 45)]),
    (4, 4, 64, 128, [(1, 400), (9, 129)]),
    (2, 1, 128, 32, [(130, 130), (67, 200), (1, 64)]),
    (4, 2, 128, 32, [(64, 1000), (257, 257), (300, 777)]),
    (6, 2, 64, 32, [(200, 431), (45, 45), (2, 900)]),
    (3, 3, 128, 64, [(129, 640)]),
    (2, 1, 64, 1, [(3, 40), (70, 300)]),
    (2, 2, 128, 4096, [(1, 3000), (90, 400)]),
    (30, 2, 64, 32, [(2, 500), (9, 9)]),
]


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 50), (False, 0), (True, 1)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_shapes(ops, shape, causal, window):
    heads, kvh, hd, page, lens = SHAPES[shape]
    P = Pool(ops, lens, kvh, hd, page, seed=shape)
    qt = ("i8", "f16", "bf16")[shape % 3]
    run_attention(ops, P, heads, qt, ("f16", "bf16", "i8")[(shape // 3 + window) % 3], causal,
                  window, seed=shape)


@pytest.mark.parametrize("qtype", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("otype", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", [[(1, 90), (2, 2)], [(150, 200), (40, 999)]])
def test_attention_types(ops, qtype, otype, hd, lens):
    run_attention(ops, Pool(ops, lens, 2, hd, seed=hd), 4, qtype, otype)


@pytest.mark.parametrize("heads,kvh,hd,lens", [
    (16, 8, 128, [(1, 20000)]), (8, 2, 64, [(4, 9000), (1, 31)]), (4, 1, 128, [(1, 7), (6, 30001)]),
    (4, 2, 128, [(100, 12345)]), (2, 2, 64, [(300, 9999), (1, 50)])])
def test_attention_long(ops, heads, kvh, hd, lens):
    """Few rows over many keys: the key range is split and joined."""
    P = Pool(ops, lens, kvh, hd, seed=9)
    n = ops.attention_chunk_workspace_bytes(P.rows, len(lens), P.max_rows, P.mp * 32, heads, kvh, hd)
    ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")       # NaN to begin with
    a = run_attention(ops, P, heads, "bf16", "bf16", workspace=ws)
    assert torch.equal(a, run_attention(ops, P, heads, "bf16", "bf16"))  # and repeatable


@pytest.mark.parametrize("new", [1, 150])
def test_attention_uneven_scales(ops, new):
    """Scales of K and V over ten binades, zero V scales, sharp softmax: the weights stay relative
    to each row's largest contribution."""
    P = Pool(ops, [(new, 700), (new, 333)], 2, 128, seed=21)
    e = torch.randint(-10, 1, P.vs.shape, device="cuda", generator=gen(2))
    P.vs.mul_(torch.exp2(e.float()))
    P.ks.mul_(torch.exp2(torch.randint(-5, 1, P.ks.shape, device="cuda", generator=gen(3)).float()))
    zero = torch.rand(P.vs.shape, device="cuda", generator=gen(5)) < 0.1
    P.vs.masked_fill_(zero, 0.0)
    P.v.view(*P.v.shape[:2], 2, 128).masked_fill_(zero[..., None], 0)
    run_attention(ops, P, 4, "f16", "f16", spread=6.0)


@pytest.mark.parametrize("scale", [2.0 ** -90, 2.0 ** 70])
def test_attention_tiny_and_huge_queries(ops, scale):
    """bf16 queries far outside f16's range: the row's power of two brings them back."""
    P = Pool(ops, [(3, 100), (140, 140)], 1, 64, seed=6)
    q, _, q64 = make_q(P, 2, "bf16", 3)
    q, q64 = (q.float() * scale).to(torch.bfloat16), q64 * scale
    o = torch.empty(P.rows, 128, device="cuda", dtype=torch.bfloat16)
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, 140, o,
                              None, 2, 1, 64, True, 0, 0.125 / scale)
    want, tol = ref_attention(P, q64, 2, True, 0, 0.125 / scale)
    check_rows(o, None, want, tol, 2, 64, P.rows)


@pytest.mark.parametrize("new", [2, 140])
def test_attention_garbage_behind_the_mask(ops, new):
    """NaN and infinite scales of tokens that a row does not see leave it alone; a row that sees a
    NaN is NaN, and no other."""
    P = Pool(ops, [(new, 150), (new, 161)], 2, 128, seed=8, spare=2)
    tab = P.tables.long() & 0xFFFF
    for s in range(2):
        kv = P.lens[s][1]
        for j in range(kv, tab.shape[1] * 32):         # behind the last token, spare pages too
            P.ks[tab[s, j // 32], j % 32] = float("nan") if j % 2 else float("inf")
            P.vs[tab[s, j // 32], j % 32] = float("inf") if j % 3 else float("nan")
    P.tables[0, -1] = -1                               # a page index beyond the pool, not needed
    o = run_attention(ops, P, 4, "i8", "f16")
    q, qs, q64 = make_q(P, 4, "i8", 1)
    last = P.lens[0][1] - 1                            # the last token of sequence 0
    for arr in (P.ks, P.vs):
        keep = arr[tab[0, last // 32], last % 32].clone()
        arr[tab[0, last // 32], last % 32] = float("nan")
        got = torch.empty_like(o)
        ops.attention_chunk_batch(q, qs, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, new,
                                  got, None, 4, 2, 128, True, 0, 128 ** -0.5)
        arr[tab[0, last // 32], last % 32] = keep
        assert got[new - 1].isnan().all()
        rest = [r for r in range(P.rows) if r != new - 1]
        assert torch.equal(got[rest], o[rest])


@pytest.mark.parametrize("new", [1, 140])
def test_attention_refuses_on_the_device(ops, q3, request, new):
    """Sequences whose arrays do not fit are skipped; keys in pages beyond the pool are not seen; a
    row that sees no key gives zeros."""
    request.node.keywords["status"] = True
    P = Pool(ops, [(new, 150), (new, 150), (new, 160), (new, 150)], 2, 128, seed=8)
    q, qs, q64 = make_q(P, 4, "f16", 1)
    want, tol = ref_attention(P, q64, 4, True, 0, 128 ** -0.5)
    P.tables[3] = -1
    P.kv_len[0] = new - 1
    P.kv_len[2] = P.mp * 32 + 1
    o = torch.full((P.rows, 512), 7.0, device="cuda", dtype=torch.float16)
    call = lambda mr: ops.attention_chunk_batch(                                   # noqa: E731
        q, qs, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 4, mr, o, None, 4, 2, 128, True,
        0, 128 ** -0.5)
    call(new)
    assert q3._lib.lib().q3_device_status() == (1 << 5) | (1 << 2) | (1 << 1)
    assert (o[:new] == 7).all() and (o[2 * new:3 * new] == 7).all()
    assert (o[3 * new:] == 0).all()
    lim = tol + 2.0 ** -11 * (want.abs() + tol)
    err = (o.double().reshape(-1, 4, 128) - want).abs()
    assert (err[new:2 * new] <= lim[new:2 * new]).all()
    if new > 1:                                        # more rows than max_rows
        o.fill_(7.0)
        call(new - 1)
        assert q3._lib.lib().q3_device_status() & (1 << 5)
        assert (o == 7).all()


def test_attention_strided_views(ops):
    P = Pool(ops, [(3, 70), (140, 300)], 2, 128, seed=5, pad_heads=3)
    q, _, q64 = make_q(P, 4, "f16", 2)
    wide = torch.zeros(P.rows, 3 * 512, device="cuda", dtype=torch.float16)
    wide[:, 512:1024] = q
    out = torch.full((P.rows, 3 * 512), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.attention_chunk_batch(wide[:, 512:1024], None, P.kv, P.n_pages, P.tables, P.mp, P.row0,
                              P.kv_len, 2, 140, out[:, 512:1024], None, 4, 2, 128, True, 0,
                              128 ** -0.5)
    want, tol = ref_attention(P, q64, 4, True, 0, 128 ** -0.5)
    check_rows(out[:, 512:1024], None, want, tol, 4, 128, P.rows)
    assert (out[:, :512] == 7).all() and (out[:, 1024:] == 7).all()


def test_attention_far_pages(ops):
    """A pool over 4 GB: byte offsets of its last pages pass 32 bits."""
    P = Pool(ops, [(1, 64), (130, 130)], 2, 128, seed=5)
    n, page_bytes = P.n_pages, 131072                  # 8 KB of each page used
    last = 40000 - n
    assert last * page_bytes > 2 ** 32
    kv2 = type(P.kv).from_buffer_copy(P.kv)
    bufs = []
    for src, sc in ((P.k, P.ks), (P.v, P.vs)):
        b = torch.empty(40000 * page_bytes, dtype=torch.int8, device="cuda")
        at = torch.as_strided(b, (n, 32 * 256), (page_bytes, 1), last * page_bytes)
        at.copy_(src.view(n, -1))
        s2 = torch.empty(last + n, 32, 2, device="cuda")
        s2[last:] = sc
        bufs.append((b, s2))
    kv2.k, kv2.v = bufs[0][0].data_ptr(), bufs[1][0].data_ptr()
    kv2.ks, kv2.vs = bufs[0][1].data_ptr(), bufs[1][1].data_ptr()
    kv2.page_bytes = page_bytes
    tables = ((P.tables.long() & 0xFFFF) + last).to(torch.int32)
    tables = torch.where(tables > 32767, tables - 65536, tables).to(torch.int16)
    assert last + n <= 65536
    q, _, q64 = make_q(P, 4, "f16", 2)
    o = torch.empty(P.rows, 512, device="cuda", dtype=torch.float16)
    ops.attention_chunk_batch(q, None, kv2, last + n, tables, P.mp, P.row0, P.kv_len, 2, 130, o,
                              None, 4, 2, 128, True, 0, 128 ** -0.5)
    want, tol = ref_attention(P, q64, 4, True, 0, 128 ** -0.5)
    check_rows(o, None, want, tol, 4, 128, P.rows)


# ------------------------------------------------------------ used together
def test_step_matches_the_fused_epilogues(ops):
    """norm + rotation + codes of the separate operators are the bits of the projections' epilogue,
    and the pages those of the scatter; then attention and the output projection on its codes."""
    from oracle import q3_oracle as O
    rng = np.random.default_rng(4)
    rows, heads, kvh, hd, hid = 21, 16, 8, 128, 512
    P = Pool(ops, [(rows, 85)], kvh, hd, seed=3)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()               # noqa: E731
    a = dev(rng.integers(-127, 128, (rows, hid)).astype(np.int8))
    a_s = dev(rng.uniform(1e-3, 1e-2, (rows, hid // 256)).astype(F))
    cos, sin = tables_f32(96, 128)
    start = 85 - rows
    pos = torch.arange(start, 85, dtype=torch.int32, device="cuda")
    out = {}
    for name, n in (("q", heads), ("k", kvh), ("v", kvh)):
        w = dev(rng.integers(-127, 128, (n * hd, hid)).astype(np.int8))
        ws = dev(rng.uniform(1e-3, 1e-2, n * hd).astype(F))
        nw = dev(rng.uniform(0.5, 1.5, hd).astype(F))
        x = torch.empty(rows, n * hd, device="cuda")
        ops.gemm_nt_group_store(a, a_s, w, ws, x, 256)
        c8 = torch.empty(rows, n * hd, dtype=torch.int8, device="cuda")
        cs = torch.empty(rows, n, device="cuda")
        if name == "v":
            ops.gemm_nt_group_store(a, a_s, w, ws, None, 256, q8=c8, qs=cs)
        else:
            ops.gemm_nt_group_store(a, a_s, w, ws, None, 256, q8=c8, qs=cs, nw=nw,
                                    cos=cos[start:85], sin=sin[start:85], inv_hd=1 / 128)
        out[name] = (x, nw, c8, cs)
    q8 = torch.empty_like(out["q"][2])
    qs = torch.empty_like(out["q"][3])
    ops.rope_rows(out["q"][0], pos, cos, sin, q8, heads, hd, nw=out["q"][1], scale=qs)
    assert torch.equal(q8, out["q"][2]) and torch.equal(qs, out["q"][3])
    other = [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
    kv2 = ops.paged_kv(*other, P.tables, kvh, hd, 32)
    ops.paged_kv_scatter(out["k"][2], out["v"][2], out["k"][3], out["v"][3], kv2, start, rows,
                         kvh * hd, kvh)
    ops.paged_kv_append_batch(out["k"][0], out["v"][0], P.kv, P.n_pages, P.tables, P.mp, P.row0,
                              P.kv_len, 1, kvh, hd, nw=out["k"][1], cos=cos, sin=sin)
    for x, y in zip((P.k, P.v, P.ks, P.vs), other):
        assert torch.equal(x, y)
    o8 = torch.empty(rows, heads * hd, dtype=torch.int8, device="cuda")
    os = torch.empty(rows, heads, device="cuda")
    ops.attention_chunk_batch(q8, qs, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 1, rows,
                              o8, os, heads, kvh, hd, True, 0, hd ** -0.5)
    q64 = q8.view(rows, heads, hd).double() * qs.double()[..., None]
    want, tol = ref_attention(P, q64, heads, True, 0, hd ** -0.5)
    check_rows(o8, os, want, tol, heads, hd, rows)
    wo = dev(rng.integers(-127, 128, (hid, heads * hd)).astype(np.int8))
    wos = dev(rng.uniform(1e-3, 1e-2, hid).astype(F))
    y = torch.empty(rows, hid, device="cuda")
    ops.gemm_nt_group_store(o8, os, wo, wos, y, 128)
    ref = O.gemm_group(o8.cpu().numpy(), os.cpu().numpy(), wo.cpu().numpy(), wos.cpu().numpy(), 128)
    assert np.array_equal(y.cpu().numpy(), ref)


def test_captured_step_replays_with_new_lengths(ops):
    """Tables, append and attention of a step in one graph; lengths, rows and tables change between
    replays, on another stream than the arrays were made on."""
    heads, kvh, hd = 4, 2, 128
    P = Pool(ops, [(1, 40), (1, 700), (1, 9)], kvh, hd, seed=7)
    x = {n: torch.randn(3, h * hd, device="cuda", generator=gen(h)).half()
         for n, h in (("q", heads), ("k", kvh), ("v", kvh))}
    cos, sin = torch.empty(704, 64, device="cuda"), torch.empty(704, 64, device="cuda")
    pos = P.kv_len - 1
    q, o = torch.empty_like(x["q"]), torch.empty_like(x["q"])
    ws = torch.empty(max(16, ops.attention_chunk_workspace_bytes(3, 3, 1, P.mp * 32, heads, kvh, hd)),
                     dtype=torch.uint8, device="cuda")

    def step():
        ops.rope_tables(cos, sin, 1e6)
        ops.rope_rows(x["q"], pos, cos, sin, q, heads, hd)
        ops.paged_kv_append_batch(x["k"], x["v"], P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len,
                                  3, kvh, hd, cos=cos, sin=sin)
        ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 3, 1,
                                  o, None, heads, kvh, hd, True, 0, hd ** -0.5, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for lens in ([40, 700, 9], [41, 640, 1], [1, 33, 704]):
        P.kv_len.copy_(torch.tensor(lens))
        pos.copy_(torch.tensor(lens) - 1)
        x["k"].mul_(1.5)
        saved = [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
        o.zero_()
        graph.replay()
        got, pages = o.clone(), [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
        for y, z in zip((P.k, P.v, P.ks, P.vs), saved):
            y.copy_(z)
        o.zero_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(o, got)
        for y, z in zip((P.k, P.v, P.ks, P.vs), pages):
            assert torch.equal(y, z)
        P.lens = [(1, n) for n in lens]
        want, tol = ref_attention(P, q.double().view(3, heads, hd), heads, True, 0, hd ** -0.5)
        check_rows(got, None, want, tol, heads, hd, 3)


def test_attention_stream_argument(ops):
    P = Pool(ops, [(1, 5000), (100, 300)], 2, 64, seed=5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    q, _, q64 = make_q(P, 4, "f16", 2)
    s.wait_stream(torch.cuda.current_stream())
    o = torch.empty(P.rows, 256, device="cuda", dtype=torch.float16)
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, 100, o,
                              None, 4, 2, 64, True, 0, 0.125, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    want, tol = ref_attention(P, q64, 4, True, 0, 0.125)
    check_rows(o, None, want, tol, 4, 64, P.rows)


def test_mixed_batch_captured_and_beside_itself(ops):
    """A batch of decode rows and prompt chunks (both attention kernels, split keys, the joins) in a
    graph, replayed after its lengths, rows and pages changed, while the same call runs on a second
    stream with a workspace of its own."""
    heads, kvh, hd = 8, 2, 128
    lens = [(1, 3000), (70, 1500), (0, 5), (300, 900), (4, 64), (129, 129)]
    P = Pool(ops, lens, kvh, hd, seed=12)
    n = len(lens)
    size = max(16, ops.attention_chunk_workspace_bytes(P.rows, n, 300, P.mp * 32, heads, kvh, hd))
    q, _, _ = make_q(P, heads, "f16", 3)
    ws = [torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = [torch.full((P.rows, heads * hd), 7.0, device="cuda", dtype=torch.float16)
           for _ in range(2)]

    def call(i):
        ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, n, 300,
                                  out[i], None, heads, kvh, hd, True, 0, hd ** -0.5, workspace=ws[i])
    call(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    side = torch.cuda.Stream()
    for step in range(3):
        q.mul_(1.1)
        lens = [(a, b - step * (b > a + 2)) for a, b in lens]
        if step:   # rows move from one sequence to another, within max_rows
            lens[0], lens[1] = (lens[0][0] + 20, lens[0][1]), (lens[1][0] - 20, lens[1][1])
        P.lens = lens
        P.row0.copy_(torch.tensor(np.cumsum([0] + [a for a, _ in lens]), dtype=torch.int32))
        P.kv_len.copy_(torch.tensor([b for _, b in lens], dtype=torch.int32))
        P.tables.copy_(P.tables.flip(0))
        for o in out:
            o.fill_(7.0)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            call(1)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out[0], out[1])
        want, tol = ref_attention(P, q.double().view(-1, heads, hd), heads, True, 0, hd ** -0.5)
        check_rows(out[0], None, want, tol, heads, hd, P.rows)


@pytest.mark.parametrize("seqs", [40, 1100])
def test_many_sequences(ops, seqs):
    """More sequences than a warp's lanes, and than its second look-up round."""
    rng = np.random.default_rng(seqs)
    lens = [(int(a), int(a) + int(b)) for a, b in zip(rng.integers(0, 4, seqs),
                                                      rng.integers(0, 60, seqs))]
    lens[seqs // 2] = (37, 64)
    P = Pool(ops, lens, 1, 64, page=16, seed=seqs)
    x = torch.randn(P.rows, 64, device="cuda", generator=gen(2)).half()
    cos, sin = tables_f32(P.mp * 16, 64)
    ops.paged_kv_append_batch(x, x, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, seqs, 1, 64,
                              cos=cos, sin=sin)
    v, r = [], 0
    for s, (a, b) in enumerate(lens):                  # the last rows' V codes, as appended
        (_, _), (v8, vs) = P.cached(s)
        v.append((v8 * vs[..., None])[b - a:b, 0])
    v = torch.cat(v)
    assert ((v - x.double()).abs() <= x.double().abs().amax(-1, keepdim=True) / 127 * 0.501).all()
    run_attention(ops, P, 2, "f16", "bf16")


def test_ragged_arrays_that_do_not_fit(ops, q3, request):
    """row0 that falls, or passes the rows: a status, the sequences that fit computed."""
    request.node.keywords["status"] = True
    P = Pool(ops, [(5, 40), (2, 300), (4, 50), (30, 60)], 2, 64, seed=2)
    q, _, q64 = make_q(P, 2, "f16", 1)
    want, tol = ref_attention(P, q64, 2, True, 0, 0.125)
    o = torch.full((P.rows, 128), 7.0, device="cuda", dtype=torch.float16)
    P.row0.copy_(torch.tensor([0, 5, 4, 11, 11 + 31], dtype=torch.int32))   # -1 rows; beyond q
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 4, 31, o,
                              None, 2, 2, 64, True, 0, 0.125)
    k = torch.randn(P.rows, 128, device="cuda")
    assert q3._lib.lib().q3_device_status() == 1 << 5
    check_rows(o[:4], None, want[:4], tol[:4], 2, 64, 4)   # sequence 0's rows but the shared one
    assert (o[11:] == 7).all()
    ops.paged_kv_append_batch(k, k, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 4, 2, 64)
    torch.cuda.synchronize()
    q3._lib.lib().q3_device_status()


def test_raw_stream_argument(ops):
    """A stream given by its handle, with a workspace from the caller's stream."""
    P = Pool(ops, [(1, 9000)], 1, 128, seed=5)
    s = torch.cuda.Stream()
    q, _, q64 = make_q(P, 2, "f16", 2)
    o = torch.empty(1, 256, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 1, 1, o,
                              None, 2, 1, 128, True, 0, 0.125, stream=s.cuda_stream)
    s.synchronize()
    want, tol = ref_attention(P, q64, 2, True, 0, 0.125)
    check_rows(o, None, want, tol, 2, 128, 1)


def test_results_complete_when_the_call_ends(ops):
    """Short sequences in long tables: none is cut, so the join has nothing to do, and what follows
    on the stream still sees every result."""
    lens = [(1 + s % 3, 3 + 7 * s % 90) for s in range(300)]
    heads, hd = 4, 64
    P = Pool(ops, lens, 2, hd, seed=11, spare=20)
    q, _, q64 = make_q(P, heads, "f16", 3)
    seen = []
    for _ in range(8):
        o = torch.full((P.rows, heads * hd), 7.0, device="cuda", dtype=torch.float16)
        ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len,
                                  len(lens), P.max_rows, o, None, heads, 2, hd, True, 0, 0.125)
        seen.append(o.clone())
    want, tol = ref_attention(P, q64, heads, True, 0, 0.125)
    check_rows(seen[0], None, want, tol, heads, hd, P.rows)
    assert all(torch.equal(x, seen[0]) for x in seen)


def test_nothing_to_do(ops):
    """No rows, and no sequences: a call that does nothing."""
    P = Pool(ops, [(0, 5), (0, 0)], 2, 64)
    x = torch.empty(0, 128, device="cuda", dtype=torch.float16)
    cos, sin = tables_f32(8, 64)
    ops.rope_tables(cos[:0], sin[:0], 1e6)
    ops.rope_rows(x, P.row0[:0], cos, sin, x, 2, 64)
    before = P.k.clone()
    for n in (2, 0):
        ops.paged_kv_append_batch(x, x, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len[:n], n, 2,
                                  64, cos=cos, sin=sin)
        ops.attention_chunk_batch(x, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len[:n], n,
                                  1, x, None, 2, 2, 64, True, 0, 0.125)
    o = torch.full((3, 128), 7.0, device="cuda", dtype=torch.float16)
    ops.attention_chunk_batch(o.clone(), None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2,
                              1, o, None, 2, 2, 64, True, 0, 0.125)   # rows that belong to nobody
    assert (o == 7).all() and torch.equal(P.k, before)


@pytest.mark.parametrize("heads,kvh,hd,page,window,lens", [
    (16, 8, 128, 32, 0, [(12, 1000), (16, 5000), (9, 9), (0, 4), (1, 300)]),   # two row tiles
    (16, 8, 128, 32, 70, [(16, 700), (13, 40), (16, 16), (2, 900)]),
    (16, 1, 128, 7, 0, [(2, 700), (1, 30)]),
    (12, 4, 64, 16, 0, [(10, 333), (5, 2000), (6, 6)]),
    (3, 1, 64, 32, 33, [(9, 1500)]),
    (2, 2, 64, 32, 0, [(17, 3000), (32, 300), (33, 33)]),          # rows one behind the most
    (4, 2, 128, 32, 0, [(1, 200), (4, 4), (2, 130)]),              # short, and few of them
    (2, 2, 64, 32, 0, [(48, 2000), (33, 300), (1, 1), (47, 47)]),
    (8, 2, 128, 16, 100, [(12, 1500), (9, 30), (5, 400)]),
    (2, 2, 64, 32, 0, [(49, 3000), (48, 300), (16, 90), (17, 33)]),
])
def test_attention_row_tiles(ops, heads, kvh, hd, page, window, lens):
    P = Pool(ops, lens, kvh, hd, page, seed=heads + len(lens))
    for q, o in (("f16", "f16"), ("i8", "i8"), ("bf16", "bf16")):
        run_attention(ops, P, heads, q, o, True, window)
    if not window:
        run_attention(ops, P, heads, "f16", "f16", False)


@pytest.mark.parametrize("seqs", [1, 37, 400])
def test_attention_row_tiles_across_slices(ops, seqs):
    """Row tiles that end inside slices: several of a sequence in one, and one in several."""
    rng = np.random.default_rng(seqs)
    lens = [(int(a), int(a + b)) for a, b in zip(rng.integers(1, 17, seqs), rng.integers(0, 900, seqs))]
    lens[0] = (16, 2500)
    run_attention(ops, Pool(ops, lens, 2, 64, page=32, seed=seqs), 4, "f16", "f16")


def test_steps_without_a_pause(ops):
    """Tables written anew and rows turned by them in place, back to back on one stream: each call
    sees what the one before it wrote, and none overwrites what one before it still reads."""
    rows, heads, hd, n = 4000, 8, 128, 8192
    cos = torch.empty(n, hd // 2, device="cuda")
    sin = torch.empty_like(cos)
    pos = torch.randint(0, n, (rows,), device="cuda", dtype=torch.int32, generator=gen(1))
    x0 = torch.randn(rows, heads * hd, device="cuda", generator=gen(2))

    def steps(x, pause):
        for i in range(12):
            ops.rope_tables(cos, sin, 1e4, pos0=1000 * i)
            pause()
            ops.rope_rows(x, pos, cos, sin, x, heads)
            pause()
        return x

    want = steps(x0.clone(), torch.cuda.synchronize)
    for _ in range(3):
        assert torch.equal(steps(x0.clone(), lambda: None), want)


def test_captured_on_forked_streams(ops):
    """Tables, rows and appends captured behind copies, on a stream that forks from the capture and
    joins it again."""
    P = Pool(ops, [(3, 70), (2, 40)], 2, 64, seed=4)
    cos, sin = tables_f32(100, 64)
    x = torch.randn(P.rows, 128, device="cuda", generator=gen(5))
    pos = torch.tensor([67, 68, 69, 38, 39], device="cuda", dtype=torch.int32)
    y, z = torch.zeros_like(x), torch.zeros_like(x)

    def step(side):
        main = torch.cuda.current_stream()
        y.copy_(x)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            ops.rope_rows(y, pos, cos, sin, y, 2, 64)
            ops.paged_kv_append_batch(y, x, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, 2,
                                      64)
        ops.rope_rows(x, pos, cos, sin, z, 2, 64)
        main.wait_stream(side)
        ops.rope_rows(y, pos, cos, sin, y, 2, 64)
        z.add_(y)

    side = torch.cuda.Stream()
    step(side)
    torch.cuda.synchronize()
    want, k, ks = z.clone(), P.k.clone(), P.ks.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(side)
    for _ in range(3):
        z.zero_(), y.zero_(), P.k.zero_(), P.ks.zero_()
        g.replay()
    torch.cuda.synchronize()
    row = (P.tables[0, 69 // 32].long() & 0xFFFF, 69 % 32)
    assert torch.equal(z, want) and torch.equal(P.k[row], k[row]) and torch.equal(P.ks[row], ks[row])
    assert (P.k[row] != 0).any()


@pytest.mark.parametrize("t,hd,inter", [("f32", 128, False), ("bf16", 64, True)])
def test_append_beyond_the_tables(ops, q3, request, t, hd, inter):
    """Tables shorter than the page table: a token at a position that they lack is not written at
    all, neither K nor V; the others are as with longer tables."""
    request.node.keywords["status"] = True
    lens = [(3, 51), (1, 50), (1, 64), (2, 97)]        # positions 48 49 50 | 49 | 63 | 95 96
    P, kvh = Pool(ops, lens, 3, hd, seed=17), 3
    k, v = (torch.randn(P.rows, kvh * hd, device="cuda", generator=gen(s)).to(TYPES[t])
            for s in (1, 2))
    cos, sin = tables_f32(97, hd)
    arrays = P.k, P.v, P.ks, P.vs
    before = [y.clone() for y in arrays]
    call = lambda n: ops.paged_kv_append_batch(                                    # noqa: E731
        k, v, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, len(lens), kvh, hd, cos=cos[:n],
        sin=sin[:n], interleaved=inter)
    call(97)
    assert q3._lib.lib().q3_device_status() == 0
    full = [y.clone() for y in arrays]
    for y, z in zip(arrays, before):
        y.copy_(z)
    call(50)
    assert q3._lib.lib().q3_device_status() == 1 << 4
    tab = P.tables.long() & 0xFFFF
    for s, j in ((0, 50), (2, 63), (3, 95), (3, 96)):
        for y, z in zip(full, before):
            y[tab[s, j // 32], j % 32] = z[tab[s, j // 32], j % 32]
    for got, want in zip(arrays, full):
        assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kvh,lens", [
    (8, 8, [(1, 60000)] * 444),                        # a slice of the keys is a sequence or more
    (64, 8, [(512, 60000)])])                          # 128 tiles: keys in one part
def test_attention_one_heavy_key(ops, heads, kvh, lens):
    """60000 keys of 2^-25.4 of the first one's weight each: together 0.14 % of the sum.  All values
    are 1, so the result is 1 if the sums over and under the fraction see the same weights.
    Weights are rounded to f16: the heavy one is a power of two but for 2^-18 (its logit's float32
    steps: 25.4 + 7 bits of 2^-24 twice), the light ones, 2^-32.4 times f16's largest power of
    two and so at least 2^-18.4, are off by at most 2^-25 each, 2^-6.6 of themselves; the result
    by half a step of f16 at 1."""
    hd, light = 64, 60000 * 2.0 ** -25.4
    P = Pool(ops, [(1, 60000)], kvh, hd)
    P.k.zero_(), P.v.fill_(100), P.ks.fill_(1.0), P.vs.fill_(0.01)
    tab = P.tables.long() & 0xFFFF
    P.k[tab[0, 0], 0] = 100                            # (a query is one in column 0 only)
    n = len(lens)
    tables = P.tables.expand(n, -1).contiguous()       # one cache, read by all
    rows = sum(a for a, _ in lens)
    row0 = torch.tensor(np.cumsum([0] + [a for a, _ in lens]), dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([b for _, b in lens], dtype=torch.int32, device="cuda")
    q = torch.zeros(rows, heads, hd, device="cuda", dtype=torch.float16)
    q[..., 0] = 1.0
    o = torch.empty(rows, heads * hd, device="cuda", dtype=torch.float16)
    ops.attention_chunk_batch(q.view(rows, -1), None, P.kv, P.n_pages, tables, P.mp, row0, kv_len, n,
                              lens[0][0], o, None, heads, kvh, hd, False, 0, 0.254 * math.log(2.0))
    tol = 2.0 ** -12 + 2.0 ** -17 + light * 2.0 ** -6.6 + 2 * 2.0 ** -11 * light
    assert tol < light / 2
    assert ((o.double() - 1.0).abs() <= tol).all(), float((o.double() - 1.0).abs().max())


@pytest.mark.parametrize("otype", ["bf16", "i8"])
@pytest.mark.parametrize("power", [-93, 110])
@pytest.mark.parametrize("new", [1, 150])
def test_attention_far_value_scales(ops, new, power, otype):
    """V scales near the ends of float32: the sums of weights over scales stay in range.  (Those of
    2^-93 times 0.005 and more pass 2^-100, as which the operator counts smaller ones.)"""
    P = Pool(ops, [(new, 3000), (new, 300)], 2, 128, seed=23)
    P.vs.mul_(2.0 ** power)
    q, _, q64 = make_q(P, 4, "bf16", 1, spread=4.0)
    o = torch.empty(P.rows, 512, device="cuda", dtype=torch.int8 if otype == "i8" else TYPES[otype])
    os = torch.empty(P.rows, 4, device="cuda") if otype == "i8" else None
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, new, o,
                              os, 4, 2, 128, True, 0, 128 ** -0.5)
    P.vs.clamp_(min=2.0 ** -100)
    want, tol = ref_attention(P, q64, 4, True, 0, 128 ** -0.5)
    check_rows(o, os, want, tol, 4, 128, P.rows)


@pytest.mark.parametrize("row0,written", [
    ([0, 5, 4, 11, 42], [0, 2]),       # -1 rows; the last sequence passes the rows
    ([0, 5, 20, 41, 50], [0, 1, 2]),   # all of the last one's rows are behind the end
    ([-3, 5, 5, 9, 9], [2]),           # rows before the first
    ([0, 41, 30, 30, 30], [0])])       # falls, and a row's last sequence has no rows
def test_append_ragged_arrays_that_do_not_fit(ops, q3, request, row0, written):
    """Sequences whose rows are not all there are skipped, with a status; others written."""
    request.node.keywords["status"] = True
    kvh, hd, rows = 2, 64, 41
    P = Pool(ops, [(5, 90), (2, 90), (4, 90), (30, 90)], kvh, hd, seed=2)
    P.row0.copy_(torch.tensor(row0, dtype=torch.int32))
    k = torch.randn(rows, kvh * hd, device="cuda", generator=gen(1))
    before = [y.clone() for y in (P.k, P.v, P.ks, P.vs)]
    ops.paged_kv_append_batch(k, k, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 4, kvh, hd)
    assert q3._lib.lib().q3_device_status() == 1 << 5
    tab = P.tables.long() & 0xFFFF
    may, must = set(), set()
    for s in written:
        a, b = row0[s], row0[s + 1]
        for r in range(a, b):
            j = 90 - (b - a) + r - a
            at = (int(tab[s, j // 32]), j % 32)
            may.add(at)
            # (a row that two sequences claim is written for one of them)
            if sum(row0[x] <= r < row0[x + 1] for x in range(4)) == 1 and row0 == sorted(row0):
                must.add(at)
    for got, old in zip((P.k, P.v, P.ks, P.vs), before):
        changed = {(int(a), int(b)) for a, b in (got != old).any(-1).nonzero()}
        assert must <= changed <= may


@pytest.mark.parametrize("new", [4, 300])
def test_row_numbers_that_wrap(ops, q3, request, new):
    """row0 whose difference fits only modulo 2^32: refused, not taken for one row."""
    request.node.keywords["status"] = True
    P = Pool(ops, [(new, 700), (3, 90)], 2, 64, seed=6)
    big = 2 ** 31
    P.row0.copy_(torch.tensor([big - 1, -big, -big + new], dtype=torch.int32))
    x = torch.randn(P.rows, 128, device="cuda", generator=gen(1)).half()
    o = torch.full((P.rows, 128), 7.0, device="cuda", dtype=torch.float16)
    before = P.k.clone()
    ops.attention_chunk_batch(x, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, new, o,
                              None, 2, 2, 64, True, 0, 0.125)
    assert q3._lib.lib().q3_device_status() == 1 << 5 and (o == 7).all()
    ops.paged_kv_append_batch(x, x, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, 2, 64)
    assert q3._lib.lib().q3_device_status() == 1 << 5 and torch.equal(P.k, before)


@pytest.mark.parametrize("otype", ["f16", "i8"])
@pytest.mark.parametrize("heads,kvh,hd,lens,most,pad", [
    (4, 4, 128, [(200, 5000)], 200, 4000), (6, 2, 64, [(90, 9000), (300, 3000), (1, 40)], 310, 999),
    (2, 1, 64, [(50, 700), (70, 3000), (256, 2000), (0, 9), (257, 300), (3, 8000)], 257, 77)])
def test_attention_padded_rows(ops, heads, kvh, hd, lens, most, pad, otype):
    """Split keys in a batch with rows behind its last sequence: a workspace of the rows that
    sequences can have, no word behind it written, and the padding left as it was."""
    P = Pool(ops, lens, kvh, hd, seed=31)
    rows, n = P.rows + pad, len(lens)
    q, _, q64 = make_q(P, heads, "f16", 4, rows=rows)
    size = ops.attention_chunk_workspace_bytes(rows, n, most, P.mp * 32, heads, kvh, hd)
    assert 0 < size <= 148 * (256 + 2 * 3 * 4 * 16) * (hd + 2) * 4   # a part a CTA; two a warp, of 16
    ws = torch.full((size + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    o = torch.full((rows, heads * hd), 7, device="cuda",
                   dtype=torch.int8 if otype == "i8" else torch.float16)
    os = torch.full((rows, heads), 7.0, device="cuda")
    ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, n, most, o,
                              os if otype == "i8" else None, heads, kvh, hd, True, 0, hd ** -0.5,
                              workspace=ws[:size])
    want, tol = ref_attention(P, q64[:P.rows], heads, True, 0, hd ** -0.5)
    check_rows(o, os, want, tol, heads, hd, P.rows)
    assert (o[P.rows:] == 7).all() and (os[P.rows:] == 7.0).all() and (ws[size:] == 0xFF).all()


@pytest.mark.parametrize("kvh,hd,page,lens", [
    (2, 64, 16, [(1 + s % 5, 5 + s % 12) for s in range(64)]),       # no table holds 17 tokens
    (2, 128, 32, [(1 + 3 * s, 60 + 3 * s) for s in range(40)]),      # whole sequences, in tiles
    (1, 128, 32, [(7, 320), (300, 320), (40, 90)]), (2, 64, 8, [(8, 8), (3, 7)])])
def test_attention_loose_max_rows(ops, kvh, hd, page, lens):
    """max_rows far over what the tables hold: the same results as with the least one."""
    P = Pool(ops, lens, kvh, hd, page, seed=14)
    tight = run_attention(ops, P, 4, "f16", "f16")
    for P.max_rows in (P.rows, 100000, 2 ** 32 - 1):
        assert torch.equal(run_attention(ops, P, 4, "f16", "f16"), tight)


def test_attention_workspace_in_a_foreign_capture(ops):
    """A call onto a captured stream from one that is not: its own workspace would go back to the
    allocator while the graph still uses it, so one must be given; then the graph replays."""
    P = Pool(ops, [(1, 9000), (100, 300)], 2, 64, seed=5)
    q, _, q64 = make_q(P, 4, "f16", 2)
    o = torch.zeros(P.rows, 256, device="cuda", dtype=torch.float16)
    size = ops.attention_chunk_workspace_bytes(P.rows, 2, 100, P.mp * 32, 4, 2, 64)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call(stream, ws=None):
        ops.attention_chunk_batch(q, None, P.kv, P.n_pages, P.tables, P.mp, P.row0, P.kv_len, 2, 100,
                                  o, None, 4, 2, 64, True, 0, 0.125, workspace=ws, stream=stream)
    other, inside = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.cuda.current_stream()
        for current in (other, torch.cuda.default_stream()):   # not part of the capture
            with torch.cuda.stream(current):
                for stream in (captured, captured.cuda_stream):
                    with pytest.raises(ValueError, match="workspace"):
                        call(stream)
                call(captured, ws)
        inside.wait_stream(captured)                   # part of it: the graph's own memory
        call(inside)
        captured.wait_stream(inside)
    want, tol = ref_attention(P, q64, 4, True, 0, 0.125)
    for _ in range(2):
        o.zero_()
        graph.replay()
        check_rows(o, None, want, tol, 4, 64, P.rows)


@pytest.mark.parametrize("power", [-20, -6, -4, -3, 0, 4, 5, 12])
@pytest.mark.parametrize("new", [3, 140])
def test_attention_small_elements_of_bf16_queries(ops, new, power):
    """One large element a row that meets zeros, all others 2^-12 of it, with their lowest bit set:
    the logits are theirs alone, so they have to be exact in the products."""
    P = Pool(ops, [(new, 200), (new, 333)], 1, 64, seed=26)
    P.k.view(-1, 64)[:, 0] = 0
    q = torch.full((P.rows, 2, 64), 2.0 ** -12 * (1 + 2.0 ** -7), device="cuda")
    q[..., 0] = 1.0
    q = (q * 2.0 ** power).to(torch.bfloat16)
    scale = 6000.0 * 2.0 ** -power                     # logits of about 10
    o = torch.empty(P.rows, 128, device="cuda", dtype=torch.float16)
    ops.attention_chunk_batch(q.view(P.rows, -1), None, P.kv, P.n_pages, P.tables, P.mp, P.row0,
                              P.kv_len, 2, new, o, None, 2, 1, 64, True, 0, scale)
    want, tol = ref_attention(P, q.double(), 2, True, 0, scale)
    check_rows(o, None, want, tol, 2, 64, P.rows)


def check_long_sums(ops, heads, kvh, hd, n, new, kv, causal=False):
    """All values are 1 under weights that differ, over many keys: the result is 1, seen to float32 by
    the scale of int8 output.  Returns the largest error.

    What it may be: each weight's rounding to f16, at most 2^-11 of it and of either sign, so at most
    2^-11 sqrt(2 ln(2 / P) sum w^2) but with probability P (the squares of weights e^x, x normal
    of deviation s: e^(s^2) / keys): 1e-5 at P = 1e-12, s = 0.8 and 500000 keys.  Sums of a
    thread over an eighth of the keys, 2^-25 an add of either sign: 4e-5 likewise.  What the tensor cores
    cut in a running sum over 8192 keys: below 2^-24 of it for each of 16 terms and the sum itself, of
    512 products, half of it since it grows: 2.6e-4."""
    page = 4096
    mp = -(-kv // page)
    k = torch.randint(-127, 128, (mp, page, kvh * hd), device="cuda", generator=gen(1),
                      dtype=torch.int8)
    v = torch.full_like(k, 100)
    ks = torch.full((mp, page, kvh), 0.01, device="cuda")
    vs = torch.full_like(ks, 0.01)
    tables = torch.arange(mp, device="cuda").to(torch.int16).expand(n, -1).contiguous()
    cache = ops.paged_kv(k, v, ks, vs, tables, kvh, hd, page)
    row0 = torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda")
    kv_len = torch.full((n,), kv, dtype=torch.int32, device="cuda")
    q = torch.randn(n * new, heads * hd, device="cuda", generator=gen(2)).half()
    o = torch.empty(n * new, heads * hd, dtype=torch.int8, device="cuda")
    os = torch.empty(n * new, heads, device="cuda")
    ops.attention_chunk_batch(q, None, cache, mp, tables, mp, row0, kv_len, n, new, o, os, heads, kvh,
                              hd, causal, 0, hd ** -0.5)
    assert (o == 127).all()
    return float((os.double() * 127 / (100 * vs[0, 0, 0].double()) - 1).abs().max())


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_long_sums_few_rows(ops, hd):
    assert check_long_sums(ops, 8, 8, hd, 444, 1, 500000) <= 2.0 ** -11


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_long_sums_many_rows(ops, hd):
    assert check_long_sums(ops, 32, 8, hd, 1, 1024, 500000) <= 2.0 ** -11        # one part
    assert check_long_sums(ops, 4, 2, hd, 1, 130, 500000) <= 2.0 ** -11          # several


@pytest.mark.parametrize("heads,kvh,hd,lens,window,otype", [
    (16, 4, 128, [(900, 20000), (300, 8193), (20, 30000), (257, 17000)], 0, "f16"),
    (32, 8, 64, [(600, 8192 + 600), (40, 40000)], 0, "i8"),
    (24, 8, 64, [(500, 33000)], 20000, "bf16"),
    (2, 1, 128, [(300, 300000)], 0, "f16"), (3, 1, 64, [(200, 200000), (1, 9)], 0, "i8")])
def test_attention_folded_sums(ops, heads, kvh, hd, lens, window, otype):
    """Key ranges over a fold, in one part and in several, of tiles that end at other key tiles than
    their CTA, whose references grow late (a few keys have far larger scales)."""
    P = Pool(ops, lens, kvh, hd, page=64, seed=33)
    P.ks.mul_(0.2)
    far = torch.rand(P.ks.shape, device="cuda", generator=gen(8)) < 2e-4
    P.ks.mul_(1.0 + 19.0 * far)
    run_attention(ops, P, heads, "f16", otype, True, window, seed=2)
