"""What is measured of the paged-cache operators: rotary tables, rotary rows,
the append of new K/V rows to the int8 pages, and the attention of a chunk of
new rows over the pages.

``run`` computes an operator in plain torch operations, or, where ``own`` is
true, by the framework's entry points (``q3b200.ops``).
"""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
PAGE = 32                    # tokens of a page of the framework's pool
EPS = 1e-6
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # rotary tables of a served model's usual context, and of a long one with scaled positions
        dict(name="tables_4k", op="tables", n=4096, rot=128, pos0=0, theta=1e6, scaling="none",
             factor=1.0, orig=0),
        dict(name="tables_128k_yarn", op="tables", n=131072, rot=128, pos0=0, theta=1e6,
             scaling="yarn", factor=4.0, orig=32768),
        # the query rows of a decode step of 64 sequences: head norm, then rotation
        dict(name="rope_decode", op="rope", rows=64, heads=16, hd=128, rot=128, inter=False,
             norm=True, type="f32", span=4096),
        # the query rows of a step full of prompt chunks
        dict(name="rope_chunk", op="rope", rows=8192, heads=16, hd=128, rot=128, inter=False,
             norm=True, type="f32", span=16384),
        # interleaved pairs in half of the head, an odd number of rows, 16-bit rows
        dict(name="rope_partial", op="rope", rows=5003, heads=40, hd=128, rot=64, inter=True,
             norm=False, type="bf16", span=32768),
        # one new token for each of 64 sequences (float32 projections, K norm)
        dict(name="append_decode", op="append", seqs=64, new=1, ctx=30, ragged=3, kvh=8, hd=128,
             rot=128, inter=False, norm=True, type="f32"),
        # prompt chunks of 16 sequences, ragged, 16-bit rows
        dict(name="append_chunk", op="append", seqs=16, new=797, ctx=50, ragged=5, kvh=8, hd=128,
             rot=128, inter=False, norm=False, type="bf16"),
        # one decode step of 64 sequences at 2048 tokens; int8 queries as the projections' epilogue writes them
        dict(name="attn_decode", op="attn", seqs=64, new=1, ctx=2047, ragged=0, heads=16, kvh=8,
             hd=128, window=0, causal=True, qtype="i8", type="f16"),
        # two sequences alone at a long, odd context: the keys are split over the card
        dict(name="attn_decode_long", op="attn", seqs=2, new=1, ctx=65010, ragged=0, heads=32,
             kvh=8, hd=128, window=0, causal=True, qtype="bf16", type="bf16"),
        # five drafted tokens to verify for each of 24 sequences, small heads
        dict(name="attn_draft", op="attn", seqs=24, new=5, ctx=3001, ragged=7, heads=12, kvh=4,
             hd=64, window=0, causal=True, qtype="f16", type="f16"),
        # an engine's step: decode rows and prompt chunks of all lengths together, a sliding window
        dict(name="attn_ragged", op="attn", seqs=16, new=385, ctx=4001, ragged=11, heads=16, kvh=8,
             hd=128, window=2048, causal=True, qtype="i8", type="f16"),
        # long prompts in large chunks: the second half of two 8192-token prompts
        dict(name="attn_chunk", op="attn", seqs=2, new=4096, ctx=4096, ragged=0, heads=16, kvh=8,
             hd=128, window=0, causal=True, qtype="bf16", type="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("tables", "rope", "append", "attn", "attn", "attn"))
    if op == "tables":
        scaling = rng.choice(("none", "linear", "yarn"))
        return dict(op=op, n=_log(rng, 16, 131072), rot=rng.choice((32, 64, 96, 128)),
                    pos0=_log(rng, 1, 100000), theta=rng.choice((1e4, 5e5, 1e6)), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0, 2.5)),
                    orig=0 if scaling != "yarn" else rng.choice((4096, 8192, 32768)))
    hd = rng.choice((64, 128, 128))
    typ = rng.choice(("f32", "f16", "bf16"))
    if op == "rope":
        return dict(op=op, rows=_log(rng, 1, 8192), heads=rng.choice((8, 15, 16, 32)), hd=hd,
                    rot=rng.choice((hd, hd, hd // 2)), inter=rng.random() < 0.5,
                    norm=rng.random() < 0.5, type=typ, span=_log(rng, 1024, 131072))
    if op == "append":
        seqs = _log(rng, 1, 64)
        return dict(op=op, seqs=seqs, new=_log(rng, 1, max(1, 12000 // seqs)), ctx=_log(rng, 1, 64),
                    ragged=rng.randrange(1, 1000), kvh=rng.choice((1, 2, 4, 8)), hd=hd,
                    rot=rng.choice((hd, hd, hd // 2)), inter=rng.random() < 0.5,
                    norm=rng.random() < 0.5, type=typ)
    kvh, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 8))
    heads = kvh * group
    new = rng.choice((1, 1, _log(rng, 2, 32), _log(rng, 2, 4096), _log(rng, 64, 4096)))
    seqs = _log(rng, 1, 64)
    ctx = _log(rng, 1, 65536)
    # no dearer than the largest listed case: query-key pairs, and keys, over all sequences
    ctx = max(1, min(ctx, 1000000 // (seqs * new * heads) * 1000 - new, 250000 // seqs))
    seqs = max(1, min(seqs, 1000000000 // (new * heads * (ctx + new))))
    qtype = rng.choice(("i8", "f16", "bf16"))
    return dict(op=op, seqs=seqs, new=new, ctx=ctx, ragged=rng.choice((0, rng.randrange(1, 1000))),
                heads=heads, kvh=kvh, hd=hd, window=rng.choice((0, 0, 0, _log(rng, 1, 8192))),
                causal=True, qtype=qtype,
                type=rng.choice(("f16", "bf16")) if qtype == "i8" else qtype)


def _lengths(case):
    """New rows and tokens already cached of every sequence; ragged ones are fixed by the case."""
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["ctx"]] * case["seqs"]
    r = random.Random(case["ragged"])
    new = [_log(r, 1, case["new"]) for _ in range(case["seqs"])]
    ctx = [r.randrange(0, case["ctx"] + 1) for _ in range(case["seqs"])]
    new[0], ctx[-1] = case["new"], case["ctx"]
    return new, ctx


def _max_pages(case):
    return -(-(case["new"] + case["ctx"]) // PAGE)


def _pairs(case):
    """Visible (row, key) pairs of all sequences, for one head."""
    new, ctx = _lengths(case)
    total = 0
    for n, c in zip(new, ctx):
        w = case["window"] or (n + c)
        # row i sees min(c + i + 1, w) keys
        full = max(0, min(n, w - c))
        total += full * c + full * (full + 1) // 2 + (n - full) * w
    return total


def work(case):
    op = case["op"]
    if op == "tables":
        return {"bytes": 4.0 * case["n"] * case["rot"], "flops": 0.0}
    if op == "rope":
        e = 4 if case["type"] == "f32" else 2
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2.0 * n * e + 4.0 * case["rows"] * (case["rot"] + 1),
                "flops": 3.0 * n + (4.0 * n if case["norm"] else 0.0)}
    new, ctx = _lengths(case)
    rows, e = sum(new), 1 if case.get("qtype") == "i8" else 2
    if op == "append":
        e = 4 if case["type"] == "f32" else 2
        n = rows * case["kvh"] * case["hd"]
        # and the pages returned as the values they stand for
        pool = case["seqs"] * _max_pages(case) * PAGE * case["kvh"] * (case["hd"] + 4)
        back = 2.0 * case["seqs"] * _max_pages(case) * PAGE * case["kvh"] * case["hd"] * 4
        return {"bytes": 2.0 * n * e + 2.0 * rows * case["kvh"] * (case["hd"] + 4) + 2.0 * pool
                + back, "flops": 12.0 * n}
    w = case["window"]
    keys = sum(c + n if not w else min(c + n, n + w - 1) for n, c in zip(new, ctx))
    qo = rows * case["heads"] * (case["hd"] * (e + 2) + (4 if case["qtype"] == "i8" else 0))
    return {"bytes": float(qo + 2 * keys * case["kvh"] * (case["hd"] + 4)),
            "flops": 4.0 * case["hd"] * case["heads"] * _pairs(case)}


def _inv_freq(case):
    """Angular frequency of each pair (64 bits) and the factor on cos and sin."""
    rot, theta, f = case["rot"], case["theta"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEV)
    inv = torch.exp(i * (-2.0 * math.log(theta) / rot))
    if case["scaling"] == "linear":
        return inv / f, 1.0
    if case["scaling"] == "yarn":
        turn = rot / (2.0 * math.log(theta))
        low = max(0, math.floor(turn * math.log(case["orig"] / (32.0 * 2.0 * math.pi))))
        high = min(rot - 1, math.ceil(turn * math.log(case["orig"] / (1.0 * 2.0 * math.pi))))
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return inv / f * ramp + inv * (1.0 - ramp), 0.1 * math.log(f) + 1.0
    return inv, 1.0


def _rope_tables_f32(span, rot):
    inv, _ = _inv_freq(dict(rot=rot, theta=1e6, factor=1.0, scaling="none"))
    ang = torch.arange(span, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cos(ang).float(), torch.sin(ang).float()


def _pool(g, pages, kvh, hd):
    """Codes and scales of a filled int8 pool: K and V of about unit size, uneven by token."""
    def codes():
        x = torch.randn(pages, PAGE, kvh * hd, device=DEV, generator=g)
        return (x * 42.0).round_().clamp_(-127, 127).to(torch.int8)

    def scales():
        return torch.rand(pages, PAGE, kvh, device=DEV, generator=g) * 0.03 + 0.01
    return dict(k=codes(), v=codes(), ks=scales(), vs=scales())


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "tables":
        # the first position changes with the seed
        s["pos0"] = case["pos0"] + seed % 61
        s["cos"] = torch.empty(case["n"], case["rot"] // 2, device=DEV)
        s["sin"] = torch.empty_like(s["cos"])
        return s
    hd = case["hd"]
    if case["op"] == "rope":
        s["x"] = torch.randn(case["rows"], case["heads"] * hd, device=DEV,
                             generator=g).to(_TYPES[case["type"]])
        s["pos"] = torch.randint(0, case["span"], (case["rows"],), device=DEV, generator=g,
                                 dtype=torch.int32)
        s["cos"], s["sin"] = _rope_tables_f32(case["span"], case["rot"])
        s["nw"] = torch.rand(hd, device=DEV, generator=g) + 0.5 if case["norm"] else None
        s["out"] = torch.empty_like(s["x"])
        return s
    new, ctx = _lengths(case)
    rows, mp, kvh = sum(new), _max_pages(case), case["kvh"]
    s["rows"] = rows
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    s["row0"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["kv_len"] = torch.tensor([n + c for n, c in zip(new, ctx)], dtype=torch.int32, device=DEV)
    pages = case["seqs"] * mp
    s["tables"] = torch.randperm(pages, device=DEV, generator=g).to(torch.int16).view(-1, mp)
    s.update(_pool(g, pages, kvh, hd))
    if case["op"] == "append":
        t = _TYPES[case["type"]]
        s["kx"] = torch.randn(rows, kvh * hd, device=DEV, generator=g).to(t)
        s["vx"] = torch.randn(rows, kvh * hd, device=DEV, generator=g).to(t)
        s["nw"] = torch.rand(hd, device=DEV, generator=g) + 0.5 if case["norm"] else None
        s["cos"], s["sin"] = _rope_tables_f32(mp * PAGE, case["rot"])
        return s
    x = torch.randn(rows, case["heads"] * hd, device=DEV, generator=g) * 1.5
    s["qs"] = None
    if case["qtype"] == "i8":
        x = x.view(rows, case["heads"], hd)
        s["qs"] = (x.abs().amax(-1) / 127.0).contiguous()
        x = (x / s["qs"][..., None]).round_().clamp_(-127, 127).view(rows, -1).to(torch.int8)
    else:
        x = x.to(_TYPES[case["qtype"]])
    s["q"] = x
    s["o"] = torch.empty(rows, case["heads"] * hd, device=DEV, dtype=_TYPES[case["type"]])
    return s


# ------------------------------------------------------------------ plain forms
def _tables(s):
    case = s["case"]
    inv, a = _inv_freq(case)
    # far positions: angles in 64 bits
    pos = torch.arange(case["n"], dtype=torch.float64, device=DEV) + s["pos0"]
    ang = pos[:, None] * inv
    return (torch.cos(ang) * a).float(), (torch.sin(ang) * a).float()


def _pair_sums(x):
    return x[..., 0::2] + x[..., 1::2]


def _head_norm(x, nw):
    """RMSNorm of the last axis; squares summed by pairs in blocks of 32, the blocks in order."""
    sq = (x * x).unflatten(-1, (-1, 32))
    blocks = _pair_sums(_pair_sums(_pair_sums(_pair_sums(_pair_sums(sq))))).squeeze(-1)
    ss = blocks[..., 0] + blocks[..., 1]
    if blocks.shape[-1] == 4:
        ss = ss + blocks[..., 2] + blocks[..., 3]
    r = 1.0 / torch.sqrt(ss * (1.0 / x.shape[-1]) + EPS)
    return x * r[..., None] * nw


def _rotate(x, cos, sin, inter):
    """x: [rows][heads][hd]; cos, sin: [rows][rot / 2] at the rows' positions."""
    half = cos.shape[-1]
    c, n = cos[:, None, :], sin[:, None, :]
    y = x.clone()
    if inter:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * c - b * n
        y[..., 1:2 * half:2] = a * n + b * c
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * c - b * n
        y[..., half:2 * half] = a * n + b * c
    return y


def _rope(s):
    case = s["case"]
    x = s["x"].float().view(case["rows"], case["heads"], case["hd"])
    if s["nw"] is not None:
        x = _head_norm(x, s["nw"])
    p = s["pos"].long()
    return _rotate(x, s["cos"][p], s["sin"][p], case["inter"]).to(s["x"].dtype).view_as(s["x"])


def _row_places(s):
    """Sequence, index within the sequence's new rows, and position of every row."""
    r = torch.arange(s["rows"], device=DEV)
    row0 = s["row0"].long()
    seq = torch.searchsorted(row0, r, right=True) - 1
    i = r - row0[seq]
    return seq, i, s["kv_len"].long()[seq] - (row0[seq + 1] - row0[seq]) + i


def _int8(x):
    """One scale a head; the codes follow the float32 steps of the framework's other cache writers
    (the quotient next to a half goes by them), so both sides have the same codes."""
    scale = x.abs().amax(-1) * (1.0 / 127.0)
    q = torch.nan_to_num((x / scale[..., None]).round()).clamp(-127, 127)
    return q.to(torch.int8), scale


def _values(s):
    """The whole pool as the values that it stands for, and its scales."""
    case = s["case"]
    shape = (-1, PAGE, case["kvh"], case["hd"])
    return [s["k"].view(shape) * s["ks"][..., None], s["v"].view(shape) * s["vs"][..., None],
            s["ks"], s["vs"]]


def _append(s):
    case = s["case"]
    seq, _, pos = _row_places(s)
    shape = (s["rows"], case["kvh"], case["hd"])
    k, v = s["kx"].float().view(shape), s["vx"].float().view(shape)
    if s["nw"] is not None:
        k = _head_norm(k, s["nw"])
    k = _rotate(k, s["cos"][pos], s["sin"][pos], case["inter"])
    page, slot = s["tables"].long()[seq, pos // PAGE] & 0xFFFF, pos % PAGE
    (k8, ks), (v8, vs) = _int8(k), _int8(v)
    s["k"][page, slot] = k8.view(s["rows"], -1)
    s["v"][page, slot] = v8.view(s["rows"], -1)
    s["ks"][page, slot], s["vs"][page, slot] = ks, vs
    return _values(s)


def _attn(s):
    case = s["case"]
    heads, kvh, hd, n = case["heads"], case["kvh"], case["hd"], case["new"]
    seqs, group = case["seqs"], case["heads"] // case["kvh"]
    pages = s["tables"].long() & 0xFFFF

    def cached(codes, scales):   # [seqs][kvh][keys][hd]
        x = codes.view(-1, PAGE, kvh, hd)[pages].float() * scales[pages][..., None]
        return x.view(seqs, -1, kvh, hd).transpose(1, 2)
    q = s["q"].float().view(-1, heads, hd)
    if s["qs"] is not None:
        q = q * s["qs"][..., None]
    row0, kv_len = s["row0"].long(), s["kv_len"].long()
    i = torch.arange(n, device=DEV)
    qp = q[(row0[:-1, None] + i).clamp_(max=s["rows"] - 1)]          # [seqs][n][heads][hd]
    qp = qp.view(seqs, n, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * n, hd)
    sc = (qp * hd ** -0.5) @ cached(s["k"], s["ks"]).transpose(2, 3)
    sc = sc.view(seqs, kvh, group, n, -1)
    j = torch.arange(sc.shape[-1], device=DEV)
    pos = (kv_len - (row0[1:] - row0[:-1]))[:, None] + i              # [seqs][n]
    seen = (j < kv_len[:, None, None]) & (j <= pos[:, :, None])
    if case["window"]:
        seen &= j > pos[:, :, None] - case["window"]
    sc.masked_fill_(~seen[:, None, None], float("-inf"))
    # rows behind a sequence's last one are padding here and may see no key
    sc -= sc.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    sc.exp_()
    total = sc.sum(-1, keepdim=True)
    o = sc.view(seqs, kvh, group * n, -1) @ cached(s["v"], s["vs"])
    o = o.view(seqs, kvh, group, n, hd) / total
    seq, at, _ = _row_places(s)
    return o.permute(0, 3, 1, 2, 4)[seq, at].to(s["o"].dtype).view(-1, heads * hd)


_PLAIN = {"tables": _tables, "rope": _rope, "append": _append, "attn": _attn}


# ------------------------------------------------------- the framework's calls
def _handle(s, ops):
    """The cache handle, which a program makes once."""
    if "kv" not in s:
        s["kv"] = ops.paged_kv(s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["case"]["kvh"],
                               s["case"]["hd"], PAGE)
    return s["kv"]


def _own(s):
    import __graft_entry__
    ops = __graft_entry__.load_package().ops
    case = s["case"]
    if case["op"] == "tables":
        ops.rope_tables(s["cos"], s["sin"], case["theta"], s["pos0"], case["scaling"],
                        case["factor"], case["orig"])
        return [s["cos"], s["sin"]]
    if case["op"] == "rope":
        ops.rope_rows(s["x"], s["pos"], s["cos"], s["sin"], s["out"], case["heads"], case["hd"],
                      nw=s["nw"], interleaved=case["inter"])
        return s["out"]
    kv, pages, mp = _handle(s, ops), s["k"].shape[0], s["tables"].shape[1]
    if case["op"] == "append":
        ops.paged_kv_append_batch(s["kx"], s["vx"], kv, pages, s["tables"], mp, s["row0"],
                                  s["kv_len"], case["seqs"], case["kvh"], case["hd"], nw=s["nw"],
                                  cos=s["cos"], sin=s["sin"], interleaved=case["inter"])
        return _values(s)
    if "ws" not in s:   # a program's own workspace, kept from step to step
        n = ops.attention_chunk_workspace_bytes(s["rows"], case["seqs"], case["new"], mp * PAGE,
                                                case["heads"], case["kvh"], case["hd"])
        s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    ops.attention_chunk_batch(s["q"], s["qs"], kv, pages, s["tables"], mp, s["row0"], s["kv_len"],
                              case["seqs"], case["new"], s["o"], None, case["heads"], case["kvh"],
                              case["hd"], case["causal"], case["window"], case["hd"] ** -0.5,
                              workspace=s["ws"])
    return s["o"]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------- in 64 bits
def _norm64(x, w):
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def _rotate64(x, cos, sin, inter):
    """Rotation of each pair as a complex product."""
    half = cos.shape[-1]
    turn = torch.complex(cos.double(), sin.double())[:, None]
    head = x[..., :2 * half]
    z = torch.complex(*((head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) if inter else
                        (head[..., :half].contiguous(), head[..., half:].contiguous()))) * turn
    y = torch.stack((z.real, z.imag), -1).flatten(-2) if inter else torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        rot, f = case["rot"], case["factor"]
        freqs, turn, a = [], rot / (2.0 * math.log(case["theta"])), 1.0
        for i in range(rot // 2):
            w = case["theta"] ** (-2.0 * i / rot)
            if case["scaling"] == "linear":
                w /= f
            elif case["scaling"] == "yarn":
                a = 0.1 * math.log(f) + 1.0
                lo = max(0, math.floor(turn * math.log(case["orig"] / (64.0 * math.pi))))
                hi = min(rot - 1, math.ceil(turn * math.log(case["orig"] / (2.0 * math.pi))))
                t = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
                w = (1.0 - t) * w + t * w / f
            freqs.append(w)
        p = torch.arange(s["pos0"], s["pos0"] + case["n"], device=DEV).double()
        z = torch.polar(torch.full((), a, dtype=torch.float64, device=DEV),
                        torch.outer(p, torch.tensor(freqs, dtype=torch.float64, device=DEV)))
        return [z.real.contiguous(), z.imag.contiguous()]
    hd = case["hd"]
    if case["op"] == "rope":
        x = s["x"].double().unflatten(-1, (-1, hd))
        x = _norm64(x, s["nw"].double()) if case["norm"] else x
        p = s["pos"].long()
        return _rotate64(x, s["cos"][p], s["sin"][p], case["inter"]).flatten(1)
    new, ctx = _lengths(case)
    kvh = case["kvh"]
    if case["op"] == "append":
        # K and V have no such values: a code next to a half is decided by float32 steps
        ks, vs, r = s["ks"].double(), s["vs"].double(), 0
        for b, (n, c) in enumerate(zip(new, ctx)):
            k = s["kx"][r:r + n].double().view(n, kvh, hd)
            k = _norm64(k, s["nw"].double()) if case["norm"] else k
            k = _rotate64(k, s["cos"][c:c + n], s["sin"][c:c + n], case["inter"])
            p = torch.arange(c, c + n, device=DEV)
            page = s["tables"][b, p // PAGE].long() & 0xFFFF
            ks[page, p % PAGE] = k.abs().amax(-1) / 127.0
            vs[page, p % PAGE] = s["vx"][r:r + n].double().view(n, kvh, hd).abs().amax(-1) / 127.0
            r += n
        return [None, None, ks, vs]
    if _pairs(case) * case["heads"] * hd > 2e12:
        return None
    out, r, group = [], 0, case["heads"] // kvh
    for b, (n, c) in enumerate(zip(new, ctx)):
        page = s["tables"][b, :-(-(n + c) // PAGE)].long() & 0xFFFF
        k = (s["k"][page].view(-1, kvh, hd).double() * s["ks"][page].view(-1, kvh, 1))[:n + c]
        v = (s["v"][page].view(-1, kvh, hd).double() * s["vs"][page].view(-1, kvh, 1))[:n + c]
        q = s["q"][r:r + n].double().view(n, kvh * group, hd)
        if s["qs"] is not None:
            q = q * s["qs"][r:r + n, :, None]
        key = torch.arange(n + c, device=DEV)
        row = torch.arange(c, c + n, device=DEV)[:, None]
        hidden = key > row
        if case["window"]:
            hidden |= key <= row - case["window"]
        heads = []
        for h in range(kvh * group):
            logits = q[:, h] @ k[:, h // group].T / math.sqrt(hd)
            logits.masked_fill_(hidden, -math.inf)
            heads.append(torch.softmax(logits, -1) @ v[:, h // group])
        out.append(torch.stack(heads, 1).flatten(1))
        r += n
    return torch.cat(out)
