"""Attention of several new tokens per sequence (bytes_amd.paged.paged_prompt_attn) against
its definition in 64 bits, and the operators of a serving step together."""
import pytest
import torch

import paged_oracle as O
import serving_oracle as S
from test_native_path_gpu import _both
from test_paged_blocks_gpu import KINDS, _dev, any_cache
from test_paged_gpu import _cos_sin, _make_cache, _rand, _table
from bytes_amd import paged as PG
from bytes_amd import paged_tables as PT

pytestmark = pytest.mark.gpu
F8, BF16, I8, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.int8, torch.int32
INF, NAN = float("inf"), float("nan")


def tolerance(out, mag, dots, D):
    """|error|: half a bf16 step of the result, 2^-8; each weight rounded to bf16, 2^-8 of the weighted
    |v| at most; scores off by D roundings of 2^-24 of their products and a few more where they are
    multiplied and shifted, in numerator and denominator; fp32 sums and exponentials 2^-16."""
    return 2.0 ** -8 * out.abs() + mag * (2.0 ** -8 + 2 * (D + 4) * 2.0 ** -24 * dots + 2.0 ** -16)


def _check(got, q, kc, vc, scale, ks, vs, table, lens, cu, window=None, sinks=0, rows=None):
    """All rows, or those of `rows`."""
    at = S.positions(q.shape[0], table, lens, cu, kc.shape[2])
    rows = list(range(q.shape[0])) if rows is None else rows
    want, mag, dots = S.attend_rows(q[rows], [at[r] for r in rows], kc, vc, scale, ks, vs, table, lens, window, sinks)
    got = got.double().cpu()[rows]
    bad = ~((got - want).abs() <= tolerance(want, mag, dots, q.shape[-1]))
    assert not bool(bad.any()), (bad.nonzero()[:5].tolist(), got[bad][:5], want[bad][:5])


def _batch(g, lens, new, bs, Hq, Hk, D, kind, layout="nhsd", extra=0):
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = any_cache(g, N, Hk, bs, D, kind, layout)
    cu = torch.tensor([0] + new).cumsum(0).to(I32)
    return _rand(g, int(cu[-1]) + extra, Hq, D), kc, vc, ks, vs, table, torch.tensor(lens, dtype=I32), cu


def _run(dev, q, kc, vc, ks, vs, table, n, cu, scale, **kw):
    return PG.paged_prompt_attn(_dev(q, dev), _dev(kc, dev), _dev(vc, dev), table.to(dev), n.to(dev), cu.to(dev), scale,
                                k_scale=_dev(ks, dev), v_scale=_dev(vs, dev), **kw)


def _wide(table, bs):
    """The table with entries for 2200 tokens more: what a row may see decides how a call is cut up."""
    return torch.cat([table, table.new_full((table.shape[0], 2200 // bs + 1), -1)], 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (28, 4, 128), (5, 5, 64), (40, 1, 128)])
@pytest.mark.parametrize("bs,layout", [(16, "nhsd"), (64, "nshd"), (1, "nhsd"), (24, "pair"), (48, "nhsd"), (200, "nhsd")])
def test_prompts(dev, kind, Hq, Hk, D, bs, layout):
    """Whole prompts, chunks, single tokens, none, more than a sequence holds; rows past the last
    sequence."""
    for i, (lens, new) in enumerate([([1], [1]), ([70, 0, 3, 129, 64], [70, 0, 1, 40, 64]), ([200, 33], [5, 40]), ([65], [65])]):
        g = torch.Generator().manual_seed(bs + i)
        q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind, layout, extra=3 * (i % 2))
        print(f"prompt {kind} Hq{Hq} Hk{Hk} D{D} bs{bs} {layout} lens {lens} new {new}", flush=True)
        out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5)
        assert out.shape == q.shape and out.dtype == BF16
        _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu)
        out = _run(dev, q, kc, vc, ks, vs, _wide(table, bs), n, cu, D ** -0.5)
        _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D,bs", [(160, 2, 64, 16), (160, 2, 64, 20), (256, 8, 64, 200), (80, 2, 128, 24), (256, 8, 128, 16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 2), (65, 1), (40, 65), (130, 4)])
def test_many_rows(dev, kind, Hq, Hk, D, bs, window, sinks):
    """Rows enough for tiles of 128 and of 256 that no one shares."""
    g = torch.Generator().manual_seed(Hq + bs)
    lens, new = [300, 90, 257, 40], [210, 90, 3, 1]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind, extra=2)
    kw = dict(window=window, sinks=sinks) if window else {}
    print(f"many rows {kind} Hq{Hq} D{D} bs{bs} {kw}", flush=True)
    out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5, **kw)
    rows = list(range(0, q.shape[0], 11)) + list(range(207, 212)) + list(range(298, q.shape[0]))
    _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu, window, sinks, rows)


@pytest.mark.parametrize("kind", ["bf16", I8])
@pytest.mark.parametrize("Hq,Hk,D,bs", [(14, 2, 64, 16), (6, 2, 128, 7), (8, 8, 128, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (64, 0), (65, 1), (63, 64), (40, 65), (130, 4), (2 ** 31, 7), (3, 10 ** 6)])
def test_prompts_within_a_window(dev, kind, Hq, Hk, D, bs, window, sinks):
    g = torch.Generator().manual_seed(window % 1000 + sinks % 1000)
    lens, new = [300, 90, 257, 40], [210, 90, 3, 1]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind)
    print(f"prompt window {window} sinks {sinks} {kind} Hq{Hq} D{D} bs{bs}", flush=True)
    out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5, window=window, sinks=sinks)
    rows = list(range(0, q.shape[0], 5)) + list(range(205, 215)) + list(range(298, q.shape[0]))
    _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu, window, sinks, rows)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,Hq,Hk,D,L,new,bs,window", [
    (2, 24, 8, 128, 9000, 8, 16, None), (1, 14, 2, 64, 20000, 3, 32, None), (3, 8, 1, 128, 7000, 40, 20, None),
    (1, 8, 2, 64, 12000, 5, 16, 6000), (70, 8, 2, 64, 1500, 2, 16, None), (1, 24, 8, 128, 972, 12, 16, None),
    (2, 14, 2, 64, 1468, 40, 20, None), (2, 14, 2, 64, 1800, 60, 32, 1500)])
def test_few_rows_over_long_contexts(dev, kind, B, Hq, Hk, D, L, new, bs, window):
    """Draft tokens: the keys of a row are shared out and joined."""
    g = torch.Generator().manual_seed(L)
    lens = [max(new, L - 101 * b) for b in range(B)]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, [new] * B, bs, Hq, Hk, D, kind)
    kw = dict(window=window, sinks=4) if window else {}
    out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5, **kw)
    some = [r for r in (0, new - 1, q.shape[0] // 2, q.shape[0] - 1)]
    _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu, window, kw.get("sinks", 0), some)


@pytest.mark.parametrize("Hq,Hk,D", [(160, 1, 64), (257, 1, 128), (384, 2, 64)])
def test_groups_of_more_heads_than_a_workgroup_has_rows(dev, Hq, Hk, D):
    """One token's heads are several row tiles: fewer tokens than tiles."""
    g = torch.Generator().manual_seed(Hq)
    for lens, new in (([1], [1]), ([40, 70], [3, 1])):
        q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, 16, Hq, Hk, D, "bf16")
        _check(_run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5), q, kc, vc, D ** -0.5, ks, vs, table, n, cu)


def test_long_prompt_rows(dev):
    """Rows all over a prompt of many tiles, against the decode of each as the last token."""
    g = torch.Generator().manual_seed(1)
    Hq, Hk, D, bs, L = 8, 2, 128, 16, 5000
    q, kc, vc, ks, vs, table, n, cu = _batch(g, [L], [L], bs, Hq, Hk, D, "bf16")
    for kw in ({}, dict(window=700, sinks=4)):
        out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5, **kw)
        rows = [0, 1, 63, 64, 127, 1000, 2047, 2048, 4095, 4998, 4999]
        _check(out, q, kc, vc, D ** -0.5, ks, vs, table, n, cu, kw.get("window"), kw.get("sinks", 0), rows)
        some = torch.arange(0, L, 97)
        ref = PG.paged_decode_attn(q[some, :, None].to(dev), kc.to(dev), vc.to(dev), table.expand(len(some), -1).to(dev),
                                   (some + 1).to(I32).to(dev), D ** -0.5, **kw)
        assert float((out[some.to(dev)] - ref[:, :, 0]).float().norm() / ref.float().norm()) < 0.005


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [16, 20])
@pytest.mark.parametrize("wide", [False, True])
def test_holes_garbage_and_lengths(dev, kind, bs, wide):
    """Blocks that are gone or do not exist, sequences without any, lengths past the table and below
    their new tokens; NaN and infinities in every row that no sequence holds."""
    g = torch.Generator().manual_seed(bs)
    Hq, Hk, D = 8, 2, 64
    lens, new = [200, 333, 90, 12, 640, 7], [60, 80, 90, 12, 50, 20]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind)
    table[0, 1], table[1, 3], table[1, 4] = -1, kc.shape[0], 2 ** 31 - 1
    table[2] = -1
    table[3, 0] = -2 ** 31
    if wide:
        table = _wide(table, bs)
    n[4] = table.shape[1] * bs + 30                  # the last 30 have no position
    held = torch.zeros(kc.shape[0], bs, dtype=torch.bool)
    for b in range(6):
        for _, i, o in O.held_tokens(table, n, kc.shape[0], bs, b):
            held[i, o] = True
    i, o = (~held).nonzero().T
    dirty = [kc.clone(), vc.clone()]
    for c, val in zip(dirty, (NAN, NAN if kind in ("fp8", F8) else INF)):
        if kind == I8:
            c[i, :, o] = -128
        else:
            f = c.float()
            f[i, :, o] = val
            c.view(torch.uint8).copy_(f.to(c.dtype).view(torch.uint8))
    scales = [ks, vs]
    if torch.is_tensor(ks):
        none = ~held.any(1)
        scales = [ks.clone(), vs.clone()]
        scales[0][none] = scales[1][none] = NAN
    for kw in ({}, dict(window=50, sinks=3)):
        out = _run(dev, q, *dirty, *scales, table, n, cu, 0.1, **kw)
        assert not bool(out[cu[2]:cu[4]].any()) and not bool(out[cu[5] - 30:cu[5]].any())
        assert not bool(out[cu[5]:cu[5] + 13].any())   # 20 new tokens of a sequence of 7
        _check(out, q, kc, vc, 0.1, ks, vs, table, n, cu, kw.get("window"), kw.get("sinks", 0))
    neg = torch.tensor([-5, 0, -2 ** 31 + 100, 0, -1, 0], dtype=I32)
    assert not bool(_run(dev, q, kc, vc, ks, vs, table, neg, cu, 0.1).any())


@pytest.mark.parametrize("kind", ["bf16", "fp8", F8])
@pytest.mark.parametrize("D,split,Hq,Hk", [(64, False, 4, 2), (128, False, 4, 2), (128, True, 4, 2), (128, True, 12, 2),
                                           (64, False, 256, 2), (128, False, 448, 8)])
def test_infinite_and_nan_values_reach_the_rows_that_see_them(dev, kind, D, split, Hq, Hk):
    """Values and keys that are infinite or NaN, in tiles that some rows see and others do not."""
    g = torch.Generator().manual_seed(D)
    bs = 16
    L, m = (6000, 15 if Hq == 4 else 20) if split else (150, 150)
    q, kc, vc, ks, vs, table, n, cu = _batch(g, [L], [m], bs, Hq, Hk, D, kind)
    bad = {L - m + 5: 3, L - m + 12: 40, L - 1: 63}   # position: dim
    at = lambda p: (int(table[0, p // bs]), p % bs)                          # noqa: E731
    f = vc.float()
    for i, (p, d) in enumerate(bad.items()):
        f[at(p)[0], :, at(p)[1], d] = NAN if kind != "bf16" or i == 1 else (INF if i == 0 else -INF)
    dirty = f.to(vc.dtype)
    for kw in ({}, dict(window=9, sinks=2)):
        out = _run(dev, q, kc, dirty, ks, vs, table, n, cu, 0.1, **kw).double().cpu()
        rows = list(range(0, m, 3 if split or Hq > 4 else 1)) + [m - 1]
        pos = S.positions(m, table, n, cu, bs)
        w, s = kw.get("window"), kw.get("sinks", 0)
        want, mag, dots = S.attend_rows(q[rows], [pos[r] for r in rows], kc, vc, 0.1, ks, vs, table, n, w, s)
        got = out[rows]
        hit = torch.zeros_like(got, dtype=torch.bool)
        for r, row in enumerate(rows):
            p = L - m + row
            for i, (t, d) in enumerate(bad.items()):
                if t <= p and (w is None or t > p - w or t < s):
                    hit[r, :, d] = True
                    x = f[at(t)[0], 0, at(t)[1], d]
                    assert bool((got[r, :, d].isnan() if x.isnan() else got[r, :, d] == x).all()), (row, t)
        assert bool(((got - want).abs() <= tolerance(want, mag, dots, D))[~hit].all())
    # a NaN key: its row's weight for those that see it, nothing for the others
    f = kc.float()
    p = L - m + 7
    f[at(p)[0], :, at(p)[1], 0] = NAN
    out = _run(dev, q, f.to(kc.dtype), vc, ks, vs, table, n, cu, 0.1, window=4)
    assert bool(out[7:11].isnan().all()) and not bool(out[:7].isnan().any()) and not bool(out[11:].isnan().any())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [16, 20])
def test_drafts_over_holes_and_garbage(dev, kind, bs):
    """Few rows over long tables, which are dealt out: blocks that are gone, sequences without any or without new
    tokens, lengths past the table and below zero, rows past the last sequence; the same twice and on a graph."""
    g = torch.Generator().manual_seed(bs + 5)
    Hq, Hk, D = 8, 2, 64
    lens, new = [5000, 333, 90, 12, 2640, 7, 3000, 1], [6, 8, 5, 0, 7, 9, 2, 1]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind, extra=4)
    table[0, 3:70], table[0, 100], table[1, 4] = -1, kc.shape[0], 2 ** 31 - 1
    table[2] = -1
    n[4] = table.shape[1] * bs + 3                   # its last 3 have no position
    n[6] = -5
    args = [_dev(x, dev) for x in (q, kc, vc, ks, vs, table, n, cu)]
    for kw in ({}, dict(window=1500, sinks=40), dict(window=2, sinks=0)):
        call = lambda: _run(dev, *args, 0.1, **kw)   # noqa: E731
        out = call()
        assert not bool(out[cu[-1]:].any()) and not bool(out[cu[2]:cu[3]].any()) and not bool(out[cu[6]:cu[7]].any())
        assert not bool(out[cu[5] - 3:cu[5]].any()) and not bool(out[cu[5]:cu[5] + 2].any())
        _check(out, q, kc, vc, 0.1, ks, vs, table, n, cu, kw.get("window"), kw.get("sinks", 0))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = call()
        for _ in range(2):
            graph.replay()
            assert torch.equal(again, call()) and torch.equal(again, out)


def test_large_scores(dev):
    """Scores far apart, running maxima that move in every tile and by little, scales that are negative, zero,
    large."""
    g = torch.Generator().manual_seed(3)
    Hq, Hk, D, bs, L = 4, 2, 64, 16, 400
    for kind in ("bf16", I8):
        q, kc, vc, ks, vs, table, n, cu = _batch(g, [L], [L], bs, Hq, Hk, D, kind)
        if kind == "bf16":
            for p in range(L):                       # keys that grow: the maximum moves on
                kc[int(table[0, p // bs]), :, p % bs] *= 0.05 * p ** 0.5
        for scale in (1.0, -0.7, 0.0, 1e-30, 8.0):
            for t in (table, _wide(table, bs)):
                out = _run(dev, q, kc, vc, ks, vs, t, n, cu, scale)
                _check(out, q, kc, vc, scale, ks, vs, table, n, cu, rows=list(range(0, L, 7)) + [L - 1])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cu", [[0, 40, 10, 64, 64], [5, 5, 9, 64, 70], [-3, 20, 2 ** 31 - 1, -2 ** 31, 30], [64, 64, 64, 64, 64],
                                [0, 10 ** 6, 0, 10 ** 6, 0]])
def test_offsets_that_are_no_offsets(dev, cu, wide):
    """Offsets that descend, overlap or leave the rows: results that nobody reads, and the next call is right."""
    g = torch.Generator().manual_seed(6)
    lens = [100, 6000 if wide else 90, 64, 300]
    q, kc, vc, ks, vs, table, n, good = _batch(g, lens, [20, 4, 30, 10], 16, 8, 2, 64, "bf16")
    args = [x.to(dev) for x in (q, kc, vc, table, n)]
    print(f"offsets {cu} {wide}", flush=True)
    PG.paged_prompt_attn(*args, torch.tensor(cu, dtype=I32, device=dev), 0.125)
    torch.cuda.synchronize()
    _check(PG.paged_prompt_attn(*args, good.to(dev), 0.125), q, kc, vc, 0.125, ks, vs, table, n, good)


def test_strided_queries_and_shared_blocks(dev):
    """Queries as views of a fused projection; sequences that share their first blocks; one block twice."""
    g = torch.Generator().manual_seed(4)
    Hq, Hk, D, bs = 8, 2, 64, 16
    lens, new = [100, 100, 80], [30, 20, 80]
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, "bf16")
    table[1, :4] = table[0, :4]
    table[2, 3] = table[2, 1]
    fused = _rand(g, int(cu[-1]), Hq + 2 * Hk, D)
    fused[:, :Hq] = q
    out = PG.paged_prompt_attn(fused.to(dev)[:, :Hq], kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), cu.to(dev), 0.125)
    _check(out, q, kc, vc, 0.125, 1.0, 1.0, table, n, cu)
    odd = torch.empty(int(cu[-1]), Hq, D + 1, dtype=BF16, device=dev)[..., 1:].copy_(q)      # rows off 16 bytes: copied
    assert torch.equal(PG.paged_prompt_attn(odd, kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), cu.to(dev), 0.125), out)


def test_native_path_and_wrapper_agree(dev, monkeypatch):
    g = torch.Generator().manual_seed(9)
    for kind in KINDS:
        for L, new in ((100, 37), (9000, 4)):
            q, kc, vc, ks, vs, table, n, cu = (_dev(x, dev) for x in _batch(g, [L, 50], [new, 9], 16, 8, 2, 64, kind))
            a = (q, kc, vc, table, n, cu, 0.125)
            sc = dict(k_scale=ks, v_scale=vs)
            _both(monkeypatch, PG.paged_prompt_attn, *a, **sc)
            _both(monkeypatch, PG.paged_prompt_attn, *a, window=30, sinks=4, **sc)
            _both(monkeypatch, PG.paged_prompt_attn, *a[:3], table.long(), *a[4:], taken=False, **sc)


def test_streams_share_nothing(dev):
    """Two calls at once on two streams, over caches of their own."""
    g = torch.Generator().manual_seed(2)
    work = []
    for i in range(2):
        x = [_dev(t, dev) for t in _batch(g, [9000, 3000], [6, 40], 16, 8, 2, 128, [I8, "bf16"][i])]
        work.append((x, dict(k_scale=x[3], v_scale=x[4])))
    call = lambda x, sc: (PG.paged_prompt_attn(x[0], *x[1:3], *x[5:], 0.09, **sc),       # noqa: E731
                          PG.paged_decode_attn(x[0][[0, 6], :, None], *x[1:3], *x[5:7], 0.09, window=5000, sinks=4, **sc))
    want = [call(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, w in zip(streams, work):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(call(*w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g_, w_ in zip(got, want) for a, b in zip(g_, w_))


# ---------------------------------------------------------------------------
# a serving loop of all of them
# ---------------------------------------------------------------------------
class Server:
    """Rows of requests over one pool: chunks of prompts, then drafts of which some are taken back."""
    B, W, bs, Hq, Hk, D, N, T = 5, 12, 16, 8, 2, 64, 48, 160

    def __init__(self, dev, kind, window, sinks):
        g = torch.Generator().manual_seed(11)
        self.dev, self.kind, self.window, self.sinks = dev, kind, window, sinks
        B, W, bs, Hq, Hk, D, N, T = self.B, self.W, self.bs, self.Hq, self.Hk, self.D, self.N, self.T
        self.state = PT.paged_pool(N, B, W, dev)
        if kind in (I8, F8):
            self.kc, self.vc = (torch.zeros(N, Hk, bs, D, dtype=torch.uint8, device=dev).view(kind) for _ in "kv")
            self.ks, self.vs = torch.zeros(N, Hk, device=dev), torch.zeros(N, Hk, device=dev)
        else:
            self.kc, self.vc = (t.to(dev) for t in _make_cache(g, N, Hk, bs, D, False))
            self.ks = self.vs = 1.0
        self.cos, self.sin = (t.to(dev) for t in _cos_sin(W * bs, D))
        # what the rows' tokens are made of: their keys, values and queries by (row, position)
        self.k, self.v, self.q = (_rand(g, B, W * bs, h, D).to(dev) for h in (Hk, Hk, Hq))
        self.keep, self.new = torch.zeros(B, dtype=I32, device=dev), torch.zeros(B, dtype=I32, device=dev)

    def step(self):
        """One step on the device alone: tables, append, attention of the new tokens."""
        table, lens, free, rng = self.state
        r = PT.paged_resize(table, lens, free, rng, self.new, self.T, self.bs, keep=self.keep, window=self.window, sinks=self.sinks)
        b, p = r.seqs.clamp(min=0).long(), r.positions.clamp(min=0).long()
        sc = dict(k_scale=self.ks, v_scale=self.vs)
        q = PG.paged_kv_append(self.k[b, p], self.v[b, p], self.kc, self.vc, table, lens, cu_seqlens=r.cu_seqlens,
                               q=self.q[b, p], cos=self.cos, sin=self.sin, **sc)
        see = dict(window=self.window, sinks=self.sinks) if self.window else {}
        rows = PG.paged_prompt_attn(q, self.kc, self.vc, table, lens, r.cu_seqlens, self.D ** -0.5, **sc, **see)
        last = (r.cu_seqlens[1:] - 1).clamp(min=0).long()
        one = PG.paged_decode_attn(q[last][:, :, None], self.kc, self.vc, table, lens, self.D ** -0.5, **sc, **see)
        return r, q, rows, one


STEPS = [([10 ** 6] * 5, [40, 25, 0, 70, 7]), ([10 ** 6] * 5, [40, 4, 33, 1, 4]), ([78, 27, 33, 71, 9], [4, 4, 4, 40, 4]),
         ([80, 0, 35, 108, 13], [4, 64, 4, 20, 4]), ([81, 64, 0, 0, 14], [4, 30, 40, 0, 4]), ([85, 90, 40, 0, 18], [1, 1, 1, 50, 1])]


@pytest.mark.parametrize("kind,window,sinks", [("bf16", None, 0), (I8, None, 0), (F8, 40, 4), ("bf16", 33, 16)])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(dev, kind, window, sinks, captured):
    """Chunked prompts, rejected drafts, requests that end and others in their rows, blocks that leave a window:
    every step's rows against their definition over what the cache holds, and against the tokens themselves.
    Captured: the same step as a graph, replayed."""
    sv = Server(dev, kind, window, sinks)
    step = sv.step
    if captured:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            sv.step()                                # nothing asked for: nothing changes
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sv.step()
        def step():
            graph.replay()
            return out
    for i, (keep, new) in enumerate(STEPS):
        sv.keep.copy_(torch.tensor(keep, dtype=I32)), sv.new.copy_(torch.tensor(new, dtype=I32))
        r, q, rows, one = step()
        torch.cuda.synchronize()
        table, lens, cu = sv.state[0].cpu(), sv.state[1].cpu(), r.cu_seqlens.cpu()
        assert r.granted.tolist() == new, i
        ks, vs = (x.cpu() if torch.is_tensor(x) else x for x in (sv.ks, sv.vs))
        raw = torch.uint8 if kind == F8 else sv.kc.dtype
        kc, vc = (c.view(raw).cpu().view(sv.kc.dtype) for c in (sv.kc, sv.vc))
        n = int(cu[-1])
        _check(rows, q.cpu(), kc, vc, sv.D ** -0.5, ks, vs, table, lens, cu, window, sinks,
               sorted(set(range(0, n, 6)) | set((cu[1:] - 1).clamp(min=0).tolist())) + [n, sv.T - 1])
        for b in range(sv.B):
            if new[b]:                               # the last new token, as decode and as prompt
                a, c = rows[cu[b + 1] - 1].float(), one[b, :, 0].float()
                assert float((a - c).norm() / c.norm()) < 0.01, (i, b)
            for p, blk, off in O.held_tokens(table, lens, sv.N, sv.bs, b)[::17]:       # the cache holds the rows' tokens
                y = O.rotate(sv.k[b, p].double().cpu(), sv.cos.cpu(), sv.sin.cpu(), p, False)[0]
                x = S.values(kc, ks)[blk, :, off]
                assert float((x - y).norm() / y.norm()) < {BF16: 0.004, I8: 0.02, F8: 0.04}[sv.kc.dtype], (i, b, p)
