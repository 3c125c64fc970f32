"""Paged dense caches (bytes_amd.paged) against 64-bit restatements of their
formulas, at the sizes, masks and layouts where they can go wrong."""
import math

import pytest
import torch

import paged_oracle as O
from test_native_path_gpu import _both
from bytes_amd import _lib
from bytes_amd import attention_kernels as AK
from bytes_amd import paged as PG
from bytes_amd import quest as QU
from bytes_amd import sparse as SP

pytestmark = pytest.mark.gpu
F8, BF16 = torch.float8_e4m3fn, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _rand(g, *shape):
    return torch.randn(*shape, generator=g).to(BF16)


def _same(a, b):
    """The same bytes."""
    r = torch.uint8 if a.dtype == F8 else torch.int16
    return torch.equal(a.contiguous().view(r).cpu(), b.contiguous().view(r).cpu())


def _table(g, lens, bs, spare=3, slack=2):
    """A table of distinct blocks in random order, -1 past each sequence: (table, number of blocks)."""
    need = [-(-n // bs) for n in lens]
    N = sum(need) + spare
    order = torch.randperm(N, generator=g).to(torch.int32)
    t = torch.full((len(lens), max(need) + slack), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t, N


def _make_cache(g, N, Hk, bs, D, fp8, layout="nhsd"):
    """(k, v) in the asked storage order, as [N, Hk, bs, D] views."""
    if layout == "nshd":
        k, v = _rand(g, N, bs, Hk, D).transpose(1, 2), _rand(g, N, bs, Hk, D).transpose(1, 2)
    elif layout == "pair":                           # keys and values of a block side by side
        kv = _rand(g, N, 2, Hk, bs, D)
        kv = (kv / 0.03).to(F8) if fp8 else kv
        return kv[:, 0], kv[:, 1]
    else:
        k, v = _rand(g, N, Hk, bs, D), _rand(g, N, Hk, bs, D)
    return ((k / 0.03).to(F8), (v / 0.03).to(F8)) if fp8 else (k, v)


def _cos_sin(P, R, base=10000.0):
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    a = torch.arange(P, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _keep_storage(t, dev):
    """t on the device with the same strides."""
    out = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev)
    r = torch.uint8 if t.dtype == F8 else BF16
    out.view(r).copy_(t.view(r))
    return out


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _check_append(dev, k, v, q, kc, vc, table, lens, cu, cos, sin, interleaved, meta, ks, vs):
    """One append against the formulas: stored rows within a rounding, every other
    byte of the caches as it was, the min / max of what is stored, the rotated queries."""
    N, Hk, bs, D = kc.shape
    T = k.shape[0]
    fp8 = kc.dtype == F8
    dk, dv = _keep_storage(kc, dev), _keep_storage(vc, dev)
    dmeta = tuple(m.to(dev) for m in meta) if meta is not None else None
    out = PG.paged_kv_append(k.to(dev), v.to(dev), dk, dv, table.to(dev), lens.to(dev),
                             cu_seqlens=None if cu is None else cu.to(dev), q=None if q is None else q.to(dev),
                             cos=None if cos is None else cos.to(dev), sin=None if sin is None else sin.to(dev),
                             interleaved=interleaved, meta=dmeta, k_scale=ks, v_scale=vs)
    gk, gv = dk.cpu(), dv.cpu()
    wk, wv = gk.clone(), gv.clone()
    raw = torch.uint8 if fp8 else BF16
    # a rounding to the cache's type is off by at most half a step; the rotation's three fp32
    # roundings and the division's one are each 2^-24 of the products' magnitudes
    half = 2.0 ** -4 if fp8 else 2.0 ** -8
    tiny = 2.0 ** -10 if fp8 else 0.0                   # half of e4m3's smallest step
    touched, want_q = {}, torch.zeros(T, 0 if q is None else q.shape[1], D, dtype=torch.float64)
    for t, b, p in O.placed(T, table, lens, cu, bs):
        if q is not None:
            y, mag = O.rotate(q[t].double(), cos, sin, p, interleaved)
            want_q[t] = y
            err = (out[t].double().cpu() - y).abs()
            assert bool((err <= 2.0 ** -8 * y.abs() + 2.0 ** -22 * mag).all()), (t, b, p)
        i, o = int(table[b, p // bs]), p % bs
        if not 0 <= i < N:
            continue
        y, mag = O.rotate(k[t].double(), cos, sin, p, interleaved)
        y, mag = y / ks, mag / ks
        if fp8:
            y = y.clamp(-448, 448)
        err = (gk[i, :, o].double() - y).abs()
        assert bool((err <= half * y.abs() + 2.0 ** -21 * mag + tiny).all()), (t, b, p)
        yv = v[t].double() / vs
        if fp8:
            yv = yv.clamp(-448, 448)
            err = (gv[i, :, o].double() - yv).abs()
            assert bool((err <= half * yv.abs() + 2.0 ** -21 * yv.abs() + tiny).all()), (t, b, p)
        else:
            assert torch.equal(gv[i, :, o], v[t])
        touched.setdefault(i, []).append(o)
        wk.view(raw)[i, :, o], wv.view(raw)[i, :, o] = kc.view(raw)[i, :, o], vc.view(raw)[i, :, o]
    assert _same(wk, kc) and _same(wv, vc), "rows that no new token names changed"
    if q is not None:
        rows = {t for t, _, _ in O.placed(T, table, lens, cu, bs)}
        for t in range(T):
            assert t in rows or not bool(out[t].any()), t
    else:
        assert out is None
    if meta is not None:
        for got, old, fold in ((dmeta[0].cpu(), meta[0], torch.amin), (dmeta[1].cpu(), meta[1], torch.amax)):
            want = old.clone()
            for i, offs in touched.items():
                new = fold(gk[i][:, sorted(offs)].float(), 1)
                want[i] = (new if 0 in offs else fold(torch.stack([new, old[i].float()]), 0)).to(BF16)
            assert torch.equal(got, want)
    return gk, gv, out


HEADS = [(14, 2, 64), (28, 4, 128), (8, 1, 128), (5, 5, 64)]


@pytest.mark.parametrize("Hq,Hk,D", HEADS)
@pytest.mark.parametrize("fp8,bs,rot,interleaved", [
    (False, 16, 64, False), (True, 16, 64, False), (False, 7, 32, True), (True, 32, 16, True), (False, 1, 48, False),
    (True, 128, 0, False)])
def test_append_single_tokens(dev, Hq, Hk, D, fp8, bs, rot, interleaved):
    """One token each: first rows, last rows of a block, block starts, an empty row, lengths past the table."""
    g = torch.Generator().manual_seed(Hq + bs)
    lens = [1, 2 * bs, 2 * bs + 1, 0, 3 * bs - 1, 77]
    table, N = _table(g, lens, bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8)
    qkv = _rand(g, len(lens), Hq + 2 * Hk, D)
    cos, sin = _cos_sin(table.shape[1] * bs, rot) if rot else (None, None)
    meta = (_rand(g, N, Hk, D), _rand(g, N, Hk, D))
    ks, vs = (0.03, 0.07) if fp8 else (1.0, 1.0)
    lens = torch.tensor(lens, dtype=torch.int32)
    a = (qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], qkv[:, :Hq], kc, vc)
    _check_append(dev, *a, table, lens, None, cos, sin, interleaved, meta, ks, vs)
    over = lens.clone()
    over[1], over[4] = table.shape[1] * bs + 5, 2 ** 31 - 1
    _check_append(dev, *a, table, over, None, cos, sin, interleaved, None, ks, vs)


@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (7, 3, 128)])
@pytest.mark.parametrize("fp8,bs,rot,interleaved,layout", [
    (False, 16, 64, False, "nhsd"), (True, 16, 32, True, "nshd"), (False, 5, 0, False, "pair"),
    (True, 64, 64, False, "pair"), (False, 100, 16, True, "nshd"), (False, 1, 64, False, "nhsd")])
def test_append_ragged_prompts(dev, Hq, Hk, D, fp8, bs, rot, interleaved, layout):
    """Prompts of 0 to 131 tokens behind 0 to 40 that are there already, rows past
    the last sequence, a hole in the table, more new tokens than the length says."""
    g = torch.Generator().manual_seed(D + bs)
    new = [131, 0, 1, 33, 16, 10, 64]
    past = [0, 5, 40, 3, 16, 0, 31]
    lens = [n + m for n, m in zip(new, past)]
    lens[5] = 4                                          # of ten new tokens the last four have a position
    table, N = _table(g, lens, bs)
    if (past[3] + 20) // bs < -(-lens[3] // bs):
        table[3, (past[3] + 20) // bs] = -1              # evicted
    table[6, past[6] // bs] = N + 2                      # no such block
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8, layout)
    T = sum(new) + 9
    qkv = _rand(g, T, Hq + 2 * Hk, D)
    cos, sin = _cos_sin(table.shape[1] * bs + 11, rot) if rot else (None, None)
    if rot:                                              # views of one table
        both = torch.cat([cos, sin], 1)
        cos, sin = both[:, :rot // 2], both[:, rot // 2:]
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    meta = (_rand(g, N, Hk, D), _rand(g, N, Hk, D))
    ks, vs = (0.05, 0.02) if fp8 else (1.0, 1.0)
    lens = torch.tensor(lens, dtype=torch.int32)
    a = (qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], qkv[:, :Hq], kc, vc, table, lens, cu, cos, sin, interleaved)
    _check_append(dev, *a, meta, ks, vs)
    _check_append(dev, a[0], a[1], None, *a[3:], None, ks, vs)


def test_append_many_sequences(dev):
    """More sequences than a wave has lanes, most of them with no new token."""
    g = torch.Generator().manual_seed(3)
    new = [(i * 7) % 5 if i % 3 == 0 else 0 for i in range(200)]
    lens = [n + (i * 13) % 30 for i, n in enumerate(new)]
    table, N = _table(g, lens, 8)
    kc, vc = _make_cache(g, N, 2, 8, 64, False)
    qkv = _rand(g, sum(new), 8, 64)
    cos, sin = _cos_sin(table.shape[1] * 8, 64)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    _check_append(dev, qkv[:, 4:6], qkv[:, 6:], qkv[:, :4], kc, vc, table, torch.tensor(lens, dtype=torch.int32), cu, cos,
                  sin, False, (_rand(g, N, 2, 64), _rand(g, N, 2, 64)), 1.0, 1.0)


def test_append_special_values(dev):
    """fp8 caches: values beyond the range and infinities become +-448, NaN stays NaN
    (and reaches the min / max); bf16 values are copied bit for bit."""
    g = torch.Generator().manual_seed(4)
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    k, v = _rand(g, 3, 1, 64), _rand(g, 3, 1, 64)
    k[0, 0, :6] = torch.tensor([1e4, -1e4, INF, -INF, NAN, 447.0], dtype=BF16)
    v[1, 0, :4] = torch.tensor([INF, NAN, -500.0, 2.0 ** -9], dtype=BF16)
    cu = torch.tensor([0, 3], dtype=torch.int32)
    for dt in (F8, BF16):
        kc, vc = (torch.zeros(2, 1, 16, 64, device=dev).to(dt) for _ in range(2))
        meta = tuple(torch.zeros(2, 1, 64, dtype=BF16, device=dev) for _ in range(2))
        PG.paged_kv_append(k.to(dev), v.to(dev), kc, vc, table.to(dev), lens.to(dev), cu_seqlens=cu.to(dev), meta=meta)
        gk, gv = kc[1, 0].float().cpu(), vc[1, 0].float().cpu()
        if dt == F8:
            assert gk[0, :4].tolist() == [448.0, -448.0, 448.0, -448.0] and math.isnan(gk[0, 4]) and gk[0, 5] == 448.0
            assert gv[1, 0] == 448.0 and math.isnan(gv[1, 1]) and gv[1, 2] == -448.0 and gv[1, 3] == 2.0 ** -9
        else:
            assert _same(kc[1, 0, :3].cpu(), k[:, 0]) and _same(vc[1, 0, :3].cpu(), v[:, 0])
        assert math.isnan(meta[0][1, 0, 4].item()) and math.isnan(meta[1][1, 0, 4].item())
        assert meta[1][1, 0, 0].item() == (448.0 if dt == F8 else k[0, 0, 0].float().item())


@pytest.mark.parametrize("fp8", [False, True])
def test_append_in_pieces_equals_at_once(dev, fp8):
    """A prompt at once, in two chunks, and token by token: the same bytes in caches and min / max."""
    g = torch.Generator().manual_seed(5)
    n, bs, Hq, Hk, D = 75, 16, 6, 2, 128
    table, N = _table(g, [n], bs)
    qkv = _rand(g, n, Hq + 2 * Hk, D).to(dev)
    cos, sin = (t.to(dev) for t in _cos_sin(table.shape[1] * bs, 128))
    sc = 0.03 if fp8 else 1.0
    got = []
    for cuts in ([0, n], [0, 37, n], list(range(n + 1))):
        kc, vc = (torch.zeros(N, Hk, bs, D, device=dev).to(F8 if fp8 else BF16) for _ in range(2))
        meta = tuple(torch.full((N, Hk, D), 7.0, dtype=BF16, device=dev) for _ in range(2))
        qs = []
        for a, b in zip(cuts, cuts[1:]):
            x = qkv[a:b]
            qs.append(PG.paged_kv_append(x[:, Hq:Hq + Hk], x[:, Hq + Hk:], kc, vc, table.to(dev),
                                         torch.tensor([b], dtype=torch.int32, device=dev),
                                         cu_seqlens=torch.tensor([0, b - a], dtype=torch.int32, device=dev) if b - a > 1 else None,
                                         q=x[:, :Hq], cos=cos, sin=sin, meta=meta, k_scale=sc, v_scale=sc))
        got.append((kc, vc, *meta, torch.cat(qs)))
    for other in got[1:]:
        for x, y in zip(got[0], other):
            assert _same(x, y)
    # the metadata of full blocks is quest_page_minmax's
    if not fp8:
        kmin, kmax = QU.quest_page_minmax(got[0][0], bs)
        for i in table[0, :n // bs].tolist():
            assert torch.equal(got[0][2][i], kmin[i, :, 0]) and torch.equal(got[0][3][i], kmax[i, :, 0])


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def _tol(out, mag, dots, D):
    """|error| of a decode's output: half a bf16 step of the result; weights as sums of two
    bf16 numbers, each rounding at most 2^-8 of what it rounds (2^-16 of the weighted |v|);
    scores off by D roundings of 2^-24 of their products, twice (numerator and
    denominator); fp32 sums and exponentials 2^-16."""
    return 2.0 ** -8 * out.abs() + mag * (2.0 ** -16 + 2 * D * 2.0 ** -24 * dots + 2.0 ** -16)


def _check_decode(dev, got, q, kc, vc, scale, ks, vs, table, lens, picks=None):
    want, mag, dots = O.attend(q, kc, vc, scale, ks, vs, table, lens, picks)
    got = got.double().cpu().reshape(want.shape)
    bad = ~((got - want).abs() <= _tol(want, mag, dots, q.shape[-1]))
    assert not bool(bad.any()), (bad.nonzero()[:5].tolist(), got[bad][:5], want[bad][:5])


LENS = [[1], [0, 3, 0], [130, 1, 64, 0, 257], [1000, 999], [31, 32, 33, 127, 128, 129, 15, 16, 17, 0]]


@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (28, 4, 128), (40, 2, 128), (3, 3, 64), (33, 1, 64), (24, 8, 128)])
@pytest.mark.parametrize("fp8,bs,layout", [(False, 16, "nhsd"), (True, 16, "nshd"), (False, 32, "pair"), (True, 64, "nhsd"),
                                           (False, 1, "nhsd"), (False, 24, "nshd"), (True, 7, "pair"),
                                           (False, 8, "nhsd"), (False, 1000, "nhsd")])
def test_decode(dev, Hq, Hk, D, fp8, bs, layout):
    for i, lens in enumerate(LENS):
        g = torch.Generator().manual_seed(100 * i + bs)
        table, N = _table(g, lens, bs)
        kc, vc = _make_cache(g, N, Hk, bs, D, fp8, layout)
        q = _rand(g, len(lens), Hq, 1, D)
        ks, vs = (0.03, 0.05) if fp8 else (1.0, 1.0)
        n = torch.tensor(lens, dtype=torch.int32)
        print(f"decode Hq{Hq} Hk{Hk} D{D} fp8={fp8} bs{bs} {layout} lens {lens}", flush=True)
        out = PG.paged_decode_attn(q.to(dev), _keep_storage(kc, dev), _keep_storage(vc, dev), table.to(dev), n.to(dev),
                                   D ** -0.5, k_scale=ks, v_scale=vs)
        assert out.shape == q.shape and out.dtype == BF16
        _check_decode(dev, out, q, kc, vc, D ** -0.5, ks, vs, table, n)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bs", [16, 20, 64])
def test_decode_holes_garbage_and_lengths(dev, fp8, bs):
    """Evicted blocks, blocks that do not exist, sequences without any, lengths past
    the table; NaN and infinities in every row that no sequence holds."""
    g = torch.Generator().manual_seed(bs)
    Hq, Hk, D = 8, 2, 128
    lens = [200, 333, 90, 5, 640]
    table, N = _table(g, lens, bs, slack=0)
    table[0, 1], table[1, 3], table[1, 4] = -1, N, 2 ** 31 - 1
    table[2] = -1
    table[3, 0] = -2 ** 31
    n = torch.tensor([200, 333, 90, 5, 10 ** 6], dtype=torch.int32)    # the last: all that its row names
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8)
    bad = torch.ones(N, bs, dtype=torch.bool)
    for b in range(5):
        for _, i, o in O.held_tokens(table, n, N, bs, b):
            bad[i, o] = False
    q = _rand(g, 5, Hq, 1, D)
    dirty = []
    for c, val in ((kc, NAN), (vc, NAN if fp8 else INF)):
        f = c.float()
        f[bad.nonzero()[:, 0], :, bad.nonzero()[:, 1]] = val
        dirty.append(f.to(c.dtype))
    out = PG.paged_decode_attn(q.to(dev), dirty[0].to(dev), dirty[1].to(dev), table.to(dev), n.to(dev), 0.1)
    assert not bool(out[2:4].any())                       # rows with nothing to attend to
    _check_decode(dev, out, q, kc, vc, 0.1, 1.0, 1.0, table, n)
    neg = torch.tensor([-5, 0, -2 ** 31, 0, -1], dtype=torch.int32)
    assert not bool(PG.paged_decode_attn(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), neg.to(dev), 0.1).any())
    # int64 tables and lengths; ids past 32 bits name no block
    wide = table.long()
    wide[1, 3] = 2 ** 32 + 1
    same = PG.paged_decode_attn(q.to(dev), dirty[0].to(dev), dirty[1].to(dev), wide.to(dev), n.long().to(dev), 0.1)
    assert torch.equal(same, out)


def test_decode_large_scores_and_nonfinite_rows(dev):
    """Scores of +-1e4 (one key takes all the weight), a NaN key of one sequence that
    stays in its sequence and KV head."""
    g = torch.Generator().manual_seed(9)
    lens = [300, 300]
    table, N = _table(g, lens, 16)
    kc, vc = _make_cache(g, N, 2, 16, 64, False)
    q = _rand(g, 2, 8, 1, 64)
    n = torch.tensor(lens, dtype=torch.int32)
    out = PG.paged_decode_attn((q * 100).to(dev), kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), 10.0)
    _check_decode(dev, out, q * 100, kc, vc, 10.0, 1.0, 1.0, table, n)
    kc[int(table[0, 3]), 1, 2, 5] = NAN
    out = PG.paged_decode_attn(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), 0.1).float().cpu()
    assert bool(out[0, 4:].isnan().all()) and bool(torch.isfinite(out[0, :4]).all()) and bool(torch.isfinite(out[1]).all())


@pytest.mark.parametrize("L", [100, 3000])
def test_infinite_values_that_take_part(dev, L):
    """An infinite value gives its infinity in its dim, whatever the weight (1 of a
    single token, one that two bf16 numbers hold exactly or not), and nothing elsewhere;
    both signs in one dim give NaN."""
    g = torch.Generator().manual_seed(L)
    lens, Hq, Hk, D, bs = [L, 1, L - 7], 8, 2, 64, 16
    table, N = _table(g, lens, bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    q = _rand(g, 3, Hq, 1, D)
    q[2] = 0.0                                            # equal weights
    n = torch.tensor(lens, dtype=torch.int32)
    vc[int(table[0, 2]), 0, 3, 5], vc[int(table[0, 4]), 0, 9, 6] = INF, -INF
    vc[int(table[0, 1]), 0, 0, 7], vc[int(table[0, 5]), 0, 0, 7] = INF, -INF
    vc[int(table[1, 0]), 1, 0, 63], vc[int(table[2, 3]), 1, 15, 0] = -INF, INF
    meta = tuple(t.to(dev) for t in _page_meta(kc, table, lens, bs))
    outs = [PG.paged_decode_attn(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), 0.1),
            PG.paged_quest_decode(q.to(dev), kc.to(dev), vc.to(dev), meta, table.to(dev), n.to(dev), L + bs, 0.1)]
    want, mag, dots = O.attend(q, kc, vc, 0.1, 1.0, 1.0, table, n)
    fin = torch.isfinite(want)
    for out in outs:
        got = out.double().cpu().reshape(want.shape)
        for b, h, d, x in ((0, 0, 5, INF), (0, 0, 6, -INF), (1, 4, 63, -INF), (2, 4, 0, INF)):
            assert bool((want[b, h:h + 4, d] == x).all()) and bool((got[b, h:h + 4, d] == x).all()), (b, h, d, got[b, h:h + 4, d])
        assert bool(got[0, :4, 7].isnan().all())
        assert int((~fin).sum()) == 5 * 4 and bool(((got - want).abs() <= _tol(want, mag, dots, D))[fin].all())


@pytest.mark.parametrize("B,Hq,Hk,D,L,bs,fp8", [(3, 28, 4, 128, 9001, 16, False), (1, 14, 2, 64, 40000, 16, False),
                                                (70, 8, 8, 64, 700, 16, True), (150, 4, 1, 128, 300, 12, False)])
def test_decode_long_and_wide(dev, B, Hq, Hk, D, L, bs, fp8):
    """Long contexts, more sequences than a wave has lanes; equal to the dense decode of
    the same rows within both kernels' roundings."""
    g = torch.Generator().manual_seed(L)
    lens = [max(0, L - (L // (b + 2)) * (b % 3) - 7 * b) if b % 11 != 5 else 0 for b in range(B)]
    table, N = _table(g, lens, bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8)
    q = _rand(g, B, Hq, 1, D)
    n = torch.tensor(lens, dtype=torch.int32)
    dq, dk, dv, dt = q.to(dev), kc.to(dev), vc.to(dev), table.to(dev)
    out = PG.paged_decode_attn(dq, dk, dv, dt, n.to(dev), D ** -0.5, k_scale=0.03 if fp8 else 1.0)
    raw = torch.uint8 if fp8 else BF16
    for b in list(range(0, B, max(1, B // 12))) + [5 % B]:
        if not lens[b]:
            assert not bool(out[b].any())
            continue
        ids = dt[b, :-(-lens[b] // bs)].long()
        kk, vv = (c.view(raw)[ids].view(c.dtype).transpose(0, 1).reshape(1, Hk, -1, D)[:, :, :lens[b]].double()
                  for c in (dk, dv))
        kk = (kk * (0.03 if fp8 else 1.0)).cpu().repeat_interleave(Hq // Hk, 1)
        vv = vv.cpu().repeat_interleave(Hq // Hk, 1)
        qq = q[b:b + 1].double()
        p = torch.softmax((qq * kk).sum(-1) * D ** -0.5, -1)[..., None]
        want, mag = (p * vv).sum(2), (p * vv.abs()).sum(2)
        dots = ((qq.abs() * kk.abs()).sum(-1) * D ** -0.5).amax(-1, keepdim=True)
        err = (out[b].double().cpu().reshape(want.shape) - want).abs()
        assert bool((err <= _tol(want, mag, dots, D)).all()), b


# ---------------------------------------------------------------------------
# page bounds and page-sparse decode
# ---------------------------------------------------------------------------
def _page_meta(kc, table, lens, bs):
    N, Hk, _, D = kc.shape
    kmin, kmax = torch.full((N, Hk, D), NAN).to(BF16), torch.full((N, Hk, D), NAN).to(BF16)
    for b in range(table.shape[0]):
        by = {}
        for _, i, o in O.held_tokens(table, lens, N, bs, b):
            by.setdefault(i, []).append(o)
        for i, offs in by.items():
            r = kc[i].float()[:, offs]
            kmin[i], kmax[i] = r.amin(1).to(BF16), r.amax(1).to(BF16)
    return kmin, kmax


def _quest_inputs(Hq, Hk, D, bs, lens, fp8, seed=0):
    g = torch.Generator().manual_seed(seed + bs)
    table, N = _table(g, lens, bs)
    if len(lens) > 2 and table.shape[1] > 4:
        table[2, 1] = -1
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8)
    n = torch.tensor(lens, dtype=torch.int32)
    return _rand(g, len(lens), Hq, 1, D), kc, vc, table, n, _page_meta(kc, table, n, bs)


QLENS = [[1], [500, 0, 333, 90], [2100, 64]]


@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (7, 1, 128), (6, 6, 64), (40, 2, 128)])
@pytest.mark.parametrize("bs,local_w,fp8", [(16, 0, False), (16, 1, True), (32, 40, False), (5, 3, False), (64, 100, True)])
def test_page_scores(dev, Hq, Hk, D, bs, local_w, fp8):
    for lens in QLENS:
        q, kc, vc, table, n, meta = _quest_inputs(Hq, Hk, D, bs, lens, fp8)
        got = PG.paged_page_scores(q.to(dev), tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), bs, 0.3,
                                   local_w=local_w).cpu().double()
        want, mag = O.bounds(q, *meta, table, n, bs, 0.3, local_w)
        fin = torch.isfinite(want)
        assert torch.equal(got[~fin], want[~fin])
        # one rounding to fp32, and 64-bit sums of D terms in either order
        assert bool(((got - want).abs()[fin] <= (2.0 ** -24 * want.abs() + 2 * D * 2.0 ** -53 * mag)[fin]).all())


@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (7, 1, 128), (40, 2, 128)])
@pytest.mark.parametrize("bs,kb,local_w,fp8", [(16, 64, 0, False), (16, 1, 1, True), (32, 100, 40, False), (5, 33, 0, False),
                                               (64, 128, 0, True), (16, 10 ** 6, 0, False)])
def test_quest_decode(dev, Hq, Hk, D, bs, kb, local_w, fp8):
    for lens in QLENS:
        q, kc, vc, table, n, meta = _quest_inputs(Hq, Hk, D, bs, lens, fp8, seed=1)
        ks, vs = (0.03, 0.05) if fp8 else (1.0, 1.0)
        a = (q.to(dev), kc.to(dev), vc.to(dev), tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), kb, D ** -0.5)
        print(f"quest Hq{Hq} Hk{Hk} D{D} bs{bs} kb{kb} fp8={fp8} lens {lens}", flush=True)
        out, pages = PG.paged_quest_decode(*a, local_w=local_w, k_scale=ks, v_scale=vs, return_pages=True)
        bound, _ = O.bounds(q, *meta, table, n, bs, D ** -0.5 * ks, local_w)
        npick = min(-(-kb // bs), table.shape[1])
        want = bound.float().argsort(dim=-1, descending=True, stable=True)[..., :npick].sort(-1).values
        assert pages.dtype == torch.int32 and torch.equal(pages.cpu().long(), want)
        picks = [[set(want[b, h].tolist()) for h in range(Hq)] for b in range(len(lens))]
        _check_decode(dev, out, q, kc, vc, D ** -0.5, ks, vs, table, n, picks)
        alone = PG.paged_quest_decode(*a, local_w=local_w, k_scale=ks, v_scale=vs)
        assert torch.equal(alone, out)


def test_quest_ties_and_nonfinite_bounds(dev):
    """Equal bounds go to the lowest place, whatever the sum's order; a NaN bound ranks
    first, as in topk_indices."""
    bs, W, Hk, D = 16, 40, 1, 64
    g = torch.Generator().manual_seed(2)
    kc, vc = _make_cache(g, W, Hk, bs, D, False)
    kmin = torch.randint(-2, 1, (W, Hk, D), generator=g).to(BF16)
    kmax = kmin + torch.randint(0, 2, (W, Hk, D), generator=g).to(BF16)
    kmin[5:20], kmax[5:20] = kmin[4], kmax[4]
    kmax[33, 0, 3] = NAN
    q = torch.randint(-2, 3, (1, 4, 1, D), generator=g).to(BF16)
    q[..., 3] = 1.0
    table, n = torch.arange(W, dtype=torch.int32)[None], torch.tensor([W * bs], dtype=torch.int32)
    meta = (kmin.to(dev), kmax.to(dev))
    bound = PG.paged_page_scores(q.to(dev), meta, table.to(dev), n.to(dev), bs, 1.0)
    assert bool(bound[..., 33].isnan().all()) and bool((bound[..., 4:20] == bound[..., 4:5]).all())
    for kb in (16, 80, 300):
        out, pages = PG.paged_quest_decode(q.to(dev), kc.to(dev), vc.to(dev), meta, table.to(dev), n.to(dev), kb, 1.0,
                                           return_pages=True)
        assert torch.equal(pages, SP.topk_indices(bound, -(-kb // bs), sorted=False))
        assert bool((pages == 33).any(-1).all())


@pytest.mark.parametrize("bs,L", [(4, 20001), (2, 25000), (1, 16384), (1, 16700)])
def test_quest_many_pages(dev, bs, L):
    """More pages than a workgroup of the attention selects from (a launch of its own up
    to 16384, the top-k above)."""
    g = torch.Generator().manual_seed(8)
    Hq, Hk, D = 4, 2, 64
    kb = 100 * bs
    table, N = _table(g, [L, 777, 0], bs, slack=0)
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    n = torch.tensor([L, 777, 0], dtype=torch.int32)
    meta = _page_meta(kc, table, n, bs)
    q = _rand(g, 3, Hq, 1, D)
    a = (q.to(dev), kc.to(dev), vc.to(dev), tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), kb, 0.125)
    out, pages = PG.paged_quest_decode(*a, return_pages=True)
    alone = PG.paged_quest_decode(*a)
    qd = q.double().reshape(3, Hk, Hq // Hk, D)
    ids = table.clamp(min=0).long()
    kmin, kmax = (m.double()[ids].permute(0, 2, 3, 1) for m in meta)
    b = (qd.clamp(min=0) @ kmax.nan_to_num(0) + qd.clamp(max=0) @ kmin.nan_to_num(0)).reshape(3, Hq, -1) * 0.125
    b = b.float().masked_fill((torch.arange(table.shape[1]) * bs >= n[:, None])[:, None], -INF)
    want = b.argsort(dim=-1, descending=True, stable=True)[..., :100].sort(-1).values
    assert torch.equal(pages.cpu().long(), want) and torch.equal(alone, out)
    _check_decode(dev, out, q, kc, vc, 0.125, 1.0, 1.0, table, n,
                  [[set(want[i, h].tolist()) for h in range(Hq)] for i in range(3)])


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------
def _serve(dev, fp8=False, steps=6):
    """Prompts, then decode steps, of a padded batch through all operators."""
    g = torch.Generator().manual_seed(12)
    B, Hq, Hk, D, bs, W = 4, 8, 2, 128, 16, 40
    new = [97, 16, 300, 0]
    table = torch.randperm(B * W + 5, generator=g)[:B * W].reshape(B, W).to(torch.int32)
    table[3] = -1
    sc = 0.04 if fp8 else 1.0
    cos, sin = (t.to(dev) for t in _cos_sin(W * bs, 128))
    kc, vc = (torch.full((B * W + 5, Hk, bs, D), NAN, device=dev).to(F8 if fp8 else BF16) for _ in range(2))
    meta = tuple(torch.full((B * W + 5, Hk, D), NAN, dtype=BF16, device=dev) for _ in range(2))
    lens = torch.tensor(new, dtype=torch.int32, device=dev)
    table = table.to(dev)
    x = _rand(g, sum(new), Hq + 2 * Hk, D).to(dev)
    kw = dict(cos=cos, sin=sin, meta=meta, k_scale=sc, v_scale=sc)
    PG.paged_kv_append(x[:, Hq:Hq + Hk], x[:, Hq + Hk:], kc, vc, table, lens,
                       cu_seqlens=torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev), q=x[:, :Hq], **kw)
    live = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device=dev)
    xs = [_rand(g, B, Hq + 2 * Hk, D).to(dev) for _ in range(steps)]

    def step(x):
        lens.add_(live)
        q = PG.paged_kv_append(x[:, Hq:Hq + Hk], x[:, Hq + Hk:], kc, vc, table, lens, q=x[:, :Hq], **kw).unsqueeze(2)
        full = PG.paged_decode_attn(q, kc, vc, table, lens, D ** -0.5, k_scale=sc, v_scale=sc)
        part = PG.paged_quest_decode(q, kc, vc, meta, table, lens, 64, D ** -0.5, local_w=16, k_scale=sc, v_scale=sc)
        whole = PG.paged_quest_decode(q, kc, vc, meta, table, lens, W * bs, D ** -0.5, k_scale=sc, v_scale=sc)
        return q, full, part, whole

    return step, xs, kc, vc, meta, table, lens, sc


@pytest.mark.parametrize("fp8", [False, True])
def test_serving_loop(dev, fp8):
    step, xs, kc, vc, meta, table, lens, sc = _serve(dev, fp8)
    for x in xs:
        q, full, part, whole = step(x)
    a = (q.cpu(), kc.cpu(), vc.cpu(), 128 ** -0.5, sc, sc, table.cpu(), lens.cpu())
    _check_decode(dev, full, *a)
    _check_decode(dev, whole, *a)
    bound, _ = O.bounds(q.cpu(), meta[0].cpu(), meta[1].cpu(), table.cpu(), lens.cpu(), 16, 128 ** -0.5 * sc, 16)
    best = bound.float().argsort(dim=-1, descending=True, stable=True)[..., :4]
    _check_decode(dev, part, *a, [[set(best[b, h].tolist()) for h in range(8)] for b in range(4)])
    assert not bool(full[3].any()) and not bool(part[3].any())
    if not fp8:                                          # the contiguous operator on the same rows
        b, n = 2, int(lens[2])
        kk, vv = (c[table[b, :-(-n // 16)].long()].transpose(0, 1).reshape(1, 2, -1, 128)[:, :, :n].contiguous()
                  for c in (kc, vc))
        dense = AK.decode_attn_bf16(q[b:b + 1], kk, vv, 128 ** -0.5).float()
        assert float((dense - full[b:b + 1].float()).abs().max()) <= 2e-2


def test_serving_loop_captured(dev):
    """The whole step as a graph: replayed while lengths grow past block ends, eager work
    between the replays, equal to the eager loop bit for bit."""
    step, xs, kc, vc, meta, table, lens, _ = _serve(dev, steps=20)
    want = [tuple(t.clone() for t in step(x)) for x in xs]
    wk, wm = kc.clone(), meta[0].clone()
    step2, xs2, kc2, vc2, meta2, table2, lens2, _ = _serve(dev, steps=20)
    buf = xs2[0].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        keep = lens2.clone()
        step2(buf)                                       # warm-up: writes what the first replay writes again
        lens2.copy_(keep)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step2(buf)
    for i, x in enumerate(xs2):
        buf.copy_(x)
        graph.replay()
        if i % 3 == 0:
            torch.cuda.synchronize()
            torch.randn(1000, device=dev).sort()
        for w, r in zip(want[i], got):
            assert torch.equal(w, r), i
    assert torch.equal(lens, lens2) and _same(wk, kc2) and _same(wm, meta2[0])


def test_streams_share_nothing(dev):
    """Decodes queued on two streams at once, each result its own stream's."""
    g = torch.Generator().manual_seed(21)
    lens = [5000, 3001, 17]
    table, N = _table(g, lens, 16)
    kc, vc = _make_cache(g, N, 4, 16, 128, False)
    n = torch.tensor(lens, dtype=torch.int32).to(dev)
    meta = tuple(m.to(dev) for m in _page_meta(kc, table, torch.tensor(lens), 16))
    kc, vc, table = kc.to(dev), vc.to(dev), table.to(dev)
    qs = [_rand(g, 3, 28, 1, 128).to(dev) for _ in range(2)]
    run = lambda q: (PG.paged_decode_attn(q, kc, vc, table, n, 0.09),       # noqa: E731
                     PG.paged_quest_decode(q, kc, vc, meta, table, n, 512, 0.09))
    want = [run(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r[0], want[i][0]) and torch.equal(r[1], want[i][1])


def test_native_path_and_wrapper_agree(dev, monkeypatch):
    """The native call path and the Python wrapper: the same bits, for the layouts either takes."""
    g = torch.Generator().manual_seed(31)
    B, Hq, Hk, D, bs = 3, 14, 2, 64, 16
    lens = [300, 17, 0]
    for fp8 in (False, True):
        table, N = _table(g, lens, bs)
        kc, vc = (c.to(dev) for c in _make_cache(g, N, Hk, bs, D, fp8))
        n, table = torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev)
        sc = 0.03 if fp8 else 1.0
        meta = tuple(m.to(dev) for m in _page_meta(kc.cpu(), table.cpu(), torch.tensor(lens), bs))
        qkv = _rand(g, B, Hq + 2 * Hk, D).to(dev)
        q = qkv[:, :Hq].unsqueeze(2)                      # a strided view
        ks = dict(k_scale=sc, v_scale=sc)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, table, n, 0.125, **ks)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, table, n, **ks)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, table.long(), n, 0.125, taken=False, **ks)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, table[:, :8], n, 1, **ks)      # a view of a wider table
        wide = torch.zeros(B, Hq, 1, D + 1, dtype=BF16, device=dev)[..., 1:]
        _both(monkeypatch, PG.paged_decode_attn, wide, kc, vc, table, n, 0.125, taken=False, **ks)
        a = (q, kc, vc, meta, table, n)
        _both(monkeypatch, PG.paged_quest_decode, *a, 64, 0.125, **ks)
        _both(monkeypatch, PG.paged_quest_decode, *a, 33, 0.125, local_w=20, **ks)
        _both(monkeypatch, PG.paged_quest_decode, *a, 64, 0.125, return_pages=True, taken=False, **ks)
        cos, sin = (x.to(dev) for x in _cos_sin(table.shape[1] * bs, 32))
        x = (qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], kc, vc, table, n)
        kw = dict(q=qkv[:, :Hq], cos=cos, sin=sin, meta=meta, **ks)
        _both(monkeypatch, PG.paged_kv_append, *x, **kw)
        _both(monkeypatch, PG.paged_kv_append, *x, interleaved=True, **{**kw, "meta": None})
        cu = torch.tensor([0, 2, 3, 3], dtype=torch.int32, device=dev)
        _both(monkeypatch, PG.paged_kv_append, *x, cu_seqlens=cu, **kw)
        _both(monkeypatch, PG.paged_kv_append, *x, cu_seqlens=cu.long(), taken=False, **kw)
        got = []
        for native in (_lib.native(), _lib._NoNative()):
            monkeypatch.setattr(_lib, "_native", native)
            k2, v2, m2 = kc.clone(), vc.clone(), tuple(m.clone() for m in meta)
            assert PG.paged_kv_append(*x[:2], k2, v2, table, n, cos=cos, sin=sin, meta=m2, **ks) is None
            got.append((k2, v2, *m2))
            monkeypatch.undo()
        for u, v in zip(*got):
            assert _same(u, v)
        for bad in ((q, kc, vc[:, :1], table, n), (q, kc, vc, table[:2], n), (q, kc, vc, table, n.float()),
                    (q[..., :32], kc, vc, table, n), (q.half(), kc, vc, table, n), (q.cpu(), kc, vc, table, n),
                    (q, kc, vc, table.cpu(), n), (q, kc.transpose(2, 3), vc, table, n)):
            with pytest.raises(ValueError):
                PG.paged_decode_attn(*bad, 0.125, **ks)


def test_shared_and_repeated_blocks(dev):
    """Sequences that share a prefix, one table row for all (stride 0), a block named twice by one sequence."""
    g = torch.Generator().manual_seed(41)
    Hq, Hk, D, bs = 8, 2, 128, 16
    kc, vc = _make_cache(g, 40, Hk, bs, D, False)
    q = _rand(g, 4, Hq, 1, D)
    row = torch.randperm(40, generator=g)[:30].to(torch.int32)
    row[7] = row[3]
    n = torch.tensor([480, 100, 1, 301], dtype=torch.int32)
    shared = row.to(dev)[None].expand(4, 30)
    out = PG.paged_decode_attn(q.to(dev), kc.to(dev), vc.to(dev), shared, n.to(dev), 0.09)
    _check_decode(dev, out, q, kc, vc, 0.09, 1.0, 1.0, row[None].expand(4, 30), n)
    meta = QU.quest_page_minmax(kc.to(dev), bs)
    meta = tuple(m[:, :, 0] for m in meta)
    got, pages = PG.paged_quest_decode(q.to(dev), kc.to(dev), vc.to(dev), meta, shared, n.to(dev), 96, 0.09, return_pages=True)
    picks = [[set(pages[b, h].tolist()) for h in range(Hq)] for b in range(4)]
    _check_decode(dev, got, q, kc, vc, 0.09, 1.0, 1.0, row[None].expand(4, 30), n, picks)


@pytest.mark.parametrize("fp8", [False, True])
def test_offsets_past_32_bits(dev, fp8):
    """Blocks more than 2^32 bytes and 2^31 elements into the cache: append, decode and page-sparse decode."""
    Hq, Hk, D, bs = 8, 8, 128, 128
    per = Hk * bs * D
    N = 2 ** 31 // per * (2 if fp8 else 1) + 6
    dt = F8 if fp8 else BF16
    kc = torch.empty(N, Hk, bs, D, dtype=dt, device=dev)
    vc = torch.empty(N, Hk, bs, D, dtype=dt, device=dev)
    g = torch.Generator().manual_seed(51)
    table = torch.tensor([[N - 1, 0, N - 3], [N - 2, N - 5, -1]], dtype=torch.int32)
    lens, new = [300, 140], [300, 139]
    qkv = _rand(g, sum(new), Hq + 2 * Hk, D)
    meta = tuple(torch.zeros(N, Hk, D, dtype=BF16, device=dev) for _ in range(2))
    used = table[table >= 0].unique().long()
    for c in (kc, vc):
        c.view(torch.uint8)[used.to(dev)] = 0
    cu = torch.tensor([0, 300, 439], dtype=torch.int32)
    n = torch.tensor(lens, dtype=torch.int32)
    x = qkv.to(dev)
    q = PG.paged_kv_append(x[:, Hq:Hq + Hk], x[:, Hq + Hk:], kc, vc, table.to(dev), n.to(dev), cu_seqlens=cu.to(dev),
                           q=x[:, :Hq], meta=meta)
    assert torch.equal(q, x[:, :Hq])                      # no rotation asked for
    small_k, small_v = (torch.zeros(N if N < 8 else 8, Hk, bs, D).to(dt) for _ in range(2))
    place = {int(b): i for i, b in enumerate(used)}
    for b, i in place.items():
        small_k.view(torch.uint8)[i], small_v.view(torch.uint8)[i] = (c[b].view(torch.uint8).cpu() for c in (kc, vc))
    st = torch.tensor([[place.get(int(b), -1) for b in r] for r in table], dtype=torch.int32)
    for t, b, p in O.placed(sum(new), table, n, cu, bs):
        row = small_v[int(st[b, p // bs]), :, p % bs].float()
        assert torch.equal(row, qkv[t, Hq + Hk:].to(dt).float()), (t, b, p)
    dq = q[[299, 438]].unsqueeze(2)
    out = PG.paged_decode_attn(dq, kc, vc, table.to(dev), n.to(dev), 0.09)
    _check_decode(dev, out, dq.cpu(), small_k, small_v, 0.09, 1.0, 1.0, st, n)
    out, pages = PG.paged_quest_decode(dq, kc, vc, meta, table.to(dev), n.to(dev), 2 * bs, 0.09, return_pages=True)
    picks = [[set(pages[b, h].tolist()) for h in range(Hq)] for b in range(2)]
    _check_decode(dev, out, dq.cpu(), small_k, small_v, 0.09, 1.0, 1.0, st, n, picks)


# ---------------------------------------------------------------------------
# infinite values, weights and stored keys
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("B,Hk,L", [(1, 2, 700), (1, 2, 2100), (1, 2, 9000), (30, 8, 3000)])
def test_infinite_values_in_any_part(dev, B, Hk, L):
    """Infinite values in the first, a middle and the last of 2 to more than 32 joined
    parts (a unit's tokens are split over workgroups): that infinity, in its dim alone."""
    g = torch.Generator().manual_seed(L)
    Hq, D, bs = 2 * Hk, 64, 16
    lens = [L - 40 * b for b in range(B)]
    table, N = _table(g, lens, bs, slack=max(2, 1200 // bs - L // bs))     # past what one workgroup takes alone
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    q, n = _rand(g, B, Hq, 1, D), torch.tensor(lens, dtype=torch.int32)
    at = {}
    for b in range(B):
        for hk in range(Hk):
            for i, p in enumerate((0, 5, lens[b] // 3, lens[b] // 2, lens[b] - 140, lens[b] - 2, lens[b] - 1)):
                x = INF if (i + hk) % 2 else -INF
                vc[int(table[b, p // bs]), hk, p % bs, 3 * i + hk] = x
                at[b, hk, 3 * i + hk] = x
    meta = tuple(t.to(dev) for t in _page_meta(kc, table, lens, bs))
    a = (q.to(dev), kc.to(dev), vc.to(dev))
    t = (table.to(dev), n.to(dev))
    outs = {"decode": PG.paged_decode_attn(*a, *t, 0.1), "quest": PG.paged_quest_decode(*a, meta, *t, L + bs, 0.1)}
    some = [0] if B == 1 else [0, B // 2, B - 1]
    want, mag, dots = O.attend(q[some], kc, vc, 0.1, 1.0, 1.0, table[some], n[some])
    for name, out in outs.items():
        got = out.double().cpu().reshape(B, Hq, D)
        for (b, hk, d), x in at.items():
            assert bool((got[b, 2 * hk:2 * hk + 2, d] == x).all()), (name, b, hk, d, x, got[b, 2 * hk:2 * hk + 2, d])
        assert int((~torch.isfinite(got)).sum()) == 2 * len(at), name
        fin = torch.isfinite(want)
        assert bool(((got[some] - want).abs() <= _tol(want, mag, dots, D))[fin].all()), name


def test_infinite_values_of_selected_pages(dev):
    """The same where the pages are selected: the newest one, kept by the window, is in the last run."""
    g = torch.Generator().manual_seed(77)
    Hq, Hk, D, bs, L, kb = 4, 2, 64, 16, 5000, 1600
    table, N = _table(g, [L], bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    q, n = _rand(g, 1, Hq, 1, D), torch.tensor([L], dtype=torch.int32)
    for d, p, x in ((7, L - 1, INF), (9, L - 8, -INF)):
        vc[int(table[0, p // bs]), :, p % bs, d] = x
    meta = tuple(t.to(dev) for t in _page_meta(kc, table, [L], bs))
    out, pages = PG.paged_quest_decode(q.to(dev), kc.to(dev), vc.to(dev), meta, table.to(dev), n.to(dev), kb, 0.1,
                                       local_w=1, return_pages=True)
    assert bool((pages[..., -1] == (L - 1) // bs).all())
    out = out.float().cpu()[0, :, 0]
    assert bool((out[:, 7] == INF).all()) and bool((out[:, 9] == -INF).all())
    assert int((~torch.isfinite(out)).sum()) == 2 * Hq


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("W", [6, 40, 400])               # 4 and 8 waves of one workgroup, and the split over the grid
@pytest.mark.parametrize("fp8", [False, True])
def test_weights_are_fp32(dev, fp8, W, D):
    """Values that cancel to 2^-14 of their size and less show what the weights lose.

    Scores are exact (one product each, 0 the largest), so a weight is off by the
    rounding of scale * log2(e) and of its product with a score of at most 1 in size
    (2 * 2^-24 of 1.5, times ln 2: 3 * 2^-24 with what they do to each other), by the
    exponential's unit (2 * 2^-24), and the sum by a rounding per addition: of at most
    seven values (less than 27 * 2^-24 however a weight is cut into products).  Together
    2^-19 of the weighted |v|, beside the rounding of the result."""
    dt = F8 if fp8 else BF16
    # scores whose weights two bf16 numbers miss by the most, upwards and downwards
    up, down = (((0.140625, 0.021484375, 0.9375, 0.34375), (0.875, 0.46875, 0.109375, 0.625)) if fp8 else
                ((0.71875, 0.96875, 0.84375, 0.296875), (0.671875, 0.8125, 0.390625, 0.359375)))
    Hq, bs, m = 8, 16, 5
    kc, vc = (torch.zeros(3, 1, bs, D) for _ in range(2))
    q = torch.zeros(1, Hq, 1, D, dtype=BF16)
    for h in range(Hq):                                   # head h looks at dim h of the keys, and alone at dims h + 8 i of the values
        q[0, h, 0, h] = 1.0
        a, b = up[h % 4], down[(h + h // 4) % 4]
        kc[1, 0, 1, h], kc[1, 0, 2:2 + m, h] = -a, -b
        for i, d in enumerate(range(h, D, 8)):
            x = 128.0 + 16.0 * (i % 8) if fp8 else 1.0 + i / 16
            vc[1, 0, 1, d] = x
            rest = x * math.exp(0.5 * (b - a))
            for j in range(m):                            # what the others take away again
                y = float(torch.tensor(rest).to(dt).float())
                vc[1, 0, 2 + j, d] = -y
                rest -= y
    assert torch.equal(kc.to(dt).float(), kc) and torch.equal(vc.to(dt).float(), vc)
    kc, vc = kc.to(dt), vc.to(dt)
    table = torch.full((1, W), -1, dtype=torch.int32)
    table[0, 0] = 1
    n = torch.tensor([2 + m], dtype=torch.int32)
    meta = tuple(t.to(dev) for t in _page_meta(kc, table, [2 + m], bs))
    want, mag, _ = O.attend(q, kc, vc, 0.5, 1.0, 1.0, table, n)
    own = torch.arange(D)[None, None] % 8 == torch.arange(Hq)[None, :, None]
    assert bool((want.abs() <= 2.0 ** -14 * mag)[own].all())
    a, t = (q.to(dev), kc.to(dev), vc.to(dev)), (table.to(dev), n.to(dev))
    for out in (PG.paged_decode_attn(*a, *t, 0.5), PG.paged_quest_decode(*a, meta, *t, 64, 0.5)):
        err = (out.double().cpu().reshape(want.shape) - want).abs()
        bad = ~(err <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * mag)
        assert not bool(bad.any()), float((err / mag)[bad].max())


def test_append_refuses_memory_written_twice(dev):
    """Expanded caches and one tensor for two, through the native call path and the wrapper."""
    bf = lambda *s: torch.zeros(*s, dtype=BF16, device=dev)                  # noqa: E731
    kc, vc, new = bf(4, 2, 16, 64), bf(4, 2, 16, 64), bf(1, 2, 64)
    t, n = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    mn, mx = bf(4, 2, 64), bf(4, 2, 64)
    for k, v, m in ((kc[:1].expand(4, 2, 16, 64), vc, None), (kc, vc[:, :1].expand(4, 2, 16, 64), None), (kc, kc, None),
                    (kc, vc, (mn, mn))):
        with pytest.raises(ValueError):
            PG.paged_kv_append(new, new, k, v, t, n, meta=m)
    assert PG.paged_kv_append(new, new, kc, vc, t, n, meta=(mn, mx)) is None


@pytest.mark.parametrize("gap", [0, 40, 100])
@pytest.mark.parametrize("L,W", [(40, 10), (600, 40), (3000, 300)])
def test_infinite_values_of_small_weights(dev, gap, L, W):
    """An infinite value stays one while its weight is at least 2^-100 of the largest, which
    a token of the same tile, another wave's or a later part has."""
    g = torch.Generator().manual_seed(gap + L)
    Hq, Hk, D, bs = 2, 1, 64, 16
    table, N = _table(g, [L, L], bs, slack=max(0, W - -(-L // bs)))
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    kc[..., 0] = -1.0                                     # every score is minus half the gap ..
    q = torch.zeros(2, Hq, 1, D, dtype=BF16)
    q[..., 0] = 1.0
    for b, p in enumerate((20, L - 1)):                   # .. but one token's
        kc[int(table[b, p // bs]), 0, p % bs, 0] = 1.0
    for b in range(2):
        vc[int(table[b, 0]), 0, 3, 5], vc[int(table[b, (L - 3) // bs]), 0, (L - 3) % bs, 6] = INF, -INF
    scale = gap / 2 * math.log(2)
    n = torch.tensor([L, L], dtype=torch.int32)
    meta = tuple(t.to(dev) for t in _page_meta(kc, table, [L, L], bs))
    a = (q.to(dev), kc.to(dev), vc.to(dev))
    t = (table.to(dev), n.to(dev))
    for out in (PG.paged_decode_attn(*a, *t, scale), PG.paged_quest_decode(*a, meta, *t, L + bs, scale)):
        out = out.float().cpu()
        assert bool((out[..., 5] == INF).all()) and bool((out[..., 6] == -INF).all())
        assert int((~torch.isfinite(out)).sum()) == 2 * 2 * Hq


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("single", [False, True])
def test_stored_keys_are_the_exact_rotation(dev, single, interleaved):
    """Keys in a bf16 cache bit for bit: the exact sum of the exact products, rounded to
    fp32 and from there to bf16 (with the products rounded to fp32 some differ); their
    min / max with them."""
    g = torch.Generator().manual_seed(91 + single)
    T, Hk, D, bs = 2048, 4, 128, 16
    k = _rand(g, T, Hk, D)
    W = 1 if single else T // bs
    cos, sin = _cos_sin(W * bs, D, base=37.0)
    if single:                                            # a token each, at every row of a block
        table, n, cu = torch.arange(T, dtype=torch.int32)[:, None], torch.arange(T, dtype=torch.int32) % bs + 1, None
        p = torch.arange(T) % bs
    else:
        table, n, cu = torch.randperm(W, generator=g).to(torch.int32)[None], torch.tensor([T], dtype=torch.int32), [0, T]
        p = torch.arange(T)
    N = table.numel()
    kc, vc = (torch.zeros(N, Hk, bs, D, dtype=BF16, device=dev) for _ in range(2))
    meta = tuple(torch.zeros(N, Hk, D, dtype=BF16, device=dev) for _ in range(2))
    PG.paged_kv_append(k.to(dev), k.to(dev), kc, vc, table.to(dev), n.to(dev), cos=cos.to(dev), sin=sin.to(dev), meta=meta,
                       cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev),
                       interleaved=interleaved)
    x, c, s = k.double(), cos.double()[p][:, None], sin.double()[p][:, None]
    i = torch.arange(D // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + D // 2)
    y = x.clone()
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    want = y.float().to(BF16)
    b = torch.arange(T) if single else torch.zeros(T, dtype=torch.long)
    got = kc.cpu()[table[b, p // bs].long(), :, p % bs]
    assert torch.equal(got, want)
    if not single:
        pages = want.reshape(W, bs, Hk, D).float()
        assert torch.equal(meta[0].cpu()[table[0].long()].float(), pages.amin(1))
        assert torch.equal(meta[1].cpu()[table[0].long()].float(), pages.amax(1))


# ---------------------------------------------------------------------------
# selection and page-sparse attention: every size of the selection, other layouts
# ---------------------------------------------------------------------------
def _want_pages(q, meta, table, n, bs, scale, npick):
    """The best npick places per head by (bound descending, place ascending), ascending; from
    sums of bf16 products in fp64."""
    B, Hq, _, D = q.shape
    Hk = meta[0].shape[1]
    qd = q.double().reshape(B, Hk, Hq // Hk, D)
    ids = table.clamp(min=0).long()
    lo, hi = (m.double()[ids].permute(0, 2, 3, 1).nan_to_num(0) for m in meta)
    b = (torch.matmul(qd.clamp(min=0), hi) + torch.matmul(qd.clamp(max=0), lo)).reshape(B, Hq, -1) * scale
    b = b.float().masked_fill((torch.arange(table.shape[1]) * bs >= n[:, None])[:, None], -INF)
    return b.argsort(dim=-1, descending=True, stable=True)[..., :npick].sort(-1).values


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("npick", [1, 300, 1023, 1024, 2047, 2048, 4095])
def test_quest_selection_sizes(dev, npick, ties):
    """Sequences of 1023 to 4096 pages, at both ends of every size of the selection in the
    attention kernel; ties: bounds of a few values only."""
    g = torch.Generator().manual_seed(npick)
    Hq, Hk, D = 4, 2, 64
    lens = [1023, 1024, 1025, 2047, 2048, 2049, 4096, 3001]
    table, N = _table(g, lens, 1, slack=0)
    kc, vc = _make_cache(g, N, Hk, 1, D, False)
    q = _rand(g, len(lens), Hq, 1, D)
    if ties:
        kc, q = (torch.randint(0, 2, x.shape, generator=g).to(BF16) for x in (kc, q))
    n = torch.tensor(lens, dtype=torch.int32)
    meta = (kc[:, :, 0].contiguous(), kc[:, :, 0].contiguous().clone())      # pages of one token
    a = (q.to(dev), kc.to(dev), vc.to(dev), tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), npick, 0.125)
    alone = PG.paged_quest_decode(*a)                     # selects in the attention kernel
    out, pages = PG.paged_quest_decode(*a, return_pages=True)
    want = _want_pages(q, meta, table, n, 1, 0.125, npick)
    assert torch.equal(pages.cpu().long(), want) and torch.equal(alone, out)
    _check_decode(dev, alone, q, kc, vc, 0.125, 1.0, 1.0, table, n,
                  [[set(want[b, h].tolist()) for h in range(Hq)] for b in range(len(lens))])


@pytest.mark.parametrize("W,L,npick", [(4096, 4096, 4095), (5000, 4990, 4980)])
def test_quest_runs_of_as_many_pages_as_a_list_holds(dev, W, L, npick):
    """So many heads and pages of one token that a run of a head's picks is bounded by the
    kernel's list and not by the grid."""
    g = torch.Generator().manual_seed(W)
    B, Hq, Hk, D = 16, 64, 1, 64
    table = torch.randperm(W, generator=g).to(torch.int32)[None].expand(B, W).contiguous()
    kc, vc = _make_cache(g, W, Hk, 1, D, False)
    q = _rand(g, B, Hq, 1, D)
    n = torch.tensor([L - 2 * b for b in range(B)], dtype=torch.int32)
    meta = (kc[:, :, 0].contiguous(), kc[:, :, 0].contiguous().clone())
    a = (q.to(dev), kc.to(dev), vc.to(dev), tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), npick, 0.125)
    alone = PG.paged_quest_decode(*a)
    out, pages = PG.paged_quest_decode(*a, return_pages=True)
    assert torch.equal(alone, out)
    some, heads = [0, 7, 15], [0, 9, 63]
    sub = q[some][:, heads]
    want = _want_pages(sub, meta, table[some], n[some], 1, 0.125, npick)
    assert torch.equal(pages.cpu().long()[some][:, heads], want)
    _check_decode(dev, alone[some][:, heads], sub, kc, vc, 0.125, 1.0, 1.0, table[some], n[some],
                  [[set(want[b, h].tolist()) for h in range(3)] for b in range(3)])


@pytest.mark.parametrize("pages,npick", [(1001, 7), (2047, 500), (4093, 4000)])
def test_quest_c_entries_with_unpadded_bounds(dev, pages, npick):
    """The C entries on bounds whose rows are not whole 16-byte chunks: the wrapper's bits."""
    g = torch.Generator().manual_seed(pages)
    B, Hq, Hk, D, bs = 2, 6, 2, 64, 1
    table, N = _table(g, [pages, pages - 1], bs, slack=0)
    kc, vc = (c.to(dev) for c in _make_cache(g, N, Hk, bs, D, False))
    q = _rand(g, B, Hq, 1, D).to(dev)
    table, n = table.to(dev), torch.tensor([pages, pages - 1], dtype=torch.int32, device=dev)
    meta = (kc[:, :, 0].contiguous(), kc[:, :, 0].contiguous().clone())
    want = PG.paged_quest_decode(q, kc, vc, meta, table, n, npick, 0.125)
    bound = PG.paged_page_scores(q, meta, table, n, bs, 0.125)
    assert bound.shape[-1] % 4 and bound.stride(1) == pages
    size = _lib.size_query("bytes_paged_quest_workspace_size", B, Hq, Hk, D, 0, bs, pages, npick)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    out = torch.empty(B, Hq, D, dtype=BF16, device=dev)
    p = _lib.ptr
    _lib.call("bytes_paged_quest_attn", p(q), q.stride(0), q.stride(1), p(kc), kc.stride(0), kc.stride(1), kc.stride(2),
              p(vc), vc.stride(0), vc.stride(1), vc.stride(2), 0, p(bound), bound.stride(0), bound.stride(1), None, 0, 0,
              npick, p(table), table.stride(0), p(n), p(out), out.stride(0), out.stride(1), B, Hq, Hk, D, bs, N, pages,
              0.125, 1.0, p(ws), ws.numel(), _lib.stream_of(q))
    assert torch.equal(out.unsqueeze(2), want)


@pytest.mark.parametrize("layout", ["nshd", "pair"])
@pytest.mark.parametrize("Hq,Hk,D,bs,fp8", [(14, 2, 64, 16, False), (7, 1, 128, 32, True), (6, 3, 128, 5, False),
                                            (8, 8, 64, 64, True)])
def test_quest_decode_of_strided_caches(dev, Hq, Hk, D, bs, fp8, layout):
    g = torch.Generator().manual_seed(bs + D)
    lens = [700, 0, 333]
    table, N = _table(g, lens, bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, fp8, layout)
    q, n = _rand(g, 3, Hq, 1, D), torch.tensor(lens, dtype=torch.int32)
    meta = _page_meta(kc, table, lens, bs)
    ks, vs = (0.03, 0.05) if fp8 else (1.0, 1.0)
    for kb in (128, 10 ** 5):
        out, pages = PG.paged_quest_decode(q.to(dev), _keep_storage(kc, dev), _keep_storage(vc, dev),
                                           tuple(m.to(dev) for m in meta), table.to(dev), n.to(dev), kb, D ** -0.5,
                                           k_scale=ks, v_scale=vs, return_pages=True)
        npick = min(-(-kb // bs), table.shape[1])
        want = _want_pages(q, meta, table, n, bs, D ** -0.5 * ks, npick)
        assert torch.equal(pages.cpu().long(), want)
        _check_decode(dev, out, q, kc, vc, D ** -0.5, ks, vs, table, n,
                      [[set(want[b, h].tolist()) for h in range(Hq)] for b in range(3)])


def test_window_of_more_blocks_than_are_picked(dev):
    """All blocks of the window are equally best, the lowest first; kb of local_w +
    block_size tokens always reaches the newest."""
    g = torch.Generator().manual_seed(61)
    Hq, Hk, D, bs, lens = 4, 2, 64, 16, [1000, 993, 992, 40]
    table, N = _table(g, lens, bs)
    kc, vc = _make_cache(g, N, Hk, bs, D, False)
    q, n = _rand(g, 4, Hq, 1, D).to(dev), torch.tensor(lens, dtype=torch.int32)
    meta = tuple(m.to(dev) for m in _page_meta(kc, table, n, bs))
    a = (q, kc.to(dev), vc.to(dev), meta, table.to(dev), n.to(dev))
    w = 100
    _, pages = PG.paged_quest_decode(*a, 64, 0.125, local_w=w, return_pages=True)
    for b in range(3):
        first = (lens[b] - w) // bs
        assert bool((pages[b].cpu() == torch.arange(first, first + 4)).all())
    _, pages = PG.paged_quest_decode(*a, w + bs, 0.125, local_w=w, return_pages=True)
    for b in range(3):
        assert bool((pages[b, :, -1] == (lens[b] - 1) // bs).all())
