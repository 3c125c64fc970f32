"""Caches in 8 bits with a scale for each block and KV head, and decode within a window:
against 64-bit restatements, at the sizes, masks and layouts where they can go wrong."""
import math

import pytest
import torch

import paged_oracle as O
import serving_oracle as S
from test_native_path_gpu import _both
from test_paged_gpu import _cos_sin, _keep_storage, _make_cache, _rand, _table, _tol
from bytes_amd import paged as PG

pytestmark = pytest.mark.gpu
F8, BF16, I8, I32, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.int8, torch.int32, torch.float32
INF, NAN = float("inf"), float("nan")
TYPES = [I8, F8]


def _bytes(t):
    return t.contiguous().view(torch.uint8) if t.element_size() == 1 else t.contiguous().view(torch.int16)


def _codes(g, dtype, *shape):
    """Any codes of the type but NaN."""
    if dtype == I8:
        return torch.randint(-127, 128, shape, generator=g).to(I8)
    return (torch.randn(*shape, generator=g) * 100).clamp(-448, 448).to(F8)


def block_cache(g, N, Hk, bs, D, dtype, layout="nhsd"):
    """(k, v, ks, vs): codes in the asked storage order, scales that differ from block to block."""
    if layout == "nshd":
        k, v = (_codes(g, dtype, N, bs, Hk, D).transpose(1, 2) for _ in "kv")
    elif layout == "pair":
        kv = _codes(g, dtype, N, 2, Hk, bs, D)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = (_codes(g, dtype, N, Hk, bs, D) for _ in "kv")
    ks, vs = (0.01 * torch.rand(N, Hk, generator=g) + 0.002 for _ in "kv")
    return k, v, ks, vs


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _check_append(dev, k, v, q, kc, vc, ks, vs, table, lens, cu, cos, sin, interleaved):
    """One append against its definition; returns what it left on the device."""
    N, Hk, bs, D = kc.shape
    T, int8 = k.shape[0], kc.dtype == I8
    dk, dv, dks, dvs = (_keep_storage(kc, dev), _keep_storage(vc, dev), ks.to(dev), vs.to(dev)) if not int8 else (
        torch.empty_strided(kc.shape, kc.stride(), dtype=I8, device=dev).copy_(kc),
        torch.empty_strided(vc.shape, vc.stride(), dtype=I8, device=dev).copy_(vc), ks.to(dev), vs.to(dev))
    put = lambda t: None if t is None else t.to(dev)                          # noqa: E731
    out = PG.paged_kv_append(k.to(dev), v.to(dev), dk, dv, table.to(dev), lens.to(dev), cu_seqlens=put(cu), q=put(q),
                             cos=put(cos), sin=put(sin), interleaved=interleaved, k_scale=dks, v_scale=dvs)
    rows = S.block_rows(T, table, lens, cu, bs, N)
    for name, new, old, got, s_old, s_got in (("k", k, kc, dk.cpu(), ks, dks.cpu()), ("v", v, vc, dv.cpu(), vs, dvs.cpu())):
        left = _bytes(got).clone()
        for i, mine in rows.items():
            offs = torch.tensor([m[0] for m in mine])
            x = torch.stack([(O.rotate(new[t].double(), cos, sin, p, interleaved)[0] if name == "k" else new[t].double())
                             for _, t, _, p in mine])                        # [n, Hk, D]
            o0 = int(offs.min())
            for h in range(Hk):
                a = float(x[:, h].abs().max())
                fit = S.fitting(a, int8)
                want = fit if o0 == 0 else max(fit, float(s_old[i, h]))
                s = float(s_got[i, h])
                # keys are rounded to fp32 once, the scale's division once: 2^-24 each; a power of two may be
                # the next where a lies within such a rounding of its limit
                near = abs(s - want) <= 2.0 ** -22 * want
                if not int8 and fit == want and fit > 0:
                    edge = S.fitting(a * (1 + 2.0 ** -22), int8), S.fitting(a * (1 - 2.0 ** -22), int8)
                    near = near or s in edge
                assert near, (name, i, h, s, want)
                # new rows: half a step of int8; half a step (2^-4) of e4m3, and half its smallest (2^-10)
                # units of the scale; x / s is rounded to fp32 first
                err = (got[i, h, offs].double() * s - x[:, h]).abs()
                lim = s * 0.5 if int8 else 2.0 ** -4 * x[:, h].abs() + s * 2.0 ** -10
                assert bool((err <= lim + 2.0 ** -21 * x[:, h].abs()).all()), (name, i, h, float((err - lim).max()))
                if o0 and s != float(s_old[i, h]):
                    was = old[i, h, :o0].double() * float(s_old[i, h])
                    err = (got[i, h, :o0].double() * s - was).abs()
                    lim = s * 0.5 if int8 else 2.0 ** -4 * was.abs() + s * 2.0 ** -10
                    assert s > float(s_old[i, h]) and bool((err <= lim + 2.0 ** -21 * was.abs()).all()), (name, i, h)
                    left[i, h, :o0] = _bytes(old)[i, h, :o0]
                left[i, h, offs] = _bytes(old)[i, h, offs]
        assert torch.equal(left, _bytes(old)), f"{name}: rows that no new token names changed"
        untouched = torch.ones(N, dtype=torch.bool)
        untouched[list(rows)] = False
        assert torch.equal(s_got[untouched], s_old[untouched])
    if q is not None:
        want = torch.zeros(T, q.shape[1], D, dtype=torch.float64)
        lim = torch.zeros_like(want)
        for t, b, p in O.placed(T, table, lens, cu, bs):
            want[t], mag = O.rotate(q[t].double(), cos, sin, p, interleaved)
            lim[t] = 2.0 ** -8 * want[t].abs() + 2.0 ** -22 * mag
        assert bool(((out.double().cpu() - want).abs() <= lim).all())
    else:
        assert out is None
    return dk, dv, dks, dvs


HEADS = [(14, 2, 64), (28, 4, 128), (8, 1, 128), (5, 5, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", HEADS)
@pytest.mark.parametrize("bs,rot,interleaved,layout", [(16, 64, False, "nhsd"), (7, 32, True, "nshd"), (1, 48, False, "nhsd"),
                                                       (128, 0, False, "pair")])
def test_append_single_tokens(dev, dtype, Hq, Hk, D, bs, rot, interleaved, layout):
    """First rows, last rows, rows whose scale grows and rows whose does not; an empty row, lengths past
    the table, a block that does not exist."""
    g = torch.Generator().manual_seed(Hq + bs)
    lens = [1, 2 * bs, 2 * bs + 1, 0, 3 * bs - 1, 77, 40, 30]
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = block_cache(g, N, Hk, bs, D, dtype, layout)
    qkv = _rand(g, len(lens), Hq + 2 * Hk, D)
    qkv[::2] *= 4                                    # every other token's scale grows
    cos, sin = _cos_sin(table.shape[1] * bs, rot) if rot else (None, None)
    table[6, (40 - 1) // bs] = -1
    n = torch.tensor(lens, dtype=I32)
    n[7] = table.shape[1] * bs + 5
    _check_append(dev, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], qkv[:, :Hq], kc, vc, ks, vs, table, n, None, cos, sin, interleaved)
    _check_append(dev, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], None, kc, vc, ks, vs, table, n, None, None, None, False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("bs,rot,interleaved,layout", [
    (16, 64, False, "nhsd"), (32, 16, True, "pair"), (8, 64, False, "nshd"), (1, 64, False, "nhsd"), (37, 32, True, "nhsd"),
    (17, 0, False, "nshd"), (100, 64, False, "nhsd")])
def test_append_ragged_prompts(dev, dtype, Hq, Hk, D, bs, rot, interleaved, layout):
    """Chunks that start and end anywhere in a block, one token, none, more than a sequence holds; rows
    past the last sequence."""
    g = torch.Generator().manual_seed(bs)
    lens, new = [50, 3, 0, 129, 64, 20, 33], [50, 1, 0, 40, 64, 27, 16]
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = block_cache(g, N, Hk, bs, D, dtype, layout)
    cu = torch.tensor([0] + new).cumsum(0).to(I32)
    qkv = _rand(g, int(cu[-1]) + 5, Hq + 2 * Hk, D)
    qkv[::3] *= 3
    cos, sin = _cos_sin(table.shape[1] * bs, rot) if rot else (None, None)
    table[4, 1 if table.shape[1] > 1 else 0] = N     # names no block
    _check_append(dev, qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:], qkv[:, :Hq], kc, vc, ks, vs, table,
                  torch.tensor(lens, dtype=I32), cu, cos, sin, interleaved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("single", [True, False])
def test_append_special_values(dev, dtype, single):
    """Rows of zeros, subnormals, infinities and NaN, scales that no append leaves."""
    g = torch.Generator().manual_seed(1)
    Hk, D, bs, B = 2, 64, 4, 9
    lens = [2] * B
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = block_cache(g, N, Hk, bs, D, dtype)
    for i, s in enumerate((0.0, NAN, -1.0, INF)):
        ks[table[i, 0]] = vs[table[i, 0]] = s
    x = _rand(g, B, Hk, D)
    x[4] = 0
    ks[table[4, 0]], vs[table[4, 0]] = 0.0, 0.0
    x[5, 0, 3], x[5, 1, 7] = INF, -INF
    x[6, 0, 5] = NAN
    x[7] = x[7] * 2.0 ** -126
    ks[table[7, 0]], vs[table[7, 0]] = 0.0, 0.0
    x[8] = NAN
    cu = None if single else torch.arange(B + 1, dtype=I32)
    d = [t.to(dev) for t in (kc, vc, ks, vs)]
    PG.paged_kv_append(x.to(dev), x.to(dev), d[0], d[1], table.to(dev), torch.tensor(lens, dtype=I32, device=dev),
                       cu_seqlens=None if cu is None else cu.to(dev), k_scale=d[2], v_scale=d[3])
    int8 = dtype == I8
    for c, s in ((d[0].cpu(), d[2].cpu()), (d[1].cpu(), d[3].cpu())):
        for b in range(B):
            i = int(table[b, 0])
            code, sc = c[i, :, 1].double(), s[i].double()
            if b == 4:
                assert not bool(sc.any()) and not bool(code.any())
                continue
            if b == 8:                               # no number: the scale stays, codes are NaN (0 in int8)
                assert bool((code == 0).all() if int8 else code.isnan().all())
                continue
            want = x[b].double().clamp(-S.BF16_MAX, S.BF16_MAX)
            nan = want.isnan()
            assert bool(torch.isfinite(sc).all()) and bool((sc >= 0).all()), b
            if int8:
                assert bool((code[nan] == 0).all())
            else:
                assert torch.equal(code.isnan(), nan)
            err = (code * sc[:, None] - want).abs()
            # (a subnormal scale of int8 has steps of 2^-149 itself)
            lim = sc[:, None] * 0.5 + 127 * 2.0 ** -149 if int8 else 2.0 ** -4 * want.abs() + sc[:, None] * 2.0 ** -10
            assert bool((err <= lim + 2.0 ** -21 * want.abs())[~nan].all()), b
            if b < 4:                                # a scale that no append leaves counts as 0
                # (a / 127 is rounded to fp32: 2^-24 of it at most; a power of two is at most twice a / 448)
                assert bool((sc <= want.abs().amax(-1) / (127 if int8 else 224) * (1 + 2.0 ** -24)).all()), b


@pytest.mark.parametrize("dtype", TYPES)
def test_append_at_once_and_in_pieces(dev, dtype):
    """Chunks of whole blocks leave the bytes that one prompt leaves; token by token, rows are within what
    they may lose each time their scale grows."""
    g = torch.Generator().manual_seed(5)
    Hk, D, bs, n = 2, 128, 16, 80
    table, N = _table(g, [n], bs)
    cache = [t.to(dev) for t in block_cache(g, N, Hk, bs, D, dtype)]
    k, v = _rand(g, n, Hk, D).to(dev), _rand(g, n, Hk, D).to(dev)
    cos, sin = (t.to(dev) for t in _cos_sin(table.shape[1] * bs, 64))
    t = table.to(dev)
    def fill(sizes):
        c = [x.clone() for x in cache]
        at = 0
        for m in sizes:
            cu = None if m == 1 else torch.tensor([0, m], dtype=I32, device=dev)
            PG.paged_kv_append(k[at:at + m], v[at:at + m], c[0], c[1], t, torch.tensor([at + m], dtype=I32, device=dev),
                               cu_seqlens=cu, cos=cos, sin=sin, k_scale=c[2], v_scale=c[3])
            at += m
        return c
    whole, blocks, single = fill([n]), fill([32, 16, 32]), fill([1] * n)
    held = table[0, :n // bs].tolist()
    for a, b in zip(whole, blocks):
        assert torch.equal(_bytes(a) if a.dtype != F32 else a, _bytes(b) if b.dtype != F32 else b)
    for c, s in ((0, 2), (1, 3)):
        a, b = whole[s][held], single[s][held]
        assert torch.equal(a, b)                     # the largest value is in the last scale, whenever it came
        va, vb = (x[c][held].double() * x[s][held].double()[..., None, None] for x in (whole, single))
        if dtype == F8:                              # powers of two: the same but for the format's subnormals
            assert bool(((va - vb).abs() <= a.double()[..., None, None] * 2.0 ** -9).all())
        else:                                        # at most 15 roundings again, of scales that grow
            assert bool(((va - vb).abs() <= a.double()[..., None, None] * 0.5 * 16).all())
            assert float((va - vb).norm() / va.norm()) < 0.02


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------
def _check_decode(got, q, kc, vc, scale, ks, vs, table, lens, window=None, sinks=0):
    """The tolerance of the decode over one scale (test_paged_gpu._tol); a block's scale is
    another fp32 rounding of each score and weight, which its last term covers.  Weights
    below 2^-126 of the row's largest become 0 (fp32's normal range), and results below it
    may: n weights of at most 2^-126 times the largest |v| that a sequence holds, and
    2^-126."""
    n = [max(0, min(int(x), table.shape[1] * kc.shape[2])) for x in lens]
    want, mag, dots = S.attend_rows(q[:, :, 0], [(b, x - 1) if x else None for b, x in enumerate(n)], kc, vc, scale, ks, vs,
                                    table, lens, window, sinks)
    got = got.double().cpu().reshape(want.shape)
    top = S.values(vc, vs).abs().amax((1, 2, 3))     # of each block
    tiny = torch.zeros(len(n), 1, 1, dtype=torch.float64)
    for b, x in enumerate(n):
        ids = table[b, :-(-x // kc.shape[2])].long()
        tiny[b] = 2.0 ** -126 * (1 + x * float(max([float(top[i]) for i in ids if 0 <= i < len(top)], default=0.0)))
    bad = ~((got - want).abs() <= _tol(want, mag, dots, q.shape[-1]) + tiny)
    assert not bool(bad.any()), (bad.nonzero()[:5].tolist(), got[bad][:5], want[bad][:5])


def _dev(t, dev):
    if not torch.is_tensor(t):
        return t
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t) if t.dtype != F8 else _keep_storage(t, dev)


LENS = [[1], [0, 3, 0], [130, 1, 64, 0, 257], [1000, 999], [31, 32, 33, 127, 128, 129, 15, 16, 17, 0]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (28, 4, 128), (33, 1, 64), (24, 8, 128)])
@pytest.mark.parametrize("bs,layout", [(16, "nhsd"), (64, "nshd"), (1, "nhsd"), (24, "pair"), (7, "pair"), (1000, "nhsd")])
def test_decode(dev, dtype, Hq, Hk, D, bs, layout):
    for i, lens in enumerate(LENS):
        g = torch.Generator().manual_seed(100 * i + bs)
        table, N = _table(g, lens, bs)
        kc, vc, ks, vs = block_cache(g, N, Hk, bs, D, dtype, layout)
        q = _rand(g, len(lens), Hq, 1, D)
        n = torch.tensor(lens, dtype=I32)
        print(f"decode {dtype} Hq{Hq} Hk{Hk} D{D} bs{bs} {layout} lens {lens}", flush=True)
        out = PG.paged_decode_attn(q.to(dev), _dev(kc, dev), _dev(vc, dev), table.to(dev), n.to(dev), D ** -0.5,
                                   k_scale=ks.to(dev), v_scale=vs.to(dev))
        assert out.shape == q.shape and out.dtype == BF16
        _check_decode(out, q, kc, vc, D ** -0.5, ks, vs, table, n)


def any_cache(g, N, Hk, bs, D, kind, layout="nhsd"):
    if kind in (I8, F8):
        return block_cache(g, N, Hk, bs, D, kind, layout)
    kc, vc = _make_cache(g, N, Hk, bs, D, kind == "fp8", layout)
    return (kc, vc, 0.03, 0.05) if kind == "fp8" else (kc, vc, 1.0, 1.0)


KINDS = ["bf16", "fp8", I8, F8]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D", [(14, 2, 64), (8, 4, 128)])
@pytest.mark.parametrize("bs", [16, 5, 64])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (32, 4), (33, 0), (100, 31), (100, 33), (64, 64), (500, 4), (2 ** 31, 5),
                                          (7, 10 ** 6)])
def test_decode_within_a_window(dev, kind, Hq, Hk, D, bs, window, sinks):
    """Windows and sinks that end inside and at the ends of tiles and blocks, touch, overlap, are longer than
    the sequence."""
    g = torch.Generator().manual_seed(bs + sinks)
    lens = [1, 31, 100, 132, 0, 333, 1000, 161]
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = any_cache(g, N, Hk, bs, D, kind)
    q = _rand(g, len(lens), Hq, 1, D)
    n = torch.tensor(lens, dtype=I32)
    print(f"window {window} sinks {sinks} {kind} Hq{Hq} D{D} bs{bs}", flush=True)
    out = PG.paged_decode_attn(q.to(dev), _dev(kc, dev), _dev(vc, dev), table.to(dev), n.to(dev), D ** -0.5, window=window,
                               sinks=sinks, k_scale=_dev(ks, dev), v_scale=_dev(vs, dev))
    _check_decode(out, q, kc, vc, D ** -0.5, ks, vs, table, n, window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [16, 20])
def test_what_a_window_leaves_out_is_not_read(dev, kind, bs):
    """Blocks behind the window gone, NaN in rows that are not seen, blocks that do not exist, sequences
    without any, scales that are NaN where nothing is held, lengths past the table."""
    g = torch.Generator().manual_seed(bs)
    Hq, Hk, D, window, sinks = 8, 2, 128, 70, 5
    lens = [300, 333, 90, 5, 640]
    table, N = _table(g, lens, bs, slack=0)
    table[0, 200 // bs:(300 - 70) // bs - 1] = -1    # gone
    table[1, (333 - 30) // bs] = N
    table[2] = -1
    n = torch.tensor([300, 333, 90, 5, 10 ** 6], dtype=I32)
    kc, vc, ks, vs = any_cache(g, N, Hk, bs, D, kind)
    seen = torch.zeros(N, bs, dtype=torch.bool)
    for b in range(5):
        toks = O.held_tokens(table, n, N, bs, b)
        end = min(int(n[b]), table.shape[1] * bs)
        for p, i, o in toks:
            seen[i, o] = p >= end - window or p < sinks
    q = _rand(g, 5, Hq, 1, D)
    dirty = [kc.clone(), vc.clone(), ks, vs]
    i, o = (~seen).nonzero().T
    for c in dirty[:2]:
        if kind == I8:
            c[i, :, o] = -128
        else:
            f = c.float()
            f[i, :, o] = NAN
            c.copy_(f.to(c.dtype)) if c.dtype != F8 else c.view(torch.uint8).copy_(f.to(F8).view(torch.uint8))
    if torch.is_tensor(ks):
        none = ~seen.any(1)
        dirty[2], dirty[3] = ks.clone(), vs.clone()
        dirty[2][none] = dirty[3][none] = NAN
    out = PG.paged_decode_attn(q.to(dev), *(_dev(t, dev) for t in dirty[:2]), table.to(dev), n.to(dev), 0.1, window=window,
                               sinks=sinks, k_scale=_dev(dirty[2], dev), v_scale=_dev(dirty[3], dev))
    assert not bool(out[2].any())
    _check_decode(out, q, kc, vc, 0.1, ks, vs, table, n, window, sinks)


@pytest.mark.parametrize("B,Hq,Hk,D,L,bs,kind,window", [
    (3, 40, 2, 128, 20000, 16, I8, None), (70, 8, 2, 64, 2500, 32, F8, None), (2, 24, 8, 128, 30000, 16, "bf16", 9000),
    (66, 8, 2, 64, 4000, 64, "fp8", 3000), (4, 4, 1, 128, 17000, 24, I8, 10000)])
def test_decode_long_and_wide(dev, B, Hq, Hk, D, L, bs, kind, window):
    """Contexts that several workgroups share, more sequences than a wave has lanes: the last row against
    its definition, all rows against the same tokens without a window or block scales."""
    g = torch.Generator().manual_seed(L)
    lens = [max(1, L - 37 * b) for b in range(B)]
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = any_cache(g, N, Hk, bs, D, kind)
    q = _rand(g, B, Hq, 1, D)
    n = torch.tensor(lens, dtype=I32)
    sinks = 4 if window else 0
    out = PG.paged_decode_attn(q.to(dev), _dev(kc, dev), _dev(vc, dev), table.to(dev), n.to(dev), D ** -0.5, window=window,
                               sinks=sinks, k_scale=_dev(ks, dev), v_scale=_dev(vs, dev))
    some = [0, B // 2, B - 1]
    _check_decode(out[some], q[some], kc, vc, D ** -0.5, ks, vs, table[some], n[some], window, sinks)
    if window is None:                               # the same values in one scale's units, rounded: near
        near = [(c.float() * s[:, :, None, None]).to(BF16).to(dev) for c, s in ((kc, ks), (vc, vs))]
        ref = PG.paged_decode_attn(q.to(dev), *near, table.to(dev), n.to(dev), D ** -0.5)
        assert float((out.float() - ref.float()).norm() / ref.float().norm()) < 0.02


def test_decode_large_scores_and_scales(dev):
    """Scores far apart, scales of 0 and near the ends of fp32, a negative `scale`."""
    g = torch.Generator().manual_seed(3)
    Hq, Hk, D, bs = 8, 2, 64, 16
    lens = [100, 40, 65, 3]
    table, N = _table(g, lens, bs)
    kc, vc, ks, vs = block_cache(g, N, Hk, bs, D, I8)
    ks[table[0, 1]], vs[table[0, 2]], vs[table[1, 0]] = 0.0, 0.0, 1e30
    vs[table[2, 0]] = 1e-30
    q = _rand(g, 4, Hq, 1, D)
    n = torch.tensor(lens, dtype=I32)
    for scale in (1.0, -0.5, 0.0, 20.0):
        out = PG.paged_decode_attn(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), n.to(dev), scale, k_scale=ks.to(dev),
                                   v_scale=vs.to(dev))
        _check_decode(out, q, kc, vc, scale, ks, vs, table, n)


@pytest.mark.parametrize("kind", [I8, F8])
def test_offsets_past_32_bits(dev, kind):
    """Blocks more than 2^32 bytes into the cache: append, decode and prompt."""
    Hq, Hk, D, bs, N = 8, 2, 128, 16, 1100000        # 4.5 GB of each
    kc, vc = (torch.zeros(N, Hk, bs, D, dtype=torch.uint8, device=dev).view(kind) for _ in "kv")
    ks, vs = torch.zeros(N, Hk, device=dev), torch.zeros(N, Hk, device=dev)
    g = torch.Generator().manual_seed(2)
    ids = torch.tensor([[N - 1, N - 3, 5, N - 7]], dtype=I32)
    L = 60
    k, v, q = _rand(g, L, Hk, D), _rand(g, L, Hk, D), _rand(g, L, Hq, D)
    n, cu = torch.tensor([L], dtype=I32), torch.tensor([0, L], dtype=I32)
    PG.paged_kv_append(k.to(dev), v.to(dev), kc, vc, ids.to(dev), n.to(dev), cu_seqlens=cu.to(dev), k_scale=ks, v_scale=vs)
    at = ids[0].long()
    raw = torch.uint8 if kind == F8 else I8
    small = [c.view(raw)[at].cpu().view(kind) for c in (kc, vc)] + [ks[at].cpu(), vs[at].cpu()]
    st = torch.arange(4, dtype=I32)[None]
    got = small[0].double() * small[2].double()[:, :, None, None]
    want = k.double().transpose(0, 1).reshape(Hk, -1, D)
    assert float((got.transpose(0, 1).reshape(Hk, -1, D)[:, :L] - want).norm() / want.norm()) < 0.04
    out = PG.paged_decode_attn(q[-1:, :, None].to(dev), kc, vc, ids.to(dev), n.to(dev), 0.09, k_scale=ks, v_scale=vs)
    _check_decode(out, q[-1:, :, None], *small[:2], 0.09, *small[2:], st, n)
    rows = PG.paged_prompt_attn(q.to(dev), kc, vc, ids.to(dev), n.to(dev), cu.to(dev), 0.09, k_scale=ks, v_scale=vs)
    assert float((rows[-1] - out[0, :, 0]).float().norm() / out.float().norm()) < 0.01


def test_native_path_and_wrapper_agree(dev, monkeypatch):
    g = torch.Generator().manual_seed(9)
    Hq, Hk, D, bs = 8, 2, 64, 16
    lens = [100, 3, 47]
    table, N = _table(g, lens, bs)
    t, n = table.to(dev), torch.tensor(lens, dtype=I32, device=dev)
    q = _rand(g, 3, Hq, 1, D).to(dev)
    k, v = _rand(g, 3, Hk, D).to(dev), _rand(g, 3, Hk, D).to(dev)
    cos, sin = (x.to(dev) for x in _cos_sin(t.shape[1] * bs, 64))
    for kind in KINDS:
        kc, vc, ks, vs = (_dev(x, dev) for x in any_cache(g, N, Hk, bs, D, kind))
        sc = dict(k_scale=ks, v_scale=vs)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, t, n, 0.125, window=20, sinks=3, **sc)
        _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, t.long(), n, 0.125, window=20, taken=False, **sc)
        if kind in (I8, F8):
            _both(monkeypatch, PG.paged_decode_attn, q, kc, vc, t, n, 1, **sc)
            raw = torch.uint8
            def append(cu):
                c = [x.clone() for x in (kc, vc, ks, vs)]
                out = PG.paged_kv_append(k, v, c[0], c[1], t, n, cu_seqlens=cu, q=q[:, :, 0], cos=cos, sin=sin, k_scale=c[2],
                                         v_scale=c[3])
                return (out, c[0].view(raw), c[1].view(raw), c[2], c[3])
            _both(monkeypatch, append, None)
            _both(monkeypatch, append, torch.tensor([0, 1, 2, 3], dtype=I32, device=dev))


def test_one_element_scales_on_the_gpu(dev):
    """A cache of one block and head: two [1, 1] fp32 tensors are its block scales, other tensors of one element numbers."""
    g = torch.Generator().manual_seed(7)
    q, cl, bt = (t.to(dev) for t in (_rand(g, 1, 8, 1, 64), torch.tensor([40], dtype=I32), torch.zeros(1, 1, dtype=I32)))
    kc, vc = ((torch.randn(1, 1, 64, 64, generator=g) * 30).to(F8).to(dev) for _ in "kv")
    one = torch.ones(1, 1, device=dev)
    want = PG.paged_decode_attn(q, kc, vc, bt, cl, 0.125, k_scale=0.03, v_scale=0.25)
    for k, v in ((one * 0.03, 0.25), (0.03, one * 0.25), (one.double() * 0.03, one.double() * 0.25), (one[0] * 0.03, one * 0.25)):
        got = PG.paged_decode_attn(q, kc, vc, bt, cl, 0.125, k_scale=k, v_scale=v)
        exact = PG.paged_decode_attn(q, kc, vc, bt, cl, 0.125, k_scale=float(k), v_scale=0.25)
        assert torch.equal(got, exact)
        assert torch.equal(PG.paged_prompt_attn(q[:, :, 0], kc, vc, bt, cl, cl.new_tensor([0, 1]), 0.125, k_scale=k, v_scale=v),
                           PG.paged_prompt_attn(q[:, :, 0], kc, vc, bt, cl, cl.new_tensor([0, 1]), 0.125, k_scale=float(k), v_scale=0.25))
    by_block = PG.paged_decode_attn(q, kc, vc, bt, cl, 0.125, k_scale=one * 0.03, v_scale=one * 0.25)
    assert float((by_block.float() - want.float()).norm() / want.float().norm()) < 0.005
    b = [t.to(BF16) for t in (kc, vc)]               # a bf16 cache's are 1.0
    assert torch.equal(PG.paged_decode_attn(q, *b, bt, cl, 0.125, k_scale=one, v_scale=one), PG.paged_decode_attn(q, *b, bt, cl, 0.125))
