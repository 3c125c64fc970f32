"""Tables, block scales, windows and prompts without a GPU: what they refuse, and what
they hand to the C ABI."""
import contextlib
import ctypes

import pytest
import torch

import serving_oracle as S
from bytes_amd import _lib
from bytes_amd import paged as PG
from bytes_amd import paged_tables as PT

F8, BF16, I8, I32, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.int8, torch.int32, torch.float32


@pytest.fixture
def calls(monkeypatch):
    """Launches are recorded and not made; CPU tensors stand for the GPU's."""
    made = []
    for m in (PG, PT):
        monkeypatch.setattr(m.C, "cuda_tensors", lambda *ts: [t.device for t in ts] and ts[0].device)
        monkeypatch.setattr(m, "call", lambda name, *a: made.append((name, a)))
        monkeypatch.setattr(m, "size_query", lambda name, *a: made.append((name, a)) or 4096)
        monkeypatch.setattr(m, "stream_of", lambda t: 0)
    monkeypatch.setattr(PG.torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "_native", _lib._NoNative())
    return made


def _inputs(B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4, dtype=I8, T=None):
    T = B if T is None else T
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt)                        # noqa: E731
    return dict(k=z(T, Hk, D), v=z(T, Hk, D), q3=z(T, Hq, D), q=z(B, Hq, 1, D), kc=z(N, Hk, bs, D).to(dtype),
                vc=z(N, Hk, bs, D).to(dtype), ks=z(N, Hk, dt=F32), vs=z(N, Hk, dt=F32), bt=z(B, W, dt=I32), cl=z(B, dt=I32),
                cu=z(B + 1, dt=I32), cos=z(W * bs, D // 2, dt=F32), sin=z(W * bs, D // 2, dt=F32))


def _append(x, **kw):
    a = dict(cos=x["cos"], sin=x["sin"], q=x["q3"], k_scale=x["ks"], v_scale=x["vs"])
    a.update(kw)
    return PG.paged_kv_append(x["k"], x["v"], x["kc"], x["vc"], x["bt"], x["cl"], **a)


def _decode(x, **kw):
    a = dict(k_scale=x["ks"], v_scale=x["vs"])
    a.update(kw)
    return PG.paged_decode_attn(x["q"], x["kc"], x["vc"], x["bt"], x["cl"], 0.125, **a)


def _prompt(x, **kw):
    a = dict(k_scale=x["ks"], v_scale=x["vs"])
    a.update(kw)
    return PG.paged_prompt_attn(x["q3"], x["kc"], x["vc"], x["bt"], x["cl"], x["cu"], 0.125, **a)


OPS = [_append, _decode, _prompt]


def test_calls_reach_the_abi_with_its_signatures(calls):
    for dtype in (I8, F8):
        x = _inputs(dtype=dtype)
        assert _append(x).shape == (3, 8, 64) and _append(x, q=None, cos=None, sin=None) is None
        assert _decode(x).shape == (3, 8, 1, 64) and _decode(x, window=5, sinks=2).shape == (3, 8, 1, 64)
        assert _prompt(x).shape == (3, 8, 64)
    plain = dict(k_scale=1.0, v_scale=1.0)
    x = _inputs(dtype=BF16, T=7)
    x["q"] = x["q"][:3]
    assert _prompt(x, **plain).shape == (7, 8, 64) and _decode(x, window=3, **plain).shape == (3, 8, 1, 64)
    z = lambda *s: torch.zeros(*s, dtype=I32)                                # noqa: E731
    out = PT.paged_resize(z(3, 4), z(3), z(12), z(2), z(3), 20, 16, keep=z(3), window=5)
    assert [t.shape[0] for t in out] == [4, 3, 20, 20, 20] and out.slots.dtype == torch.int64
    seen = set()
    for name, a in calls:
        sig = _lib.SIGNATURES[name]
        assert len(a) == len(sig) - (1 if name.endswith("_size") else 0), name
        seen.add(name)
    assert {"bytes_paged_kv_append_blocks", "bytes_paged_window_attn", "bytes_paged_prompt_attn", "bytes_paged_resize"} <= seen


def test_types_scales_and_windows(calls):
    for dtype, typ in ((I8, 3), (F8, 2)):
        x = _inputs(dtype=dtype)
        x["ks"], x["vs"] = torch.zeros(12, 2, 2)[..., 0], torch.zeros(2, 12).t()         # any strides
        _decode(x)
        a = calls[-1][1]
        assert a[11] == typ and a[13:15] == (4, 2) and a[16:18] == (1, 12)
        assert a[-7:-3] == (2 ** 30, 0, 0.125, 1.0)                          # no window; scale, v_scale
        _decode(x, window=2 ** 40, sinks=7)
        assert calls[-1][1][-7:-5] == (2 ** 30, 7)
    x = _inputs(dtype=F8)
    _prompt(x, k_scale=0.5, v_scale=0.25, window=9, sinks=4)
    a = calls[-1][1]
    assert a[11] == 1 and a[12] is None and a[15] is None and a[-7:-3] == (9, 4, 0.0625, 0.25)
    calls.clear()                                    # one scale in a tensor of one element is a number
    _decode(x, k_scale=torch.tensor(0.5), v_scale=torch.tensor([0.25]))
    assert calls[-1][0] == "bytes_paged_decode_attn" and calls[-1][1][-5:-3] == (0.0625, 0.25)
    _decode(x, k_scale=torch.full((1, 1), 0.5), v_scale=0.25)
    assert calls[-1][0] == "bytes_paged_decode_attn" and calls[-1][1][-5:-3] == (0.0625, 0.25)
    x = _inputs(dtype=F8, Hk=1, N=1, W=1)            # a cache of one block and head has such a scale
    _decode(x)
    assert calls[-1][0] == "bytes_paged_window_attn" and calls[-1][1][11] == 2


def _bad(name, **change):
    return pytest.param(change, id=name)


@pytest.mark.parametrize("change", [
    _bad("cache dtypes differ", vc=lambda t: t.to(F8)),
    _bad("cache dtype", kc=lambda t: t.to(torch.uint8), vc=lambda t: t.to(torch.uint8)),
    _bad("bf16 cache", kc=lambda t: t.to(BF16), vc=lambda t: t.to(BF16)),
    _bad("cache shapes differ", vc=lambda t: t[1:]),
    _bad("rows off 16 bytes", kc=lambda t: torch.zeros(12, 2, 16, 65, dtype=I8)[..., 1:]),
    _bad("row stride off 16 bytes", vc=lambda t: torch.zeros(12, 2, 16, 72, dtype=I8)[..., :64]),
    _bad("scales of one kind", ks=lambda t: 0.5),
    _bad("scale dtype", ks=lambda t: t.double()),
    _bad("scale shape", vs=lambda t: t[1:]),
    _bad("scale rank", vs=lambda t: t.reshape(-1)),
    _bad("table rank", bt=lambda t: t[0]),
    _bad("table dtype", bt=lambda t: t.float()),
    _bad("table without columns", bt=lambda t: t[:, :0]),
    _bad("lengths shape", cl=lambda t: t[:2]),
    _bad("head dim", kc=lambda t: t[..., :32], vc=lambda t: t[..., :32], k=lambda t: t[..., :32], v=lambda t: t[..., :32],
         q=lambda t: t[..., :32], q3=lambda t: t[..., :32]),
])
@pytest.mark.parametrize("op", OPS)
def test_refuses_caches_scales_and_tables(calls, op, change):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        op(x)
    assert not [n for n, _ in calls if not n.endswith("_size")]


@pytest.mark.parametrize("op", OPS)
def test_refuses_int8_without_block_scales(calls, op):
    with pytest.raises(ValueError):
        op(_inputs(), k_scale=0.5, v_scale=0.5)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-1), dict(window=4, sinks=-1), dict(sinks=4)])
@pytest.mark.parametrize("op", [_decode, _prompt])
@pytest.mark.parametrize("plain", [True, False])
def test_refuses_windows(calls, op, kw, plain):
    x = _inputs(dtype=BF16 if plain else I8)
    with pytest.raises(ValueError):
        op(x, **kw, **(dict(k_scale=1.0, v_scale=1.0) if plain else {}))
    assert not calls


def test_append_refuses(calls):
    x = _inputs()
    meta = (torch.zeros(12, 2, 64, dtype=BF16), torch.zeros(12, 2, 64, dtype=BF16))
    with pytest.raises(ValueError, match="meta"):
        _append(x, meta=meta)
    with pytest.raises(ValueError, match="same memory"):
        _append({**x, "vs": x["ks"]})
    with pytest.raises(ValueError, match="expanded"):
        _append({**x, "vs": x["vs"][:1].expand(12, 2)})
    with pytest.raises(ValueError, match="page-sparse"):
        PG.paged_quest_decode(x["q"], x["kc"], x["vc"], meta, x["bt"], x["cl"], 32, 0.1, k_scale=x["ks"], v_scale=x["vs"])
    assert not calls
    assert _decode({**x, "vs": x["ks"]}).shape == (3, 8, 1, 64)              # reads only


@pytest.mark.parametrize("change", [
    _bad("query rank", q3=lambda t: t[:, :, None]), _bad("query dtype", q3=lambda t: t.half()),
    _bad("heads", q3=lambda t: t[:, :7]), _bad("no heads", q3=lambda t: t[:, :0]),
    _bad("cu shape", cu=lambda t: t[:3]), _bad("cu dtype", cu=lambda t: t.float()),
])
def test_prompt_refuses(calls, change):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        _prompt(x)
    assert not [n for n, _ in calls if not n.endswith("_size")]


def test_prompt_without_rows(calls):
    x = _inputs(T=0)
    assert _prompt(x).shape == (0, 8, 64) and not calls


def _resize(calls_=None, B=3, W=4, N=12, T=20, bs=16, **kw):
    z = lambda *s: torch.zeros(*s, dtype=I32)                                # noqa: E731
    a = dict(block_table=z(B, W), context_lens=z(B), free_blocks=z(N), free_range=z(2), new_lens=z(B))
    rest = dict(keep=kw.pop("keep", None), window=kw.pop("window", None), sinks=kw.pop("sinks", 0))
    a.update(kw)
    return PT.paged_resize(*a.values(), T, bs, **rest)


@pytest.mark.parametrize("kw", [
    dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), dict(block_table=torch.zeros(3, dtype=I32)),
    dict(block_table=torch.zeros(3, 0, dtype=I32)), dict(block_table=torch.zeros(4, 3, dtype=I32).t()),
    dict(block_table=torch.zeros(1, 4, dtype=I32).expand(3, 4)), dict(block_table=torch.zeros(2, 4, dtype=I32)),
    dict(block_table=torch.zeros(9, dtype=I32).as_strided((3, 4), (2, 1))),
    dict(context_lens=torch.zeros(6, dtype=I32)[::2]), dict(context_lens=torch.zeros(3)),
    dict(free_blocks=torch.zeros(0, dtype=I32)), dict(free_blocks=torch.zeros(3, 4, dtype=I32)),
    dict(free_blocks=torch.zeros(24, dtype=I32)[::2]), dict(free_range=torch.zeros(3, dtype=I32)),
    dict(new_lens=torch.zeros(4, dtype=I32)), dict(new_lens=torch.zeros(3, dtype=torch.int64)),
    dict(keep=torch.zeros(2, dtype=I32)), dict(keep=torch.zeros(3)), dict(T=-1), dict(bs=0), dict(bs=2 ** 29), dict(T=2 ** 31),
    dict(window=0), dict(window=5, sinks=-1), dict(sinks=3)])
def test_resize_refuses(calls, kw):
    with pytest.raises(ValueError):
        _resize(**kw)
    assert not calls


def test_resize_refuses_one_tensor_for_two(calls):
    t = torch.zeros(3, dtype=I32)
    for kw in (dict(context_lens=t, new_lens=t), dict(context_lens=t, keep=t)):
        with pytest.raises(ValueError, match="own"):
            _resize(**kw)
    assert not calls
    _resize(new_lens=t, keep=t)


def test_pool():
    table, lens, free, rng = PT.paged_pool(10, 2, 3, "cpu")
    assert table.tolist() == [[-1] * 3] * 2 and lens.tolist() == [0, 0]
    assert free.tolist() == list(range(10)) and rng.tolist() == [0, 10]
    for bad in ((0, 2, 3), (10, 0, 3), (10, 2, 0)):
        with pytest.raises(ValueError):
            PT.paged_pool(*bad, "cpu")


def test_cpu_tensors_are_refused():
    x = _inputs()
    for op in OPS:
        with pytest.raises(ValueError, match="GPU"):
            op(x)
    with pytest.raises(ValueError, match="GPU"):
        _resize()


def test_oracle_of_the_tables():
    """The restatement on a step worked out by hand: blocks of 4, a window of 3."""
    table, lens, ring, rng = [[7, 8, -1, -1], [1, 2, 3, -1]], [8, 9], [0, 4, 5, 6, 9, 9, 9, 9, 9, 9], [0, 4]
    cu, granted, seqs, pos, slots = S.resize(table, lens, ring, rng, [1, 5], 8, 4, keep=[6, 9], window=3, sinks=0)
    # the first keeps 6 of 8 and needs no block; the second's first block lies before token 7, and it enters a fourth
    assert granted == [1, 5] and cu == [0, 1, 6] and lens == [7, 14]
    assert table == [[-1, 8, -1, -1], [-1, 2, 3, 0]]
    assert rng == [1, 5] and ring[4:6] == [7, 1]
    assert slots == [8 * 4 + 2, 3 * 4 + 1, 3 * 4 + 2, 3 * 4 + 3, 0, 1, -1, -1]
    assert seqs == [0, 1, 1, 1, 1, 1, -1, -1] and pos == [6, 9, 10, 11, 12, 13, -1, -1]


def test_c_entries_refuse():
    """The C entries check for themselves and launch nothing."""
    lib, p, n = _lib.lib(), 64, ctypes.c_size_t(0)   # p: never dereferenced
    ref = ctypes.byref(n)
    c4 = (p, 64, 64, 64)
    u = lib.bytes_paged_window_workspace_size
    assert u(4, 8, 2, 64, 3, 16, 100, 50, 4, ref) == 0
    for bad in ((4, 7, 2, 64, 3, 16, 100, 50, 4), (4, 8, 2, 96, 3, 16, 100, 50, 4), (4, 8, 2, 64, 4, 16, 100, 50, 4),
                (4, 8, 2, 64, -1, 16, 100, 50, 4), (4, 8, 2, 64, 3, 0, 100, 50, 4), (4, 8, 2, 64, 3, 16, 100, 0, 4),
                (4, 8, 2, 64, 3, 16, 100, 50, -1), (4, 8, 2, 64, 3, 2 ** 20, 2 ** 11, 50, 4)):
        assert u(*bad, ref), bad
    w = lib.bytes_paged_prompt_workspace_size
    assert w(40, 4, 8, 2, 64, 16, 100, 50, 4, ref) == 0 and w(0, 4, 8, 2, 64, 16, 100, 50, 4, ref) == 0 and n.value == 0
    for bad in ((-1, 4, 8, 2, 64, 16, 100, 50, 4), (40, 0, 8, 2, 64, 16, 100, 50, 4), (40, 4, 9, 2, 64, 16, 100, 50, 4),
                (40, 4, 8, 2, 32, 16, 100, 50, 4), (40, 4, 8, 2, 64, 0, 100, 50, 4), (40, 4, 8, 2, 64, 16, 100, 0, 4)):
        assert w(*bad, ref), bad
    assert u(4, 8, 2, 64, 3, 16, 100, 50, 4, None) and w(40, 4, 8, 2, 64, 16, 100, 50, 4, None)
    assert lib.bytes_paged_resize_workspace_size(0, ref) and lib.bytes_paged_resize_workspace_size(3, None)

    def window(B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4096, q=p, typ=3, ks=p, vs=p, win=2 ** 30, sinks=0, ws=p, wb=1 << 30):
        return lib.bytes_paged_window_attn(q, 64, 64, *c4, *c4, typ, ks, 2, 1, vs, 2, 1, p, W, p, p, 64, 64, B, Hq, Hk, D, bs,
                                           N, W, win, sinks, 1.0, 1.0, ws, wb, None)
    for bad in (dict(q=None), dict(B=0), dict(B=65536), dict(Hq=7), dict(D=32), dict(bs=0), dict(N=0), dict(W=0),
                dict(W=2 ** 27), dict(ws=None), dict(wb=100), dict(typ=4), dict(typ=-1), dict(ks=None), dict(vs=None),
                dict(typ=2, ks=None), dict(win=0), dict(sinks=-1)):
        assert window(**bad), bad

    def prompt(T=40, B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4096, q=p, typ=3, ks=p, vs=p, win=2 ** 30, sinks=0, ws=p,
               wb=1 << 30, cu=p):
        return lib.bytes_paged_prompt_attn(q, 64, 64, *c4, *c4, typ, ks, 2, 1, vs, 2, 1, p, W, p, cu, p, 64, 64, T, B, Hq, Hk,
                                           D, bs, N, W, win, sinks, 1.0, 1.0, ws, wb, None)
    for bad in (dict(q=None), dict(cu=None), dict(T=-1), dict(B=0), dict(Hq=7), dict(D=32), dict(bs=0), dict(N=0), dict(W=0),
                dict(W=2 ** 27), dict(ws=None), dict(wb=100), dict(typ=4), dict(ks=None), dict(vs=None), dict(win=0),
                dict(sinks=-1), dict(T=2 ** 30, Hq=8, Hk=1)):
        assert prompt(**bad), bad
    assert prompt(T=0) == 0                          # nothing to do

    def append(T=3, B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4, rot=64, P=64, q=p, qo=p, typ=3, ks=p, vs=p, cu=None, cos=p, k=p):
        return lib.bytes_paged_kv_append_blocks(k, 64, 64, p, 64, 64, q, 64, 64, qo, 64, 64, *c4, *c4, typ, ks, 2, 1, vs, 2, 1,
                                                p, W, p, cu, cos, 32, cos, 32, P, rot, 0, T, B, Hq, Hk, D, bs, N, W, None)
    for bad in (dict(k=None), dict(T=4), dict(T=-1), dict(B=0), dict(Hk=0), dict(D=96), dict(rot=24), dict(rot=80), dict(P=63),
                dict(cos=None), dict(q=None), dict(qo=None), dict(Hq=0), dict(typ=1), dict(typ=4), dict(ks=None),
                dict(vs=None), dict(bs=0), dict(N=0), dict(W=0), dict(W=2 ** 27)):
        assert append(**bad), bad
    assert append(T=0, cu=p) == 0

    def resize(B=3, W=4, N=12, T=20, bs=16, win=0, sinks=0, table=p, ws=p, wb=1 << 20, seqs=p):
        return lib.bytes_paged_resize(table, W, p, p, p, None, p, p, p, seqs, p, p, B, W, N, T, bs, win, sinks, ws, wb, None)
    for bad in (dict(B=0), dict(W=0), dict(N=0), dict(T=-1), dict(bs=0), dict(win=-1), dict(sinks=-1), dict(sinks=2),
                dict(table=None), dict(ws=None), dict(wb=10), dict(seqs=None), dict(W=2 ** 27), dict(T=2 ** 30 + 1)):
        assert resize(**bad), bad


def test_one_element_scales_of_a_cache_of_one_block_and_head(calls):
    """Tensors of one element are numbers, as they are for every other cache, unless both can be nothing but the
    scales of an 8-bit cache's only block and head."""
    one = torch.ones(1, 1)
    x = _inputs(dtype=BF16, Hk=1, N=1, W=1)
    meta = (torch.zeros(1, 1, 64, dtype=BF16), torch.zeros(1, 1, 64, dtype=BF16))
    for op in OPS:
        assert op(x, k_scale=one, v_scale=one).shape[1] == 8                 # (a bf16 cache's: 1.0)
        with pytest.raises(ValueError, match="no scale"):
            op(x, k_scale=one * 0.5, v_scale=one)
    assert {n for n, _ in calls if not n.endswith("_size")} == {"bytes_paged_kv_append", "bytes_paged_decode_attn",
                                                               "bytes_paged_prompt_attn"}
    x = _inputs(dtype=F8, Hk=1, N=1, W=1)
    for k, v in ((one * 0.5, 0.25), (0.5, one * 0.25), (one.double() * 0.5, one.double() * 0.25), (one * 0.5, torch.tensor(0.25)),
                 (torch.tensor([0.5]), one * 0.25)):
        calls.clear()
        _decode(x, k_scale=k, v_scale=v), _append(x, k_scale=k, v_scale=v), _prompt(x, k_scale=k, v_scale=v)
        made = {n: a for n, a in calls if not n.endswith("_size")}
        assert made["bytes_paged_decode_attn"][-5:-3] == (0.0625, 0.25)
        assert made["bytes_paged_kv_append"][-11:-9] == (0.5, 0.25)
        assert made["bytes_paged_prompt_attn"][11] == 1 and made["bytes_paged_prompt_attn"][-5:-3] == (0.0625, 0.25)
    calls.clear()                                    # the page-sparse decode knows numbers only
    PG.paged_quest_decode(x["q"], x["kc"], x["vc"], meta, x["bt"], x["cl"], 16, 0.125, k_scale=one * 0.5, v_scale=one * 0.25)
    assert calls[-1][0] == "bytes_paged_quest_attn" and calls[-1][1][-5:-3] == (0.0625, 0.25)
    for dtype in (F8, I8):
        x = _inputs(dtype=dtype, Hk=1, N=1, W=1)
        _append(x), _prompt(x), _decode(x)
        assert calls[-1][0] == "bytes_paged_window_attn" and calls[-1][1][11] == (2 if dtype == F8 else 3)
