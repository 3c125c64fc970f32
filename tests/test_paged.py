"""bytes_amd.paged without a GPU: what it refuses, and what it hands to the C ABI."""
import contextlib

import pytest
import torch

from bytes_amd import _lib
from bytes_amd import paged as PG

F8, BF16, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.int32


@pytest.fixture
def calls(monkeypatch):
    """Launches are recorded and not made; CPU tensors stand for the GPU's."""
    made = []
    monkeypatch.setattr(PG.C, "cuda_tensors", lambda *ts: [t.device for t in ts] and ts[0].device)
    monkeypatch.setattr(PG, "call", lambda name, *a: made.append((name, a)))
    monkeypatch.setattr(PG, "size_query", lambda name, *a: made.append((name, a)) or 4096)
    monkeypatch.setattr(PG, "_topk", lambda s, k, **kw: torch.zeros(*s.shape[:-1], k, dtype=I32))
    monkeypatch.setattr(PG, "stream_of", lambda t: 0)
    monkeypatch.setattr(PG.torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "_native", _lib._NoNative())
    return made


def _inputs(B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4, fp8=False, T=None):
    T = B if T is None else T
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt)                       # noqa: E731
    return dict(k=z(T, Hk, D), v=z(T, Hk, D), q3=z(T, Hq, D), q=z(B, Hq, 1, D), kc=z(N, Hk, bs, D).to(F8 if fp8 else BF16),
                vc=z(N, Hk, bs, D).to(F8 if fp8 else BF16), bt=z(B, W, dt=I32), cl=z(B, dt=I32), kmin=z(N, Hk, D),
                kmax=z(N, Hk, D), cos=z(W * bs, D // 2, dt=torch.float32), sin=z(W * bs, D // 2, dt=torch.float32))


def _append(x, **kw):
    a = dict(cos=x["cos"], sin=x["sin"], q=x["q3"], meta=(x["kmin"], x["kmax"]))
    a.update(kw)
    return PG.paged_kv_append(x["k"], x["v"], x["kc"], x["vc"], x["bt"], x["cl"], **a)


def _decode(x, **kw):
    return PG.paged_decode_attn(x["q"], x["kc"], x["vc"], x["bt"], x["cl"], 0.125, **kw)


def _quest(x, kb=32, **kw):
    return PG.paged_quest_decode(x["q"], x["kc"], x["vc"], (x["kmin"], x["kmax"]), x["bt"], x["cl"], kb, 0.125, **kw)


def test_calls_reach_the_abi_with_its_signatures(calls):
    """Every recorded call has as many arguments as the ABI's signature."""
    x = _inputs()
    out = _append(x)
    assert out.shape == (3, 8, 64) and _append(x, q=None, meta=None, cos=None, sin=None) is None
    assert _decode(x).shape == (3, 8, 1, 64) and _quest(x).shape == (3, 8, 1, 64)
    out, pages = _quest(x, return_pages=True)
    assert pages.shape == (3, 8, 2)
    assert PG.paged_page_scores(x["q"], (x["kmin"], x["kmax"]), x["bt"], x["cl"], 16).shape == (3, 8, 4)
    seen = set()
    for name, a in calls:
        sig = _lib.SIGNATURES[name]
        assert len(a) == len(sig) - (1 if name.endswith("_size") else 0), name
        seen.add(name)
    assert {"bytes_paged_kv_append", "bytes_paged_decode_attn", "bytes_paged_page_scores", "bytes_paged_quest_attn"} <= seen


def test_scales_and_strides(calls):
    x = _inputs(fp8=True, T=10)
    qkv = torch.zeros(10, 12, 64, dtype=BF16)
    x["q3"], x["k"], x["v"] = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    _append(x, cu_seqlens=torch.zeros(4, dtype=I32), k_scale=0.5, v_scale=0.25, interleaved=True)
    name, a = calls[-1]
    s = dict(zip(("k_st", "k_sh"), a[1:3]))
    assert s == {"k_st": 12 * 64, "k_sh": 64} and a[20] == 1 and a[-11:-9] == (0.5, 0.25)
    assert a[-9:-2] == (10, 3, 8, 2, 64, 16, 12)                            # T, B, Hq, Hk, D, block size, blocks
    x = _inputs(fp8=True)
    calls.clear()
    _decode(x, k_scale=0.5, v_scale=0.25)
    assert calls[-1][1][-5:-3] == (0.0625, 0.25)                            # scale * k_scale, v_scale


def test_wide_tables_are_held_to_int32(calls):
    x = _inputs()
    t = torch.tensor([[2 ** 32 + 1, -5, 3, 2 ** 31]], dtype=torch.int64).repeat(3, 1)
    bt, cl = PG._tables(t, torch.tensor([5, -2 ** 40, 2 ** 40]), 3, 16)
    assert bt.dtype == I32 and bt[0].tolist() == [2 ** 31 - 1, -1, 3, 2 ** 31 - 1]
    assert cl.tolist() == [5, -1, 2 ** 31 - 1]


def test_no_tokens(calls):
    x = _inputs(T=0)
    out = _append(x, cu_seqlens=torch.zeros(4, dtype=I32))
    assert out.shape == (0, 8, 64) and not [n for n, _ in calls if n == "bytes_paged_kv_append"]


def _bad(name, **change):
    return pytest.param(change, id=name)


COMMON = [
    _bad("cache dtypes differ", vc=lambda t: t.to(F8)),
    _bad("cache dtype", kc=lambda t: t.float(), vc=lambda t: t.float()),
    _bad("cache shapes differ", vc=lambda t: t[1:]),
    _bad("cache rank", kc=lambda t: t[0], vc=lambda t: t[0]),
    _bad("no blocks", kc=lambda t: t[:0], vc=lambda t: t[:0]),
    _bad("no rows", kc=lambda t: t[:, :, :0], vc=lambda t: t[:, :, :0]),
    _bad("rows off 16 bytes", kc=lambda t: torch.zeros(12, 2, 16, 65, dtype=BF16)[..., 1:]),
    _bad("row stride off 16 bytes", vc=lambda t: torch.zeros(12, 2, 16, 65, dtype=BF16)[..., :64]),
    _bad("strided dims", kc=lambda t: torch.zeros(12, 2, 64, 16, dtype=BF16).transpose(2, 3)),
    _bad("table rank", bt=lambda t: t[0]),
    _bad("table dtype", bt=lambda t: t.float()),
    _bad("table without columns", bt=lambda t: t[:, :0]),
    _bad("lengths dtype", cl=lambda t: t.double()),
    _bad("lengths shape", cl=lambda t: t[:2]),
    _bad("lengths rank", cl=lambda t: t[:, None]),
    _bad("positions past 2^30", bt=lambda t: torch.zeros(3, 1, dtype=I32).expand(3, 2 ** 26 + 1)),
]


@pytest.mark.parametrize("change", COMMON)
@pytest.mark.parametrize("op", [_append, _decode, _quest])
def test_refuses_caches_and_tables(calls, op, change):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        op(x)
    assert not [n for n, _ in calls if not n.endswith("_size")]


@pytest.mark.parametrize("op", [_append, _decode, _quest])
@pytest.mark.parametrize("kw", [dict(k_scale=2.0), dict(v_scale=0.5)])
def test_refuses_scales_of_a_bf16_cache(calls, op, kw):
    with pytest.raises(ValueError, match="scale"):
        op(_inputs(), **kw)


@pytest.mark.parametrize("op", [_append, _decode, _quest])
@pytest.mark.parametrize("s", [0.0, -1.0, float("nan"), float("inf")])
def test_refuses_bad_scales(calls, op, s):
    with pytest.raises(ValueError, match="scale"):
        op(_inputs(fp8=True), k_scale=s)


@pytest.mark.parametrize("change", [
    _bad("head dim", q=lambda t: t[..., :32]),
    _bad("two tokens", q=lambda t: t.expand(3, 8, 2, 64)),
    _bad("query dtype", q=lambda t: t.half()),
    _bad("query rank", q=lambda t: t[:, :, 0]),
    _bad("heads", q=lambda t: t[:, :7]),
    _bad("batch", q=lambda t: t[:2]),
    _bad("no batch", q=lambda t: t[:0], bt=lambda t: t[:0], cl=lambda t: t[:0]),
])
@pytest.mark.parametrize("op", [_decode, _quest])
def test_refuses_queries(calls, op, change):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        op(x)


@pytest.mark.parametrize("change", [
    _bad("min dtype", kmin=lambda t: t.float()),
    _bad("max shape", kmax=lambda t: t[1:]),
    _bad("max strides", kmax=lambda t: torch.zeros(2, 12, 64, dtype=BF16).transpose(0, 1)),
])
@pytest.mark.parametrize("op", [_append, _quest])
def test_refuses_metadata(calls, op, change):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        op(x)


def test_refuses_selection_arguments(calls):
    x = _inputs()
    for bad in (dict(kb=0), dict(kb=-3), dict(local_w=-1)):
        with pytest.raises(ValueError):
            _quest(x, **bad)
    for bs in (0, -16):
        with pytest.raises(ValueError):
            PG.paged_page_scores(x["q"], (x["kmin"], x["kmax"]), x["bt"], x["cl"], bs)
    with pytest.raises(ValueError):
        PG.paged_page_scores(x["q"], (x["kmin"][..., :32], x["kmax"][..., :32]), x["bt"], x["cl"], 16)


@pytest.mark.parametrize("change,kw", [
    (dict(k=lambda t: t[:, :1]), {}), (dict(v=lambda t: t.half()), {}), (dict(v=lambda t: t[:2]), {}),
    (dict(k=lambda t: t[:2], v=lambda t: t[:2], q3=lambda t: t[:2]), {}),                     # two rows, three sequences
    (dict(q3=lambda t: t[:2]), {}), (dict(q3=lambda t: t.float()), {}), (dict(q3=lambda t: t[:, :0]), {}),
    (dict(q3=lambda t: t[..., :32]), {}),
    ({}, dict(cu_seqlens=torch.zeros(3, dtype=I32))), ({}, dict(cu_seqlens=torch.zeros(4))),
    ({}, dict(cos=None)), ({}, dict(sin=None)),
    (dict(cos=lambda t: t[:-1], sin=lambda t: t[:-1]), {}),                                   # too few positions
    (dict(cos=lambda t: t[:, :12], sin=lambda t: t[:, :12]), {}),                             # 24 dims
    (dict(cos=lambda t: t.repeat(1, 2), sin=lambda t: t.repeat(1, 2)), {}),                   # 128 dims of 64
    (dict(cos=lambda t: t[:, :0], sin=lambda t: t[:, :0]), {}),
    (dict(cos=lambda t: t.to(BF16), sin=lambda t: t.to(BF16)), {}), (dict(sin=lambda t: t[:, :16]), {}),
])
def test_refuses_new_tokens(calls, change, kw):
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError):
        _append(x, **kw)
    assert not calls


def test_cpu_tensors_are_refused():
    x = _inputs()
    for op in (_append, _decode, _quest):
        with pytest.raises(ValueError, match="GPU"):
            op(x)




def test_c_entries_refuse(monkeypatch):
    """The C entries check for themselves and launch nothing."""
    import ctypes
    lib = _lib.lib()
    n = ctypes.c_size_t(0)
    q = lib.bytes_paged_decode_workspace_size
    assert q(4, 8, 2, 64, 0, 16, 100, ctypes.byref(n)) == 0
    assert q(4, 7, 2, 64, 0, 16, 100, ctypes.byref(n)) and q(4, 8, 2, 96, 0, 16, 100, ctypes.byref(n))
    assert q(4, 8, 2, 64, 0, 0, 100, ctypes.byref(n)) and q(4, 8, 2, 64, 0, 2 ** 20, 2 ** 11, ctypes.byref(n))
    assert q(4, 8, 2, 64, 0, 16, 100, None)
    u = lib.bytes_paged_quest_workspace_size
    assert u(4, 8, 2, 64, 0, 16, 100, 10, ctypes.byref(n)) == 0 and u(4, 8, 2, 64, 0, 16, 100, 0, ctypes.byref(n))
    p = 64                                            # never dereferenced: every call below is refused
    k3, c4 = (p, 64, 64), (p, 64, 64, 64)
    # T, B, Hq, Hk, D, block size, blocks, max blocks
    def append(T=3, B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4, rot=64, P=64, q=p, qo=p, mn=p, mx=p, cu=None, cos=p, k=p):
        return lib.bytes_paged_kv_append(k, 64, 64, *k3, q, 64, 64, qo, 64, 64, *c4, *c4, 0, mn, mx, p, W, p, cu, cos, 32,
                                         cos, 32, P, rot, 0, 1.0, 1.0, T, B, Hq, Hk, D, bs, N, W, None)
    for bad in (dict(k=None), dict(T=4), dict(T=-1), dict(B=0), dict(Hk=0), dict(D=96), dict(rot=24), dict(rot=80), dict(P=63),
                dict(cos=None), dict(q=None), dict(qo=None), dict(Hq=0), dict(mn=None), dict(mx=None), dict(bs=0),
                dict(N=0), dict(W=2 ** 27)):
        assert append(**bad), bad
    assert append(T=0, B=3, cu=p) == 0                # nothing to do
    def decode(B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4096, q=p, ws=p, wb=1 << 30):
        return lib.bytes_paged_decode_attn(q, 64, 64, *c4, *c4, 0, p, W, p, p, 64, 64, B, Hq, Hk, D, bs, N, W, 1.0, 1.0, ws,
                                           wb, None)
    for bad in (dict(q=None), dict(B=0), dict(B=65536), dict(Hq=7), dict(D=32), dict(bs=0), dict(N=0), dict(W=0),
                dict(W=2 ** 27), dict(ws=None), dict(wb=100)):
        assert decode(**bad), bad
    def quest(npick=4, W=4096, bound=p, pages=None, ws=p, wb=1 << 30, **kw):
        B, Hq, Hk, D, bs, N = (kw.get(n, d) for n, d in (("B", 3), ("Hq", 8), ("Hk", 2), ("D", 64), ("bs", 64), ("N", 12)))
        return lib.bytes_paged_quest_attn(p, 64, 64, *c4, *c4, 0, bound, 64, 64, pages, 64, 64, npick, p, W, p, p, 64, 64, B,
                                          Hq, Hk, D, bs, N, W, 1.0, 1.0, ws, wb, None)
    for bad in (dict(npick=0), dict(npick=5000), dict(bound=None), dict(W=16385), dict(D=32), dict(Hq=7), dict(N=0),
                dict(npick=1000, ws=None), dict(npick=1000, wb=16), dict(W=8192, ws=None)):
        assert quest(**bad), bad
    def scores(B=3, Hq=8, Hk=2, D=64, bs=16, N=12, W=4, local=0, q=p):
        return lib.bytes_paged_page_scores(q, 64, 64, p, p, p, W, p, p, 64, 64, B, Hq, Hk, D, bs, N, W, local, -1, 1.0, None)
    for bad in (dict(q=None), dict(B=0), dict(B=70000), dict(Hq=9), dict(D=100), dict(bs=0), dict(W=0), dict(local=-1)):
        assert scores(**bad), bad


def test_append_entry_refuses_tables_without_columns():
    """The append reads a table's first column also for tokens that have no position."""
    lib, p = _lib.lib(), 64                           # never dereferenced: refused before a launch
    c4 = (p, 64, 64, 64)
    for W in (0, -1):
        for cu, rot in ((None, 0), (p, 0), (None, 64), (p, 64)):
            assert lib.bytes_paged_kv_append(p, 64, 64, p, 64, 64, p, 64, 64, p, 64, 64, *c4, *c4, 0, p, p, p, W, p, cu, p,
                                             32, p, 32, 64, rot, 0, 1.0, 1.0, 3, 3, 8, 2, 64, 16, 12, W, None) == 1


@pytest.mark.parametrize("change", [
    _bad("blocks in one place", kc=lambda t: t[:1].expand(12, 2, 16, 64)),
    _bad("heads in one place", vc=lambda t: t[:, :1].expand(12, 2, 16, 64)),
    _bad("rows in one place", vc=lambda t: t[:, :, :1].expand(12, 2, 16, 64)),
])
def test_append_refuses_caches_that_overlap_themselves(calls, change):
    """Two writes of one call to the same place; decode only reads and takes them."""
    x = _inputs()
    for n, f in change.items():
        x[n] = f(x[n])
    with pytest.raises(ValueError, match="expanded"):
        _append(x)
    assert not calls
    assert _decode(x).shape == (3, 8, 1, 64)


def test_append_refuses_one_tensor_for_two(calls):
    x = _inputs()
    for a, b in (("kc", "vc"), ("kmin", "kmax")):
        with pytest.raises(ValueError, match="same memory"):
            _append({**x, b: x[a]})
    assert not calls
    assert _decode({**x, "vc": x["kc"]}).shape == (3, 8, 1, 64)
