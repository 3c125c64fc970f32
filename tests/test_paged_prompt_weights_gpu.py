"""paged_prompt_attn over few rows: weights that lose nothing that the result shows."""
import pytest
import torch

import serving_oracle as S
from test_paged_blocks_gpu import KINDS
from test_paged_prompt_gpu import _batch, _run
from bytes_amd import paged as PG

pytestmark = pytest.mark.gpu


def tolerance(out, mag, dots, D):
    """|error|: half a bf16 step of the result, 2^-8; each weight as two bf16 numbers, of which the second, at most
    2^-7 of it, is rounded by 2^-9 of itself, 2^-16 of the weighted |v|; scores off by D roundings of 2^-24 of their
    products and a few more, in numerator and denominator; fp32 sums and exponentials 2^-16."""
    return 2.0 ** -8 * out.abs() + mag * (2.0 ** -16 + 2 * (D + 4) * 2.0 ** -24 * dots + 2.0 ** -16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,new,Hq,Hk,D,bs,window", [
    ([9000, 4000], [8, 3], 24, 8, 128, 16, None), ([9000, 4000], [8, 3], 24, 8, 128, 20, None), ([6000], [4], 14, 2, 64, 16, None),
    ([333, 245], [300, 171], 14, 2, 64, 16, 128), ([500], [500], 8, 2, 128, 16, None), ([1500, 700], [40, 90], 8, 8, 64, 24, 600)])
def test_rows_are_off_by_their_own_rounding(dev, kind, lens, new, Hq, Hk, D, bs, window):
    """Drafts and short prompts against 64 bits, without an allowance for weights of 8 bits.  (Drafts of up to 32
    rows, tokens times heads of a group: more of them over a long context take the form for many rows.)"""
    g = torch.Generator().manual_seed(sum(lens))
    q, kc, vc, ks, vs, table, n, cu = _batch(g, lens, new, bs, Hq, Hk, D, kind)
    kw = dict(window=window, sinks=4) if window else {}
    print(f"weights {kind} lens {lens} new {new} Hq{Hq} D{D}", flush=True)
    out = _run(dev, q, kc, vc, ks, vs, table, n, cu, D ** -0.5, **kw).double().cpu()
    rows = sorted(set(range(0, q.shape[0], 13)) | {q.shape[0] - 1})
    at = S.positions(q.shape[0], table, n, cu, bs)
    want, mag, dots = S.attend_rows(q[rows], [at[r] for r in rows], kc, vc, D ** -0.5, ks, vs, table, n, window, kw.get("sinks", 0))
    bad = ~((out[rows] - want).abs() <= tolerance(want, mag, dots, D))
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), bad.nonzero()[:5].tolist())


def test_a_draft_is_its_decode(dev):
    """The last draft's row and the same token decoded alone: off by a bf16 step at most, and rarely."""
    g = torch.Generator().manual_seed(5)
    for kind in KINDS:
        q, kc, vc, ks, vs, table, n, cu = _batch(g, [9000, 4000], [8, 3], 16, 24, 8, 128, kind)
        out = _run(dev, q, kc, vc, ks, vs, table, n, cu, 128 ** -0.5)[cu[1:].long() - 1]
        put = lambda t: t.to(dev) if torch.is_tensor(t) else t               # noqa: E731
        one = PG.paged_decode_attn(q[cu[1:].long() - 1][:, :, None].to(dev), put(kc), put(vc), put(table), put(n), 128 ** -0.5,
                                   k_scale=put(ks), v_scale=put(vs))[:, :, 0]
        assert float((out != one).float().mean()) < 0.05, kind
