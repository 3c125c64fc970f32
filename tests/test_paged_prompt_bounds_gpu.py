"""bytes_paged_prompt_attn over offsets and lengths that are none, with all that it writes cut out of
larger buffers whose surroundings are checked.  (test_prompt_tiles.py runs the same arithmetic on
the host over many more.)"""
import pytest
import torch

from bytes_amd import _lib
from bytes_amd import paged as PG

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32


class Call:
    """T rows of B sequences over full tables of `cap` tokens, through the C ABI."""

    def __init__(self, dev, B, T, Hq, Hk, D, cap, bs=16):
        g = torch.Generator().manual_seed(B + T)
        r = lambda *s: (torch.randn(*s, generator=g) * 0.5).to(BF16).to(dev)                 # noqa: E731
        self.B, self.T, self.Hq, self.Hk, self.D, self.bs, self.W = B, T, Hq, Hk, D, bs, cap // bs
        self.q, self.k, self.v = r(T, Hq, D), r(self.W, Hk, bs, D), r(self.W, Hk, bs, D)
        self.table = torch.stack([torch.randperm(self.W, generator=g) for _ in range(B)]).to(I32).to(dev)
        self.n = _lib.size_query("bytes_paged_prompt_workspace_size", T, B, Hq, Hk, D, bs, self.W, 2 ** 30, 0)
        self.pad = 4 << 20
        self.ws = torch.full((self.n + 2 * self.pad,), 0xA5, dtype=torch.uint8, device=dev)
        self.out = torch.full((T + 64, Hq, D), 7.0, dtype=BF16, device=dev)
        self.dev = dev

    def run(self, lens, cu):
        """-> out; nothing beside it and beside the workspace has changed."""
        lens, cu = (torch.tensor(x, dtype=I32, device=self.dev) for x in (lens, cu))
        self.out.fill_(7.0)
        q, k, v, out = self.q, self.k, self.v, self.out[32:-32]
        _lib.call("bytes_paged_prompt_attn", q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), *k.stride()[:3],
                  v.data_ptr(), *v.stride()[:3], 0, None, 0, 0, None, 0, 0, self.table.data_ptr(), self.table.stride(0),
                  lens.data_ptr(), cu.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), self.T, self.B, self.Hq,
                  self.Hk, self.D, self.bs, self.W, self.W, 2 ** 30, 0, self.D ** -0.5, 1.0, self.ws.data_ptr() + self.pad,
                  self.n, _lib.stream_of(q))
        torch.cuda.synchronize()
        assert bool((self.ws[:self.pad] == 0xA5).all()) and bool((self.ws[self.pad + self.n:] == 0xA5).all())
        assert bool((self.out[:32] == 7.0).all()) and bool((self.out[-32:] == 7.0).all())
        return out

    def check(self, lens, cu):
        """A call that is one, against the decode of some of its rows."""
        out = self.run(lens, cu)
        for b in range(self.B):
            for i in {0, (cu[b + 1] - cu[b]) // 2, cu[b + 1] - cu[b] - 1}:
                p = lens[b] - (cu[b + 1] - cu[b]) + i
                ref = PG.paged_decode_attn(self.q[None, cu[b] + i, :, None], self.k, self.v, self.table[b:b + 1],
                                           torch.tensor([p + 1], dtype=I32, device=self.dev), self.D ** -0.5)[0, :, 0].float()
                assert float((out[cu[b] + i].float() - ref).norm() / ref.norm()) < 0.01, (b, i)


CALLS = [(5, 1000, 8, 2, 128), (4, 640, 8, 2, 128), (5, 1500, 14, 2, 64), (70, 1000, 8, 1, 128)]


@pytest.mark.parametrize("B,T,Hq,Hk,D", CALLS)
def test_offsets_that_overlap(dev, B, T, Hq, Hk, D):
    """More row tiles than the workspace has room for."""
    c = Call(dev, B, T, Hq, Hk, D, 16000)
    assert c.n > 0                                   # keys in parts
    lens = [15000 - 7 * b for b in range(B)]
    for cu in ([T * (b % 2) for b in range(B + 1)], [(b * T // 3) % T for b in range(B + 1)], [0] + [2 ** 31 - 1, -5] * B):
        print(f"offsets {cu[:B + 1]}", flush=True)
        c.run(lens, cu[:B + 1])
    c.check(lens, [b * T // B for b in range(B + 1)])


@pytest.mark.parametrize("B,T,Hq,Hk,D", [(2, 700, 32, 8, 128), (5, 1500, 14, 2, 64), (70, 1000, 8, 1, 128), (3, 20, 8, 2, 64)])
def test_lengths_below_their_new_tokens(dev, B, T, Hq, Hk, D):
    """Down to -2^31: zeros, and the other sequences' rows as they are."""
    c = Call(dev, B, T, Hq, Hk, D, 6000)
    lens, cu = [5900 - 7 * b for b in range(B)], [b * T // B for b in range(B + 1)]
    want = c.run(lens, cu).clone()
    c.check(lens, cu)
    for low in (-2 ** 31, -2 ** 31 + 1, -2 ** 31 + T // B, -1, 0):
        some = [low if b % 2 else n for b, n in enumerate(lens)]
        print(f"lengths {some[:4]}", flush=True)
        out = c.run(some, cu)
        for b in range(B):
            rows = slice(cu[b], cu[b + 1])
            if b % 2:
                assert not bool(out[rows].any()), (low, b)
            elif T > 32 * B // (Hq // Hk):
                assert torch.equal(out[rows], want[rows]), (low, b)
            else:
                # few rows: keys are dealt by all lengths, so sums are cut elsewhere; each result is within 0.005 of the
                # decode's in norm (test_long_prompt_rows), so they are within twice that of each other
                diff = float((out[rows].float() - want[rows].float()).norm() / want[rows].float().norm())
                assert diff < 0.01, (low, b, diff)


@pytest.mark.parametrize("T", [8, 200, 3000])
def test_a_scale_that_is_no_number(dev, T):
    """NaN in every row that sees a token, as paged_decode_attn gives; zeros in the others."""
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(300, 2, 16, 64, generator=g).to(BF16).to(dev) for _ in "kv")
    q = torch.randn(T + 3, 8, 64, generator=g).to(BF16).to(dev)
    table = torch.randperm(300, generator=g).to(I32).to(dev).view(1, 300)
    lens, cu = torch.tensor([T - 2], dtype=I32, device=dev), torch.tensor([0, T], dtype=I32, device=dev)
    for kw in ({}, dict(window=50, sinks=3)):
        out = PG.paged_prompt_attn(q, k, v, table, lens, cu, float("nan"), **kw)
        assert bool(out[2:T].isnan().all()) and not bool(out[:2].any()) and not bool(out[T:].any())
        one = PG.paged_decode_attn(q[None, T - 1, :, None], k, v, table, lens, float("nan"), **kw)
        assert bool(one.isnan().all())
