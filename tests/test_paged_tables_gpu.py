"""bytes_amd.paged_tables against a restatement on lists: whole numbers, all equal."""
import random

import pytest
import torch

import serving_oracle as S
from test_native_path_gpu import _both
from bytes_amd import paged_tables as PT

pytestmark = pytest.mark.gpu
I32 = torch.int32


class State:
    """Tables on the device and their twin on lists."""

    def __init__(self, dev, N, B, W, bs, pad=0, seed=0):
        r = random.Random(seed)
        self.dev, self.bs, self.wide = dev, bs, torch.full((B, W + pad), 77, dtype=I32, device=dev)
        self.table, self.lens, self.free, self.range = PT.paged_pool(N, B, W, dev)
        if pad:                                      # rows with something of another's between them
            self.wide[:, :W] = self.table
            self.table = self.wide[:, :W]
        order = list(range(N))
        r.shuffle(order)
        head = r.randrange(N)
        ring = order[N - head:] + order[:N - head]
        self.free.copy_(torch.tensor(ring, dtype=I32))
        self.range.copy_(torch.tensor([head, N], dtype=I32))
        self.twin = [self.table.tolist(), self.lens.tolist(), ring, [head, N]]

    def step(self, new, T, keep=None, window=None, sinks=0):
        t = lambda x: torch.tensor(x, dtype=I32, device=self.dev)             # noqa: E731
        got = PT.paged_resize(self.table, self.lens, self.free, self.range, t(new), T, self.bs,
                              keep=None if keep is None else t(keep), window=window, sinks=sinks)
        want = S.resize(*self.twin, new, T, self.bs, keep, window or 0, sinks)
        self.check(got, want)
        return got

    def check(self, got, want):
        for name, w in zip(got._fields, want):
            assert getattr(got, name).tolist() == w, name
        for name, g, w in zip(("table", "lens", "free", "range"), (self.table, self.lens, self.free, self.range), self.twin):
            assert g.tolist() == w, name
        if self.wide.shape[1] > self.table.shape[1]:
            assert bool((self.wide[:, self.table.shape[1]:] == 77).all())


def _walk(st, r, B, W, bs, T, steps, window, sinks):
    cap = W * bs
    for i in range(steps):
        lens = st.twin[1]
        keep = None
        if r.random() < 0.7:
            keep = [r.choice([n, n, max(0, n - r.randint(0, 3 * bs)), 0, cap + 9, -4]) for n in lens]
        new = [r.choice([1, 1, r.randint(0, 4 * bs), 0, -3, r.randint(0, cap), cap + 1]) for _ in range(B)]
        st.step(new, r.choice([T, T, T // 2, 0]), keep, window, sinks)


@pytest.mark.parametrize("B,W,bs,T", [(1, 1, 1, 1), (1, 9, 16, 200), (3, 40, 5, 100), (70, 30, 16, 3000), (64, 8, 64, 2048),
                                      (65, 8, 7, 700), (600, 12, 16, 9000), (40, 300, 1, 4000)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (20, 4), (64, 33), (10 ** 9, 0)])
def test_steps(dev, B, W, bs, T, window, sinks):
    """Random steps: tokens taken back, requests ended and begun, rows, pools and batches that
    are too small, windows that leave blocks behind."""
    r = random.Random(B * 1000 + W)
    print(f"tables B{B} W{W} bs{bs} T{T} window {window} sinks {sinks}", flush=True)
    st = State(dev, max(2, B * W * 2 // 3), B, W, bs, pad=3 if B % 2 else 0, seed=B)
    _walk(st, r, B, W, bs, T, 8, window, sinks)
    used = [i for row in st.twin[0] for i in row if i >= 0]
    head, count = st.twin[3]
    free = [st.twin[2][(head + i) % len(st.twin[2])] for i in range(count)]
    assert sorted(used + free) == list(range(len(st.twin[2])))               # no block lost, none twice


@pytest.mark.parametrize("B", [512, 513, 4096, 4097, 5000])
def test_many_sequences(dev, B):
    """More sequences than a workgroup has threads, and than fit the fill's LDS."""
    r = random.Random(B)
    st = State(dev, 3 * B, B, 6, 4, seed=1)
    _walk(st, r, B, 6, 4, 4 * B, 3, None, 0)


@pytest.mark.parametrize("places", [3, 4, 5, 63, 64, 65, 130, 400])
def test_rows_that_give_back_many_blocks(dev, places):
    """Runs and ends at a thread's and a wave's limits, with holes among the blocks that come back."""
    for bs in (1, 16):
        st = State(dev, 4 * places + 8, 3, places + 2, bs, seed=places)
        n = places * bs
        st.step([n, n - 1, n], 3 * n)
        st.step([1, 0, 2], 8, keep=[n, 0, n - 1], window=2 * bs, sinks=1)   # the first row's run, the second's all
        st.step([0, n, 1], n + 8, keep=[0, 0, 3 * bs], window=2 * bs, sinks=1)   # an end past the run's holes
    hole = State(dev, 4 * places + 8, 1, places + 2, 1, seed=9)
    hole.step([places], places)
    for j in (0, places // 2):
        hole.twin[0][0][j] = hole.table[0, j] = [-1, 2 ** 30][j > 0]
    hole.step([1], 4, window=1)                      # down to the hole; what is below stays until the end
    hole.step([2], 4, keep=[0])


def test_refused_rows_and_their_followers(dev):
    """A sequence that asks for more than is free gets nothing, nor do those after it that need
    a block; those that need none do."""
    st = State(dev, 10, 4, 8, 4)
    st.step([8, 3, 4, 8], 64)                        # 2 + 1 + 1 + 2 blocks: 4 are free
    got = st.step([20, 1, 1, 1], 64)                 # 5 blocks of 4; none; 1; 1
    assert got.granted.tolist() == [0, 1, 0, 0]
    got = st.step([1, 1, 1, 1], 2, keep=[8, 2, 4, 5])
    assert got.granted.tolist() == [1, 1, 0, 0]      # two rows of the batch; the first takes a block: 3 are free
    got = st.step([1, 4, 2, 0], 64, keep=[0, 0, 0, 0])
    assert got.granted.tolist() == [1, 4, 2, 0]      # what comes back (3 + 1 + 1 + 2) counts from the next step on
    assert st.step([32, 0, 0, 0], 64, keep=[0, 0, 0, 0]).granted.tolist() == [0, 0, 0, 0]    # 8 blocks of 7
    assert st.step([32, 0, 0, 0], 64).granted.tolist() == [32, 0, 0, 0]
    assert st.step([1, 0, 0, 0], 64).granted.tolist() == [0, 0, 0, 0]        # the row is full
    assert st.step([0, 8, 1, 1], 64).granted.tolist() == [0, 8, 0, 0]        # two blocks were free


def test_garbage_state_stays_inside(dev):
    """Lengths, ranges and entries that no step leaves: every tensor's neighbours stay as they
    are, and what names no block is not given back."""
    B, W, bs, N = 5, 7, 16, 20
    pool = torch.full((4000,), 12345, dtype=I32, device=dev)
    cut = lambda at, *s: pool[at:at + torch.Size(s).numel()].view(*s)        # noqa: E731
    table, lens, free, rng = cut(100, B, W), cut(300, B), cut(400, N), cut(500, 2)
    spare = torch.ones(4000, dtype=torch.bool, device=dev)
    for at, n in ((100, B * W), (300, B), (400, N), (500, 2)):
        spare[at:at + n] = False
    bad = [-2 ** 31, -1, 0, 3, 19, 20, 2 ** 31 - 1]
    r = random.Random(3)
    for i in range(30):
        for t in (table, lens, free, rng):
            t.copy_(torch.tensor([r.choice(bad) for _ in range(t.numel())], dtype=I32).view(t.shape))
        new, keep = (torch.tensor([r.choice(bad + [5, 100]) for _ in range(B)], dtype=I32, device=dev) for _ in "ab")
        out = PT.paged_resize(table, lens, free, rng, new, 64, bs, keep=keep, window=r.choice([None, 3]))
        torch.cuda.synchronize()
        assert bool((pool[spare] == 12345).all()), i
        assert 0 <= int(rng[0]) < N and 0 <= int(rng[1]) <= N
        assert bool(((lens >= 0) & (lens <= W * bs)).all()) and int(out.cu_seqlens[-1]) <= 64


def test_slots_past_32_bits(dev):
    bs = 2 ** 24
    st = State(dev, 3000, 2, 64, bs)
    got = st.step([5, 3], 8)
    assert int(got.slots.max()) > 2 ** 31
    st.step([2 ** 25, 4], 8, keep=[bs * 0 + 5, 3])   # (does not fit the batch)


def test_captured_steps(dev):
    """A step in a graph, replayed with other requests and with eager work between the replays."""
    B, W, bs, T = 70, 20, 8, 2500
    st, r = State(dev, 900, B, W, bs, seed=4), random.Random(5)
    new, keep = (torch.zeros(B, dtype=I32, device=dev) for _ in "ab")
    args = (st.table, st.lens, st.free, st.range, new, T, bs)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        PT.paged_resize(*args, keep=keep, window=30, sinks=4)                 # nothing held: nothing changes
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = PT.paged_resize(*args, keep=keep, window=30, sinks=4)
    for i in range(6):
        n, k = [r.randint(0, 40) for _ in range(B)], [r.choice([10 ** 6, 0, 25]) for _ in range(B)]
        new.copy_(torch.tensor(n, dtype=I32)), keep.copy_(torch.tensor(k, dtype=I32))
        g.replay()
        torch.cuda.synchronize()
        st.check(out, S.resize(*st.twin, n, T, bs, k, 30, 4))
        st.step([1] * B, T, window=30, sinks=4)      # an eager step between


def test_native_path_and_wrapper_agree(dev, monkeypatch):
    t = lambda x: torch.tensor(x, dtype=I32, device=dev)                     # noqa: E731
    for kw in (dict(), dict(keep=t([0, 4, 9])), dict(keep=t([5, 5, 5]), window=8, sinks=2)):
        def run(new, T):
            state = PT.paged_pool(40, 3, 9, dev)
            PT.paged_resize(*state, t([30, 20, 10]), 100, 8)
            out = PT.paged_resize(*state, new, T, 8, **kw)
            return (*out, *state)
        _both(monkeypatch, run, t([3, 0, 20]), 40)
        _both(monkeypatch, run, t([3, 0, 20]), 0)
