"""Block tables, block-scaled appends and attention within a window from their
definitions, on the CPU and in 64 bits, for the tests: loops over sequences, tokens and
blocks."""
import math

import torch

import paged_oracle as O

F8 = torch.float8_e4m3fn
BF16_MAX = 3.3895313892515355e38


# ---------------------------------------------------------------------------
# tables
# ---------------------------------------------------------------------------
def resize(table, lens, ring, rng, new, T, bs, keep=None, window=0, sinks=0):
    """One step on lists: table [B][W], lens [B], ring [N], rng [head, count]; changes
    them in place and returns (cu, granted, seqs, positions, slots)."""
    B, W, N = len(table), len(table[0]), len(ring)
    head, count = rng
    names = lambda i: 0 <= i < N                                            # noqa: E731
    given, kept = [], []
    for b in range(B):
        n0 = min(max(lens[b], 0), W * bs)
        k = n0 if keep is None else min(n0, max(keep[b], 0))
        kept.append(k)
        back = []
        if window:
            j = max(k - window + 1, 0) // bs - 1
            while j >= -(-sinks // bs) and names(table[b][j]):
                back.insert(0, j)
                j -= 1
        back += [j for j in range(-(-k // bs), -(-n0 // bs)) if names(table[b][j])]
        for j in back:
            given.append(table[b][j])
            table[b][j] = -1
    taken = asked_blocks = asked_tokens = 0
    granted, cu = [], [0]
    rows = []
    for b in range(B):
        m = new[b] if 0 < new[b] <= W * bs - kept[b] else 0
        first = -(-kept[b] // bs)
        need = -(-(kept[b] + m) // bs) - first
        asked_blocks, asked_tokens = asked_blocks + need, asked_tokens + m
        if (need and asked_blocks > count) or asked_tokens > T:
            m = need = 0
        for j in range(first, first + need):
            table[b][j] = ring[(head + taken) % N]
            taken += 1
        granted.append(m)
        cu.append(cu[-1] + m)
        for p in range(kept[b], kept[b] + m):
            i = table[b][p // bs]
            rows.append((b, p, i * bs + p % bs if names(i) else -1))
        lens[b] = kept[b] + m
    for i, x in enumerate(given):
        ring[(head + count + i) % N] = x
    rng[0], rng[1] = (head + taken) % N, count - taken + len(given)
    rows += [(-1, -1, -1)] * (T - len(rows))
    return cu, granted, [r[0] for r in rows], [r[1] for r in rows], [r[2] for r in rows]


# ---------------------------------------------------------------------------
# appends into caches with a scale for each block and head
# ---------------------------------------------------------------------------
def fitting(a, int8):
    """The scale of values of at most a (a float)."""
    if int8:
        return a / 127
    if a == 0:
        return 0.0
    m, e = math.frexp(a)                             # a = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return 2.0 ** max(e - 9 + (m > 0.875), -126)


def block_rows(T, table, lens, cu, bs, N):
    """{(block, first new row): [(row of the block, token row, sequence, position)]} of the new tokens."""
    out = {}
    for t, b, p in O.placed(T, table, lens, cu, bs):
        i = int(table[b, p // bs])
        if 0 <= i < N:
            out.setdefault(i, []).append((p % bs, t, b, p))
    return out


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def values(c, s):
    """Cache rows as the fp64 values they stand for: s a number, or [N, Hk]."""
    return c.double() * (s.double()[:, :, None, None] if torch.is_tensor(s) else s)


def attend_rows(q, rows, kc, vc, scale, ks, vs, table, lens, window=None, sinks=0):
    """Attention of single rows: q [R, Hq, D]; rows: (sequence, position) of each, or None
    for one without (zeros).  -> out, the weighted sum of |v|, and the largest sum
    of |q k| * scale, fp64 (as paged_oracle.attend)."""
    N, Hk, bs, D = kc.shape
    R, Hq = q.shape[:2]
    kv, vv = values(kc, ks), values(vc, vs)
    out = torch.zeros(R, Hq, D, dtype=torch.float64)
    mag, dots = torch.zeros_like(out), torch.zeros(R, Hq, 1, dtype=torch.float64)
    held = {}
    for r, at in enumerate(rows):
        if at is None:
            continue
        b, p = at
        if b not in held:
            toks = O.held_tokens(table, lens, N, bs, b)
            held[b] = torch.tensor([t for t in toks], dtype=torch.int64).reshape(-1, 3)
        toks = held[b]
        see = toks[:, 0] <= p
        if window is not None:
            see &= (toks[:, 0] > p - window) | (toks[:, 0] < sinks)
        toks = toks[see]
        if not len(toks):
            continue
        ids, off = toks[:, 1], toks[:, 2]
        k = kv[ids, :, off].repeat_interleave(Hq // Hk, 1)                   # [n, Hq, D]
        v = vv[ids, :, off].repeat_interleave(Hq // Hk, 1)
        x = q[r].double()
        s = (k * x).sum(-1) * scale
        w = torch.softmax(s, 0)
        out[r] = (w[..., None] * v).sum(0)
        mag[r] = (w[..., None] * v.abs()).sum(0)
        dots[r, :, 0] = ((k * x).abs().sum(-1) * abs(scale)).amax(0)
    return out, mag, dots


def positions(T, table, lens, cu, bs):
    """(sequence, position) of every token row, None without one."""
    out = [None] * T
    for t, b, p in O.placed(T, table, lens, cu, bs):
        out[t] = (b, p)
    return out
