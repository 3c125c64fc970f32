"""The paged-cache operators from their formulas in 64 bits, on the CPU, for the
tests: loops over sequences, tokens and blocks."""
import torch

F8 = torch.float8_e4m3fn


def capacity(table, bs):
    return table.shape[1] * bs


def held_tokens(table, lens, N, bs, b):
    """(position, block, row) of the tokens of sequence b that take part."""
    n = max(0, min(int(lens[b]), capacity(table, bs)))
    row = table[b].tolist()
    return [(p, row[p // bs], p % bs) for p in range(n) if 0 <= row[p // bs] < N]


def rotate(x, cos, sin, p, interleaved):
    """x [H, D] fp64 at position p; also the sum of the products' magnitudes."""
    if cos is None:
        return x.clone(), x.abs()
    R = 2 * cos.shape[1]
    i = torch.arange(R // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    c, s = cos[p].double(), sin[p].double()
    y, mag = x.clone(), x.abs()
    y[:, lo], y[:, hi] = x[:, lo] * c - x[:, hi] * s, x[:, hi] * c + x[:, lo] * s
    mag[:, lo], mag[:, hi] = (x[:, lo] * c).abs() + (x[:, hi] * s).abs(), (x[:, hi] * c).abs() + (x[:, lo] * s).abs()
    return y, mag


def placed(T, table, lens, cu, bs):
    """(token row, sequence, position) of every new token that has a position."""
    B = table.shape[0]
    ends = list(range(B + 1)) if cu is None else cu.tolist()
    out = []
    for b in range(B):
        for t in range(ends[b], min(ends[b + 1], T)):
            p = int(lens[b]) - (ends[b + 1] - t)
            if 0 <= p < capacity(table, bs):
                out.append((t, b, p))
    return out


def attend(q, k, v, scale, k_scale, v_scale, table, lens, picks=None):
    """out [B, Hq, D] fp64 and, per element, the weighted sum of |v| and the largest
    sum of |q k| * scale: what the kernels' roundings are relative to.  picks: a
    set of table places per (b, h), or None."""
    N, Hk, bs, D = k.shape
    B, Hq = q.shape[:2]
    G = Hq // Hk
    qd, kd, vd = q.double().reshape(B, Hq, D), k.double(), v.double()
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    mag, dots = torch.zeros_like(out), torch.zeros(B, Hq, 1, dtype=torch.float64)
    for b in range(B):
        toks = held_tokens(table, lens, N, bs, b)
        for h in range(Hq):
            mine = [t for t in toks if picks is None or t[0] // bs in picks[b][h]]
            if not mine:
                continue
            ids, off = torch.tensor([t[1] for t in mine]), torch.tensor([t[2] for t in mine])
            kk, vv = kd[ids, h // G, off], vd[ids, h // G, off]
            s = kk @ qd[b, h] * (scale * k_scale)
            p = torch.softmax(s, 0)
            out[b, h] = p @ vv * v_scale
            mag[b, h] = p @ vv.abs() * v_scale
            dots[b, h, 0] = ((kk.abs() @ qd[b, h].abs()) * abs(scale * k_scale)).max()
    return out, mag, dots


def bounds(q, kmin, kmax, table, lens, bs, scale, local_w):
    """fp64 bounds [B, Hq, W] (before the rounding to fp32) and sums of magnitudes."""
    N, Hk, D = kmin.shape
    B, Hq = q.shape[:2]
    G, W = Hq // Hk, table.shape[1]
    qd = q.double().reshape(B, Hq, D)
    out = torch.full((B, Hq, W), -float("inf"), dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = max(0, min(int(lens[b]), W * bs))
        for j in range(W):
            i = int(table[b, j])
            if j * bs >= n or not 0 <= i < N:
                continue
            if local_w and j >= max(0, n - local_w) // bs:
                out[b, :, j] = float("inf")
                continue
            for h in range(Hq):
                t = qd[b, h] * torch.where(qd[b, h] >= 0, kmax[i, h // G].double(), kmin[i, h // G].double())
                out[b, h, j], mag[b, h, j] = t.sum() * scale, t.abs().sum() * abs(scale)
    return out, mag
