"""More paged-cache operators, as cases that can be timed and compared.

`op` names the operator:

  tables   a step of a batch's block tables on the GPU: tokens taken back, blocks
           given back and taken, lengths and the new tokens' slots
  append   new tokens' keys and values into an 8-bit cache with a scale for each
           block and KV head, keys (and queries) rotated by their position
  attn     attention of one new token per sequence, over such a cache or within a
           sliding window and the first tokens (sinks)
  prompt   causal attention of several new tokens per sequence over a paged cache,
           whole or within a window and the sinks

Where `own` is false, `run` computes them in elementary torch operations, else
through this package.  A cache is [blocks, KV heads, block, D]: bf16, "fp8" (e4m3
with one scale for the tensor), "e4m3" or "int8" (a scale per block and KV head,
[blocks, KV heads] fp32).  Token p of sequence b is row p % block of block
table[b, p // block]; the sequence holds lens[b] tokens, the new ones among them.
Keys and values are N(0, 1), as in every workload of this repository.
"""
import math

import torch

own = False

BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
I32, I64, I8 = torch.int32, torch.int64, torch.int8
F8_SCALE = 0.03          # an fp8 cache's one scale: N(0, 1) values then use the format's range


def listed():
    return [
        # a decode step of a batch that speculates: up to three draft tokens taken back, four more placed
        {"name": "tables_step_b32", "op": "tables", "B": 32, "L": 2000, "new": 4, "block": 16, "restart": 0, "drop": 3,
         "window": 0, "sinks": 0},
        # a large batch within a window, every eighth request ended and another's prompt in its place
        {"name": "tables_admit_b256", "op": "tables", "B": 256, "L": 6000, "new": 2000, "block": 16, "restart": 8,
         "drop": 0, "window": 1024, "sinks": 4},
        # one token each of a serving batch, two rows of it empty
        {"name": "append_e4m3_b32", "op": "append", "dtype": "e4m3", "B": 32, "Hq": 64, "Hk": 8, "D": 128, "L": 2000,
         "new": 1, "block": 16, "rot": 128, "pairs": "half", "pad": 2},
        # a chunk of four prompts of different lengths, some of whose tokens are there already
        {"name": "append_int8_prompts_b4", "op": "append", "dtype": "int8", "B": 4, "Hq": 28, "Hk": 4, "D": 128,
         "L": 3001, "new": 2048, "block": 16, "rot": 128, "pairs": "half", "pad": 0},
        # attention at the start of a chat: latency and launches count
        {"name": "attn_int8_b1_1k", "op": "attn", "dtype": "int8", "B": 1, "Hq": 14, "Hk": 2, "D": 64, "L": 1000,
         "block": 16, "window": 0, "sinks": 0, "pad": 0},
        # a large serving batch, three rows of it empty
        {"name": "attn_e4m3_b32_16k", "op": "attn", "dtype": "e4m3", "B": 32, "Hq": 64, "Hk": 8, "D": 128, "L": 16384,
         "block": 64, "window": 0, "sinks": 0, "pad": 3},
        # long chats of a model whose tokens see the latest 4096 and the first 4
        {"name": "attn_window_b16_32k", "op": "attn", "dtype": "bf16", "B": 16, "Hq": 24, "Hk": 8, "D": 128, "L": 32768,
         "block": 16, "window": 4096, "sinks": 4, "pad": 0},
        # the first prompts of a small model, a short window
        {"name": "prompt_window_b3_300", "op": "prompt", "dtype": "bf16", "B": 3, "Hq": 14, "Hk": 2, "D": 64, "L": 333,
         "new": 300, "block": 16, "window": 128, "sinks": 4},
        # a chunk of four prompts, the earlier ones in an 8-bit cache
        {"name": "prompt_e4m3_b4_3k", "op": "prompt", "dtype": "e4m3", "B": 4, "Hq": 28, "Hk": 4, "D": 128, "L": 3001,
         "new": 2048, "block": 16, "window": 0, "sinks": 0},
        # eight draft tokens of each of eight long contexts: few rows, many keys
        {"name": "prompt_drafts_b8_64k", "op": "prompt", "dtype": "bf16", "B": 8, "Hq": 24, "Hk": 8, "D": 128,
         "L": 65536, "new": 8, "block": 16, "window": 0, "sinks": 0},
        # the last quarter of a long prompt within a window
        {"name": "prompt_window_b1_32k", "op": "prompt", "dtype": "bf16", "B": 1, "Hq": 32, "Hk": 8, "D": 128,
         "L": 32768, "new": 8192, "block": 16, "window": 4096, "sinks": 4},
        # the largest: one prompt of 16K tokens, all at once
        {"name": "prompt_b1_16k", "op": "prompt", "dtype": "bf16", "B": 1, "Hq": 32, "Hk": 8, "D": 128, "L": 16384,
         "new": 16384, "block": 64, "window": 0, "sinks": 0},
    ]


# (query heads, KV heads, head dim) of the configurations, tests and harness of this repository
_HEADS = [(14, 2, 64), (28, 4, 128), (24, 8, 128), (64, 8, 128), (8, 1, 64), (32, 8, 128), (40, 2, 128), (8, 8, 64)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "prompt"])
    c = {"op": op, "block": rng.choice([8, 16, 16, 32, 64, 128, rng.randint(1, 48)])}
    if op == "tables":
        c["B"] = _log_int(rng, 1, 512)
        c["L"] = _log_int(rng, 1, 16384)
        c["restart"] = rng.choice([0, rng.randint(1, 16)])
        c["new"] = _log_int(rng, 1, max(8, 65536 // c["B"])) if c["restart"] else rng.randint(1, 8)
        c["drop"] = rng.choice([0, rng.randint(1, 7)])
        c["window"], c["sinks"] = rng.choice([(0, 0), (_log_int(rng, 1, 4096), rng.choice([0, 4, 64]))])
        return c
    c["Hq"], c["Hk"], c["D"] = Hq, Hk, D = rng.choice(_HEADS)
    if op == "append":
        c["dtype"] = rng.choice(["e4m3", "int8"])
        c["B"] = B = _log_int(rng, 1, 64)
        c["new"] = rng.choice([1, 1, _log_int(rng, 2, 32768 // B)])
        c["L"] = c["new"] + _log_int(rng, 1, 4000) - 1
        c.update(rot=rng.choice([D, D, D // 2, 32, 16, 0]), pairs=rng.choice(["half", "next"]),
                 pad=rng.randint(0, 2) if c["new"] == 1 and B > 2 else 0)
        return c
    window = (_log_int(rng, 16, 8192), rng.choice([0, 1, 4, 64]))
    if op == "attn":
        c["dtype"] = rng.choice(["e4m3", "int8", "e4m3", "int8", "bf16", "fp8"])
        c["B"] = B = _log_int(rng, 1, 64)
        c["L"] = _log_int(rng, 1, min(131072, 2 ** 28 // (B * Hk * D)))
        c["pad"] = rng.randint(0, 3) if B > 3 else 0
        c["window"], c["sinks"] = window if c["dtype"] in ("bf16", "fp8") else rng.choice([(0, 0), window])
    else:
        c["dtype"] = rng.choice(["e4m3", "int8", "bf16", "bf16", "fp8"])
        c["B"] = B = _log_int(rng, 1, 16)
        c["new"] = _log_int(rng, 2, 8192 // B)
        most = min(65536, 2 ** 28 // (B * Hk * D), 2 ** 39 // (B * c["new"] * Hq * D))     # cache and products
        c["L"] = c["new"] + _log_int(rng, 1, max(1, most - c["new"])) - 1
        c["window"], c["sinks"] = rng.choice([(0, 0), window])
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case):
    """The sequences' lengths: from L down to about L/3, hardly two alike; the last `pad` rows are empty."""
    B, L = case["B"], case["L"]
    return [max(1, L - (2 * L // 3) * b // B - 7 * b) if b < B - case.get("pad", 0) else 0 for b in range(B)]


def _news(case):
    """New tokens of each sequence, at most its length: from `new` down to about half of it."""
    return [min(n, max(1, case["new"] - (case["new"] // 2) * b // case["B"])) for b, n in enumerate(_lens(case))]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=BF16)


def _scale_of(a, dtype):
    """A block's scale for values of at most a: a / 127 for int8, the smallest power of two of at least a / 448 for e4m3."""
    if dtype == I8:
        return a / torch.full_like(a, 127.0)
    m, e = torch.frexp(a)
    k = (e - 9 + (m > 0.875).int()).clamp(min=-126)
    return torch.where(a > 0, ((k + 127) << 23).to(I32).view(F32), 0.0)


def _codes(x, s, dtype):
    """x / s rounded to the cache's type, to nearest even; beyond its range the largest value."""
    x = x / torch.where(s > 0, s, 1.0)
    return x.round().clamp(-127.0, 127.0).to(I8) if dtype == I8 else x.clamp(-448.0, 448.0).to(F8)


def _cache(g, case, N, held=None):
    """A cache's rows and what they are multiplied with; held [N]: rows of each block that are a sequence's."""
    x = _randn(g, N, case["Hk"], case["block"], case["D"])
    if case["dtype"] == "bf16":
        return x, 1.0
    if case["dtype"] == "fp8":
        return (x / F8_SCALE).to(F8), F8_SCALE
    dtype = I8 if case["dtype"] == "int8" else F8
    x = x.float()
    a = x.abs().amax(3)
    if held is not None:                           # a block's scale is that of its held rows; other blocks hold anything
        row = torch.arange(case["block"], device="cuda")
        a = a.masked_fill(((row >= held[:, None]) & (held[:, None] > 0))[:, None], 0.0)
    s = _scale_of(a.amax(2), dtype)
    return _codes(x, s[:, :, None, None], dtype), s


def _table(g, blocks, spare, more=2):
    """-> (table [B, W] of distinct blocks in random order, the order's unused rest)."""
    N = sum(blocks) + spare
    order = torch.randperm(N, generator=g, device="cuda").to(I32)
    table = torch.full((len(blocks), max(blocks) + more), -1, dtype=I32, device="cuda")
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:]


def _ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


def _prepare_tables(case, g):
    B, bs, w = case["B"], case["block"], case["window"]
    n0, more = _lens(case), max(1, case["new"])
    ends = [case["restart"] > 0 and b % case["restart"] == 0 for b in range(B)]
    keep = [0 if e else max(0, n - (b % (case["drop"] + 1))) for b, (n, e) in enumerate(zip(n0, ends))]
    new = [max(1, more - (more // 2) * b // B) if e or not case["restart"] else 1 for b, e in enumerate(ends)]
    blocks = [-(-n // bs) for n in n0]
    need = [-(-(k + m) // bs) + (-k // bs) for k, m in zip(keep, new)]
    width = max(max(blocks), max(-(-(k + m) // bs) for k, m in zip(keep, new)))
    table, rest = _table(g, blocks, sum(need) + 5, width + 2 - max(blocks))
    free = torch.full((sum(blocks) + sum(need) + 5,), -1, dtype=I32, device="cuda")
    if w:                                          # what left the window in earlier steps is in the ring already
        j = torch.arange(table.shape[1], device="cuda")
        gone = (j >= -(-case["sinks"] // bs)) & (j < (_ints(n0)[:, None] - case["drop"] - w) // bs) & (table >= 0)
        rest = torch.cat([rest, table[gone]])
        table[gone] = -1
    head = int(torch.randint(free.numel(), (1,), generator=g, device="cuda"))
    free[(head + torch.arange(rest.numel(), device="cuda")) % free.numel()] = rest
    return {"case": case, "table": table, "lens": _ints(n0), "free": free, "range": _ints([head, rest.numel()]),
            "keep": _ints(keep), "new": _ints(new), "tokens": -(-sum(new) // 64) * 64}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    if case["op"] == "tables":
        return _prepare_tables(case, g)
    B, Hq, Hk, D, bs = (case[n] for n in ("B", "Hq", "Hk", "D", "block"))
    lens = _lens(case)
    table, rest = _table(g, [-(-n // bs) for n in lens], 3)
    N = int((table >= 0).sum()) + rest.numel()
    x = {"case": case, "table": table, "lens": _ints(lens), "scale": 1.0 / math.sqrt(D)}
    new = _news(case) if "new" in case else []
    if case.get("new", 1) > 1:
        x["cu"] = _ints([0] + new).cumsum(0).to(I32)
    held = None
    if case["op"] == "append":
        x.setdefault("cu", None)
        old = _ints([n - m if n else 0 for n, m in zip(lens, new)])
        held = torch.zeros(N, dtype=I64, device="cuda")
        held[table[table >= 0].long()] = (old[:, None] - bs * torch.arange(table.shape[1], device="cuda")).clamp(
            0, bs)[table >= 0].long()
        qkv = _randn(g, sum(new) if x["cu"] is not None else B, Hq + 2 * Hk, D)      # the projection's output
        x["nq"], x["nk"], x["nv"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
        x["cos"] = x["sin"] = None
        if case["rot"]:
            freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=F64) / case["rot"])
            angle = torch.arange(table.shape[1] * bs, device="cuda", dtype=F64)[:, None] * freq
            x["cos"], x["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attn":
        x["q"] = _randn(g, B, Hq, 1, D)
    else:
        x["q"] = _randn(g, sum(new), Hq, D)
    (x["k"], x["ks"]), (x["v"], x["vs"]) = _cache(g, case, N, held), _cache(g, case, N, held)
    return x


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_tables(x):
    case, table, lens, free, ring = x["case"], x["table"], x["lens"], x["free"], x["range"]
    bs, w, T, (B, W), N = case["block"], case["window"], x["tokens"], table.shape, free.numel()
    j = torch.arange(W, device="cuda")
    n0 = lens.clamp(0, W * bs)
    kept = torch.minimum(n0, x["keep"].clamp(min=0))
    first, last = -(-kept // bs), -(-n0 // bs)
    named = (table >= 0) & (table < N)
    back = (j >= first[:, None]) & (j < last[:, None]) & named
    if w:                                          # from the window's edge down to the first place without a block
        out = (j >= -(-case["sinks"] // bs)) & (j < ((kept - w + 1) // bs)[:, None])
        back |= out & ((out & ~named).flip(1).cumsum(1).flip(1) == 0)
    room = (x["new"] > 0) & (x["new"] <= W * bs - kept)
    m = torch.where(room, x["new"], 0)
    need = -(-(kept + m) // bs) - first
    head, count = ring[0].clone(), ring[1].clone()
    taken = need.cumsum(0)
    ok = ((need == 0) | (taken <= count)) & (m.cumsum(0) <= T)
    granted = torch.where(ok, m, 0).to(I32)
    need = torch.where(ok, need, 0)
    start = need.cumsum(0) - need                  # a sequence's first block in the ring
    given = table[back]
    free[(head + count + torch.arange(given.numel(), device="cuda")) % N] = given
    table[back] = -1
    k = j - first[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    table.copy_(torch.where(fresh, free[(head + start[:, None] + k.clamp(min=0)) % N], table))
    lens.copy_(kept + granted)
    ring.copy_(torch.stack([(head + need.sum()) % N, count - need.sum() + given.numel()]))
    cu = torch.cat([granted.new_zeros(1), granted.cumsum(0)]).to(I32)
    t = torch.arange(T, device="cuda", dtype=I32)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    live = t < cu[-1]
    b = seq.clamp(max=B - 1)
    p = kept[b] + t - cu[b]
    ids = table[b, (p // bs).clamp(0, W - 1)].long()
    slot = torch.where(live & (ids >= 0) & (ids < N), ids * bs + p % bs, -1)
    return {"table": table, "lens": lens, "free": free, "range": ring, "cu": cu, "granted": granted,
            "seqs": torch.where(live, seq, -1).to(I32), "positions": torch.where(live, p, -1).to(I32), "slots": slot}


def _rotate(x, cos, sin, pairs):
    """x [T, H, D] with its first dims rotated by each row's cos, sin [T, R/2]."""
    if cos is None:
        return x
    R = 2 * cos.shape[1]
    r, rest = x[..., :R], x[..., R:]
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    if pairs == "half":
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([r, rest], -1)


def _held_values(x):
    """The cache as the values it stands for, where its numbers are whole ones."""
    out = {"k": x["k"], "v": x["v"], "ks": x["ks"], "vs": x["vs"]}
    if x["case"]["dtype"] == "int8":
        out["k"], out["v"] = ((c * s[:, :, None, None]).to(BF16) for c, s in ((x["k"], x["ks"]), (x["v"], x["vs"])))
    return out


def _plain_append(x):
    case, table, lens, dtype = x["case"], x["table"], x["lens"], x["k"].dtype
    T, bs, N = x["nk"].shape[0], case["block"], x["k"].shape[0]
    raw = torch.uint8 if dtype == F8 else I8
    t = torch.arange(T, device="cuda")
    if x["cu"] is None:
        b, p = t, lens - 1
    else:
        b = torch.searchsorted(x["cu"][1:].contiguous(), t.to(I32), right=True)
        p = lens[b] - x["cu"][b + 1] + t
    valid = p >= 0
    at = p.clamp(min=0).long()
    cos, sin = (None, None) if x["cos"] is None else (x["cos"][at], x["sin"][at])
    q = (_rotate(x["nq"].float(), cos, sin, case["pairs"]) * valid[:, None, None]).to(BF16)
    # keys from 64 bits: a scale and a code next to a border of two go by their last bits
    rows = {"k": _rotate(x["nk"].double(), cos, sin, case["pairs"]).float(), "v": x["nv"].float()}
    src = torch.where(valid, t, valid.int().argmax())            # an empty row writes the first full row's values again
    ids, off = table[b[src], at[src] // bs].long(), at[src] % bs
    off0 = torch.full((N,), bs, device="cuda").index_reduce_(0, ids, off, "amin")     # a block's first new row
    row = torch.arange(bs, device="cuda")
    out = {"q": q}
    for n, sn in (("k", "ks"), ("v", "vs")):
        new, cache, s = rows[n][src], x[n], x[sn]
        a = torch.zeros_like(s).index_reduce_(0, ids, new.abs().amax(-1), "amax")
        was = torch.where((off0 == 0)[:, None], 0.0, s)
        now = torch.where((off0 < bs)[:, None], torch.maximum(was, _scale_of(a, dtype)), s)
        ratio = torch.where(now > 0, was / torch.where(now > 0, now, 1.0), 0.0)
        grown = ((now > was) & (off0 > 0)[:, None])[ids][..., None, None] & (row < off0[ids][:, None])[:, None, :, None]
        old = cache.view(raw)[ids].view(dtype)
        again = _codes(old.float() * ratio[ids][..., None, None], torch.ones((), device="cuda"), dtype)
        cache.view(raw)[ids] = torch.where(grown, again.view(raw), old.view(raw))
        s.copy_(now)
        cache.view(raw)[ids, :, off] = _codes(new, now[ids][..., None], dtype).view(raw)
    return {**out, **_held_values(x)}


def _rows(x, n, ids, off):
    """Rows `off` of the blocks `ids` of cache n, as fp32 values: [*ids.shape, KV heads, D]."""
    c, s = x[n], x[n + "s"]
    raw = torch.uint8 if c.dtype == F8 else c.dtype
    r = c.view(raw)[ids, :, off].view(c.dtype).float()
    return r * (s[ids][..., None] if torch.is_tensor(s) else s)


def _softmax_av(s, mask, v):
    s = s.masked_fill(~mask, -float("inf"))
    m = s.amax(-1, keepdim=True)
    e = s.sub_(m.masked_fill(m == -float("inf"), 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    return e @ v / total.masked_fill(total == 0, 1.0)


def _plain_attn(x):
    case, n, w, sinks = x["case"], x["lens"][:, None], x["case"]["window"], x["case"]["sinks"]
    B, Hq, Hk, D, bs = (case[c] for c in ("B", "Hq", "Hk", "D", "block"))
    cap = x["table"].shape[1] * bs
    if w and w + sinks < cap:                      # the tokens that can take part, the sinks first
        i = torch.arange(sinks + w, device="cuda")
        t = torch.where(i < sinks, i, n - w + i - sinks)
        mask = (t < n) & (t >= torch.where(i < sinks, 0, sinks))
    else:
        t = torch.arange(cap, device="cuda").expand(B, cap)
        mask = (t < n) & ((t >= n - w) | (t < sinks)) if w else t < n
    at = t.clamp(0, cap - 1).long()
    ids = x["table"].gather(1, at // bs).long()
    mask = (mask & (ids >= 0))[:, None, None]
    ids, off = ids.clamp(min=0), at % bs
    k = _rows(x, "k", ids, off).permute(0, 2, 3, 1)
    s = x["q"].float().reshape(B, Hk, Hq // Hk, D) @ k * x["scale"]
    del k
    o = _softmax_av(s, mask, _rows(x, "v", ids, off).transpose(1, 2))
    return o.reshape(B, Hq, 1, D).to(BF16)


def _plain_prompt(x):
    case, w = x["case"], x["case"]["window"]
    Hq, Hk, D, bs = (case[c] for c in ("Hq", "Hk", "D", "block"))
    new, G = max(_news(case)), Hq // Hk
    cu, lens, table = x["cu"].long(), x["lens"][:, None], x["table"]
    B, cap = table.shape[0], table.shape[1] * bs
    i = torch.arange(new, device="cuda")
    n = (cu[1:] - cu[:-1])[:, None]
    live, row = i < n, (cu[:-1, None] + i).clamp(max=x["q"].shape[0] - 1)
    p = (lens - n + i)[:, :, None]                 # the queries' positions [B, new, 1]
    t = torch.arange(cap, device="cuda")
    seen = t <= p
    if w:
        seen &= (t > p - w) | (t < case["sinks"])
    seen &= ((table >= 0).repeat_interleave(bs, 1) & (t < lens))[:, None]
    ids = table.clamp(min=0).long().repeat_interleave(bs, 1)
    off = (t % bs).expand(B, cap)
    q = x["q"][row].float().reshape(B, new, Hk, G, D)
    o = torch.empty(B, new, Hk, G, D, device="cuda")
    k, v = _rows(x, "k", ids, off), _rows(x, "v", ids, off)
    for h in range(Hk):                            # a KV head at a time: the scores of all would not fit the card
        s = q[:, :, h].transpose(1, 2) @ k[:, None, :, h].transpose(2, 3) * x["scale"]
        o[:, :, h] = _softmax_av(s, seen[:, None], v[:, None, :, h]).transpose(1, 2)
    out = torch.zeros_like(x["q"])
    out[row[live]] = o[live].reshape(-1, Hq, D).to(BF16)
    return out


# ---------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------
def _own(x):
    from bytes_amd import paged as PG
    case = x["case"]
    if case["op"] == "tables":
        from bytes_amd import paged_tables as PT
        r = PT.paged_resize(x["table"], x["lens"], x["free"], x["range"], x["new"], x["tokens"], case["block"],
                            keep=x["keep"], window=case["window"] or None, sinks=case["sinks"])
        return {"table": x["table"], "lens": x["lens"], "free": x["free"], "range": x["range"], "cu": r.cu_seqlens,
                "granted": r.granted, "seqs": r.seqs, "positions": r.positions, "slots": r.slots}
    if case["op"] == "append":
        q = PG.paged_kv_append(x["nk"], x["nv"], x["k"], x["v"], x["table"], x["lens"], cu_seqlens=x["cu"], q=x["nq"],
                               cos=x["cos"], sin=x["sin"], interleaved=case["pairs"] == "next", k_scale=x["ks"],
                               v_scale=x["vs"])
        return {"q": q, **_held_values(x)}
    if case["op"] == "attn":
        return PG.paged_decode_attn(x["q"], x["k"], x["v"], x["table"], x["lens"], x["scale"], k_scale=x["ks"],
                                    v_scale=x["vs"], window=case["window"] or None, sinks=case["sinks"])
    return PG.paged_prompt_attn(x["q"], x["k"], x["v"], x["table"], x["lens"], x["cu"], x["scale"], k_scale=x["ks"],
                                v_scale=x["vs"], window=case["window"] or None, sinks=case["sinks"])


def run(x):
    if own:
        return _own(x)
    return {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn, "prompt": _plain_prompt}[
        x["case"]["op"]](x)


def _seen(n, w, sinks, p):
    """Tokens that position p of a sequence of n sees."""
    return p + 1 if not w else min(p + 1, w) + min(sinks, max(0, p + 1 - w))


def work(case):
    B, bs, lens = case["B"], case["block"], _lens(case)
    if case["op"] == "tables":
        restart, more = case["restart"], max(1, case["new"])
        ends = [restart > 0 and b % restart == 0 for b in range(B)]
        T = sum(max(1, more - (more // 2) * b // B) if e or not restart else 1 for b, e in enumerate(ends))
        moved = sum(-(-n // bs) for n, e in zip(lens, ends) if e) + T // bs
        return {"bytes": 24 * B + 16 * T + 8 * moved, "flops": 8 * B + 4 * T}
    Hq, Hk, D = (case[n] for n in ("Hq", "Hk", "D"))
    es, scaled = 2 if case["dtype"] == "bf16" else 1, case["dtype"] in ("e4m3", "int8")
    if case["op"] == "append":
        new = [n for n, m in zip(_news(case), lens) if m]
        T = sum(new)
        touched = sum(-(-m // bs) - (m - n) // bs for n, m in zip(new, [m for m in lens if m]))
        b = T * (Hq + 2 * Hk) * D * 2 + T * Hq * D * 2 + T * 2 * Hk * D + T * case["rot"] * 4 + touched * Hk * 16
        return {"bytes": b, "flops": 3 * T * (Hq + Hk) * case["rot"] + 4 * T * Hk * D}
    w, sinks = case["window"], case["sinks"]
    if case["op"] == "attn":
        seen, queries = sum(_seen(n, w, sinks, n - 1) for n in lens if n), B
        pairs, held = seen, seen
    else:
        new = _news(case)
        queries = sum(new)
        pairs = sum(_seen(n, w, sinks, p) for n, m in zip(lens, new) for p in range(n - m, n))
        # rows that some query sees: the first one's window, and all after it
        held = sum(min(n, _seen(n, w, sinks, n - m) + m - 1) for n, m in zip(lens, new))
    return {"bytes": 2 * held * Hk * D * es + 2 * queries * Hq * D * 2 + (held // bs * Hk * 8 if scaled else 0),
            "flops": 4 * pairs * Hq * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, one sequence at a time
# ---------------------------------------------------------------------------
def _exact_append(x, case):
    lens, new, bs, R = _lens(case), _news(case), case["block"], case["rot"]
    int8 = case["dtype"] == "int8"
    table = x["table"].tolist()
    q = torch.zeros(x["nq"].shape, dtype=F64, device="cuda")
    scales = {"k": x["ks"].double(), "v": x["vs"].double()}
    held = {n: x[n].double() * scales[n][:, :, None, None] for n in ("k", "v")}      # as the values they stand for

    def turned(rows, p):                           # [n, H, D] at positions p
        out = rows.double().clone()
        if R:
            c, s = x["cos"].double()[p][:, None], x["sin"].double()[p][:, None]
            i = torch.arange(R // 2, device="cuda")
            lo, hi = (i, i + R // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
            a, b = out[..., lo].clone(), out[..., hi].clone()
            out[..., lo], out[..., hi] = a * c - b * s, a * s + b * c
        return out

    def fitting(a):
        return a / 127 if int8 else torch.pow(torch.full_like(a, 2.0), torch.ceil(torch.log2(a / 448)))

    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        if m:
            rows = slice(at, at + n)
            p = torch.arange(m - n, m, device="cuda")
            q[rows] = turned(x["nq"][rows], p)
            y = {"k": turned(x["nk"][rows], p), "v": x["nv"][rows].double()}
            i = 0
            while i < n:                           # the new tokens of one page
                o = (m - n + i) % bs
                e = min(n, i + bs - o)
                page = table[b][(m - n + i) // bs]
                for c in ("k", "v"):
                    r = y[c][i:e].transpose(0, 1)
                    fit = fitting(r.abs().amax((1, 2)))
                    now = fit if o == 0 else torch.maximum(fit, scales[c][page])
                    if int8:                       # values between two whole multiples are not what the type holds
                        step = now[:, None, None]
                        r = (r / step).round() * step
                        held[c][page, :, :o] = (held[c][page, :, :o] / step).round() * step
                    held[c][page, :, o:o + e - i] = r
                    # rows past the new ones keep their codes: no tokens, but they come back
                    held[c][page, :, o + e - i:] = x[c][page, :, o + e - i:].double() * now[:, None, None]
                    scales[c][page] = now
                i = e
        at += n if case["new"] > 1 else 1
    if not int8:                                   # e4m3 rows come back as they are held, in units of their scale
        held = {c: held[c] / scales[c][:, :, None, None] for c in held}
    return {"q": q, "k": held["k"], "v": held["v"], "ks": scales["k"], "vs": scales["v"]}


def _exact_attn(x, case, new):
    """Attention of the last new[b] positions of each sequence, 512 of them at a time: [sum(new), Hq, D]."""
    Hq, Hk, D, bs, w = (case[n] for n in ("Hq", "Hk", "D", "block", "window"))
    G, raw = Hq // Hk, torch.uint8 if x["k"].dtype == F8 else x["k"].dtype
    q = x["q"].reshape(-1, Hq, D)
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(_lens(case), new)):
        ids = x["table"][b, :-(-n // bs)].long()
        t = torch.arange(n, device="cuda")
        for h in range(Hk if n else 0):
            k, v = (x[c][:, h].view(raw)[ids].view(x["k"].dtype).double() for c in ("k", "v"))
            for c, s in ((k, x["ks"]), (v, x["vs"])):
                c *= s[ids, h].double()[:, None, None] if torch.is_tensor(s) else s
            k, v = k.reshape(-1, D)[:n], v.reshape(-1, D)[:n]
            for i in range(0, m, 512):
                e = min(m, i + 512)
                p = torch.arange(n - m + i, n - m + e, device="cuda")[:, None]
                away = t > p
                if w:
                    away |= (t <= p - w) & (t >= case["sinks"])
                y = q[at + i:at + e, h * G:(h + 1) * G].double().reshape(-1, D)
                s = (torch.matmul(y, k.t()) * x["scale"]).reshape(e - i, G, n)
                s = torch.softmax(s.masked_fill(away[:, None], -float("inf")), -1)
                out[at + i:at + e, h * G:(h + 1) * G] = torch.matmul(s, v)
        at += m
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None                                # whole numbers: equal or not
    x = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(x, case)
    if case["op"] == "attn":
        return _exact_attn(x, case, [1] * case["B"]).reshape(case["B"], case["Hq"], 1, case["D"])
    return _exact_attn(x, case, _news(case))
