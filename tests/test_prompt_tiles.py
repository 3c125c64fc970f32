"""Which rows the workgroups of paged_prompt_attn take, and where their partial results go: the
kernels' own index arithmetic (csrc/paged_prompt_tiles.h), run on the host by a wave of 64
contexts, over offsets and lengths that are some and that are none."""
import os
import random
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
NO_WINDOW = 2 ** 30


def _some(T):
    return range(0, T, T // 24 + 1)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    """Runs calls (cus, T, B, Hk, G, D, cap, window, sinks, cu, lens): for each (waves, tiles, nsplit, nwg), the row
    tiles found (b, t0, n, r0, index, first position), and some rows' (tile, row)."""
    cxx = os.environ.get("CXX") or shutil.which("g++") or "/opt/rocm/llvm/bin/clang++"
    exe = str(tmp_path_factory.mktemp("host") / "prompt_tiles")
    # -fwrapv: sums that leave 32 bits wrap, as they do on the GPU; no fortified jumps: the contexts' go from one
    # stack to another
    subprocess.run([cxx, "-O1", "-std=c++17", "-fwrapv", "-U_FORTIFY_SOURCE", os.path.join(HERE, "prompt_tiles_host.cpp"),
                    "-o", exe], check=True)

    def run(calls):
        text = "\n".join(" ".join(str(x) for x in (*c[:9], *c[9], *c[10])) for c in calls)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=300)
        assert out.returncode == 0, out
        words = iter(out.stdout.split())
        take = lambda n: tuple(int(next(words)) for _ in range(n))           # noqa: E731
        return [(take(4), [take(6) for _ in range(take(1)[0])], [take(2) for _ in _some(c[1])]) for c in calls]

    return run


def _shape(rng, B=None):
    """Rows enough for the kernel for many, most often with the keys of a tile in several parts."""
    B = B or rng.choice([1, 2, 3, 5, 17, 63, 64, 70])
    G = rng.choice([1, 4, 7, 16, 130, 300])
    T = rng.randint(1, rng.choice([40, 700, 1500]))
    return dict(cus=256, T=T, B=B, Hk=rng.choice([1, 2, 8]), G=G, D=rng.choice([64, 128]), cap=rng.choice([300, 5000, 16384, 10 ** 5]),
                window=rng.choice([NO_WINDOW, NO_WINDOW, 3000]), sinks=0)


def _check(call, result, valid):
    T, B, G, cu, lens = call[1], call[2], call[4], call[9], call[10]
    (waves, tiles, nsplit, nwg), found, rows = result
    R = 32 * waves
    for b, t0, n, r0, index, p0 in found:            # inside the rows, inside the workspace
        assert 0 <= b <= B and 0 <= t0 and 0 <= n and t0 + n <= T, (call, b, t0, n)
        assert 0 <= r0 < n * G and r0 % R == 0, (call, b, n, r0)
        assert 0 <= index < tiles, (call, tiles, index)
        if b < B:                                    # before the sequence where it is none of its positions
            assert p0 == max(lens[b] - n, -n), (call, b, p0)
    for tile, row in rows:
        assert (tile, row) == (-1, -1) or (0 <= tile < tiles and 0 <= row < R), (call, tiles, tile, row)
    if not valid:
        return
    want, first, at = [], {}, [(-1, -1)] * T
    for b in range(B + 1):
        c0, c1 = cu[b], cu[b + 1] if b < B else T
        first = len(want)
        want += [(b, c0, c1 - c0, r, first + r // R) for r in range(0, (c1 - c0) * G, R)]
        if b < B:
            at[c0:c1] = [(first + i * G // R, i * G % R) for i in range(c1 - c0)]
    assert sorted(x[:5] for x in found) == sorted(want), call
    assert rows == [at[t] for t in _some(T)], call


def _lens(rng, shape, cu):
    return [rng.choice([0, -1, -5, 2 ** 31 - 1, shape["cap"] + 9, rng.randint(0, shape["cap"])]) for _ in range(shape["B"])]


def test_rows_of_a_batch_are_taken_once(host):
    """Ascending offsets: every row tile is taken by one workgroup, in any order, and its parts are joined from where it
    left them."""
    rng = random.Random(1)
    calls = []
    for _ in range(150):
        s = _shape(rng)
        cut = sorted(rng.randint(0, s["T"]) for _ in range(s["B"]))
        cu = [0] + (cut if rng.random() < 0.5 else cut[:-1] + [s["T"]])
        calls.append((*s.values(), cu, _lens(rng, s, cu)))
    results = host(calls)
    for c, r in zip(calls, results):
        _check(c, r, True)
    plans = [r[0] for r in results]
    assert sum(w == 8 for w, *_ in plans) > 5 and sum(w == 4 for w, *_ in plans) > 20 and sum(n > 1 for _, _, n, _ in plans) > 20


def test_offsets_that_are_no_offsets_stay_inside(host):
    """Offsets that descend, overlap or leave the rows: rows of q and places of the workspace all the same."""
    rng = random.Random(2)
    calls = [(256, 1000, 5, 2, 4, 128, 16384, NO_WINDOW, 0, [0, 1000, 0, 1000, 0, 1000], [16000] * 5),
             (256, 640, 4, 2, 4, 128, 16384, NO_WINDOW, 0, [0, 640, 0, 640, 0], [700] * 4),
             (256, 640, 70, 1, 4, 128, 16384, NO_WINDOW, 0, [0, 640] * 35 + [0], [700] * 70)]
    for _ in range(150):
        s = _shape(rng)
        some = [0, s["T"], s["T"] // 2, -3, 2 ** 31 - 1, -2 ** 31]
        cu = [rng.choice(some + [rng.randint(0, s["T"])] * 3) for _ in range(s["B"] + 1)]
        if rng.random() < 0.3:
            cu = [s["T"] * (i % 2) for i in range(s["B"] + 1)]
        calls.append((*s.values(), cu, _lens(rng, s, cu)))
    results = host(calls)
    over = 0
    for c, r in zip(calls, results):
        _check(c, r, False)
        n = [max(0, min(max(y, 0), c[1]) - min(max(x, 0), c[1])) for x, y in zip(c[9], c[9][1:])]
        over += r[0][2] > 1 and sum(-(-x * c[4] // (32 * r[0][0])) for x in n) > r[0][1]
    assert over >= 10                                # more row tiles than the workspace has room for


def test_lengths_that_are_no_lengths(host):
    """Lengths down to -2^31 and up to 2^31 - 1: rows of such a sequence have no position, and the others are taken."""
    rng = random.Random(3)
    lowest = -2 ** 31
    calls = [(256, 700, 2, 8, 4, 128, 6000, NO_WINDOW, 0, [0, 20, 700], [6000, lowest]),
             (256, 700, 1, 8, 4, 128, 6000, NO_WINDOW, 0, [0, 700], [lowest])]
    for _ in range(100):
        s = _shape(rng)
        cut = sorted(rng.randint(0, s["T"]) for _ in range(s["B"]))
        lens = [rng.choice([lowest, lowest + 1, lowest + rng.randint(0, s["T"]), -1, 0, 7, 2 ** 31 - 1, s["cap"]]) for _ in range(s["B"])]
        calls.append((*s.values(), [0] + cut, lens))
    for c, r in zip(calls, host(calls)):
        _check(c, r, True)
