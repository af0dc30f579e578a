"""Attention over the 8-bit cache on each of its paths, named: lists of 16 and 32 columns with up to 64 rows and with more, in equal
shares and in proportion, joins of more parts than a wave takes at once, the form without a list, prompts split and whole."""
import math

import pytest
import torch

import kv8_reference as ref
from kv8_plan import entries, plan
from test_gpu_kv8 import DEV, kv8, rows

pytestmark = pytest.mark.gpu


def want_of(data, exps, q, bt, lens, qsl, window=0):
    """(outputs, how far a kernel's may be) as kv8_reference.attend, a row's tokens and heads at once."""
    K, V = ref.values(data, exps)
    P, H, bs, D = K.shape
    T, Hq = q.shape[:2]
    G, scale = Hq // H, 1 / math.sqrt(D)
    out, far = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    for r in range(len(lens)):
        a, b, N = int(qsl[r]), int(qsl[r + 1]), int(lens[r])
        if a == b:
            continue
        pos = torch.arange(N)
        page = bt[r].long()[pos // bs]
        qp = N - (b - a) + torch.arange(b - a)
        see = (pos[None] <= qp[:, None]) & (pos[None] > qp[:, None] - (window or N + 1))
        for h in range(H):
            k, v = K[page, h, pos % bs], V[page, h, pos % bs]
            x = q[a:b, h * G:(h + 1) * G].double()
            s = (x.reshape(-1, D) @ k.T).view(b - a, G, N) * scale
            p = torch.softmax(s.masked_fill(~see[:, None], -math.inf), -1).reshape(-1, N)
            ds = scale * 2 ** -20 * (x.abs().reshape(-1, D) @ k.abs().T).view(b - a, G, N).masked_fill(~see[:, None], 0).amax(-1, keepdim=True)
            o = (p @ v).view(b - a, G, D)
            out[a:b, h * G:(h + 1) * G] = o
            far[a:b, h * G:(h + 1) * G] = (2 ** -8 + 2 * ds) * (p @ v.abs()).view(b - a, G, D) + 2 ** -8 * o.abs() + 1e-30
    return out, far


def some(seed, R, lo, hi, least, most, longest=()):
    g = torch.Generator().manual_seed(seed)
    prev = torch.randint(lo, hi + 1, (R,), generator=g).tolist()
    for r, n in longest:
        prev[r] = n
    return prev, torch.randint(least, most + 1, (R,), generator=g).tolist()


# name: (rows, query heads, KV heads, D, page tokens, window, kind, columns, in proportion)
PATHS = {
    "list 16, shares": (some(1, 30, 0, 1500, 0, 2, [(7, 2000)]), 8, 2, 64, 64, 0, "LISTED", 16, False),
    "list 16, proportion": (some(2, 40, 2000, 5000, 0, 3), 8, 2, 128, 64, 0, "LISTED", 16, True),
    "list 16, proportion, window": (some(2, 60, 4000, 9000, 1, 3), 4, 2, 64, 64, 3000, "LISTED", 16, True),
    "list 16, over 64 rows": (some(3, 300, 0, 150, 0, 3, [(7, 1500), (250, 1200)]), 2, 1, 64, 64, 0, "LISTED", 16, False),
    "list 16, over 64 rows, proportion": (some(4, 70, 1500, 3100, 0, 3), 8, 2, 64, 128, 0, "LISTED", 16, True),
    "list 32, shares": (some(5, 64, 0, 260, 5, 9, [(3, 1200)]), 32, 8, 64, 64, 0, "LISTED", 32, False),
    "list 32, proportion": (some(6, 40, 500, 1500, 4, 8, [(11, 1650)]), 32, 8, 64, 64, 0, "LISTED", 32, True),
    "list 32, over 64 rows, proportion": (some(7, 70, 400, 900, 4, 9, [(0, 1300)]), 32, 8, 64, 64, 0, "LISTED", 32, True),
    "list 32, three heads": (some(8, 90, 300, 1200, 5, 12, [(89, 1900)]), 24, 8, 64, 64, 0, "LISTED", 32, True),
    "direct": (some(9, 20, 0, 900, 0, 3), 8, 2, 64, 64, 0, "DIRECT", 16, None),
    "direct, many long rows": (some(10, 70, 0, 2500, 0, 1, [(5, 4000)]), 8, 2, 64, 64, 0, "DIRECT", 16, None),
    "prompt": (some(11, 40, 0, 300, 60, 200), 32, 8, 64, 64, 0, "PROMPT", 128, False),
    "prompt, split": (some(12, 3, 1000, 3000, 30, 90), 8, 2, 64, 64, 0, "PROMPT", 128, True),
}


@pytest.mark.parametrize("name", PATHS)
def test_paths(kv8, name):
    (prev, new), heads, kv, D, bs, window, kind, cols, more = PATHS[name]
    data, exps, bt, lens, qsl, T, g = rows(kv8, len(name), prev, new, kv, D, bs, pad=3)
    p = plan(kv, bs // 64, D, heads, len(prev), T, bt.shape[1], window)
    assert p[:2] == (kind, cols)
    if kind == "LISTED":
        assert (entries(kind, cols, kv, heads, bs, prev, new, window) > 4 * p[2]) == more, (p, entries(kind, cols, kv, heads, bs, prev, new, window))
    elif kind == "PROMPT":
        assert (p[2] > 1) == more
    q = (torch.randn(T, heads, D, generator=g) * 2).to(torch.bfloat16)
    got = kv8.attend(kv8.Cache8(data.to(DEV), exps.to(DEV)), q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV), window=window).cpu().double()
    want, far = want_of(data, exps, q, bt, lens, qsl, window)
    worst = float(((got - want).abs() / far.clamp(min=1e-30)).max())
    print(name, p, "worst error over its bound", round(worst, 3), flush=True)
    assert worst <= 1.0 and not got[int(qsl[-1]):].any()


# one row on one KV head (or two), so that an item has more than the 64 parts that a join takes at once
@pytest.mark.parametrize("kv,heads,n,new,kind,cols", [(1, 4, 40000, 3, "LISTED", 16), (2, 18, 262144, 2, "LISTED", 32), (1, 4, 40000, 20, "PROMPT", 128)], ids=str)
def test_joins_of_many_parts(kv8, kv, heads, n, new, kind, cols):
    data, exps, bt, lens, qsl, T, g = rows(kv8, 71, [n - new], [new], kv, 64, 256)
    p = plan(kv, 4, 64, heads, 1, T, bt.shape[1])
    assert p[:2] == (kind, cols)
    tiles = 1 if kind == "PROMPT" else -(-new // (cols // (heads // kv)))
    parts = p[2] if kind == "PROMPT" else p[2] // (kv * tiles)
    assert parts > 64
    q = (torch.randn(T, heads, 64, generator=g) * 2).to(torch.bfloat16)
    got = kv8.attend(kv8.Cache8(data.to(DEV), exps.to(DEV)), q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV)).cpu().double()
    want, far = want_of(data, exps, q, bt, lens, qsl)
    worst = float(((got - want).abs() / far).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("R,pad,n,kind,cols", [(71, 80, 1500, "LISTED", 16), (30, 31, 1500, "LISTED", 16), (71, 3, 1500, "DIRECT", 16), (3, 200, 3000, "PROMPT", 128),
                                               (150, 1400, 3000, "LISTED", 32)], ids=str)
def test_steps_of_padding_by_path(kv8, R, pad, n, kind, cols):
    """Rows that all bring nothing, in room for some tokens."""
    prev = [100] * (R - 1) + [n]
    data, exps, bt, lens, qsl, T, g = rows(kv8, 23, prev, [0] * R, 2, 64, 64, pad=pad)
    assert plan(2, 1, 64, 4, R, T, bt.shape[1])[:2] == (kind, cols)
    q = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16)
    assert not kv8.attend(kv8.Cache8(data.to(DEV), exps.to(DEV)), q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV)).any()
