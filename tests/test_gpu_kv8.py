"""The paged 8-bit cache on the GPU against plain 64-bit forms: bytes after an append, values read back, attention."""
import math

import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def kv8(hip):
    import lfm3_kv800_amd.kv8 as m
    return m


def rows(kv8, seed, prev, new, H, D, bs, spare=2, pad=0, cols=0):
    """A cache with random codes, tables of shuffled pages, lengths and starts of rows with prev + new positions."""
    g = torch.Generator().manual_seed(seed)
    last = [p + c for p, c in zip(prev, new)]
    need = [-(-x // bs) for x in last]
    width = max(need + [1]) + cols
    perm = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    bt, at = torch.full((len(prev), width), -1, dtype=torch.int32), 0
    for r, c in enumerate(need):
        bt[r, :c] = perm[at:at + c]
        at += c
    P = sum(need) + spare
    data = torch.randn(P, H, bs // 64, 2, 64 * D, generator=g).mul_(96).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    exps = torch.randint(118, 123, (P, H, bs // 64, 2), generator=g).to(torch.uint8)
    qsl = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int64)
    return data, exps, bt, torch.tensor(last, dtype=torch.int64), qsl, sum(new) + pad, g


def same(a, b):
    """Equal bytes, but for the sign of a NaN code."""
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    return bool(((a == b) | nan).all())


def tables(n, F, D):
    fr = torch.arange(n, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, 2 * F, 2, dtype=torch.float64) / D)
    return fr.cos().to(torch.bfloat16), fr.sin().to(torch.bfloat16)


APPENDS = [([0], [1]), ([63], [1]), ([64], [1]), ([5], [59]), ([5], [60]), ([0, 0, 0], [64, 65, 1]), ([130, 0, 17, 64], [3, 200, 0, 128]),
           ([1000, 3, 62, 127, 128], [1, 5, 2, 1, 7])]


@pytest.mark.parametrize("prev,new", APPENDS, ids=str)
@pytest.mark.parametrize("H,D,bs,F", [(4, 128, 128, 32), (4, 128, 64, 64), (1, 64, 256, 8), (8, 64, 64, 32), (3, 128, 192, 0)])
def test_append_bytes(kv8, prev, new, H, D, bs, F):
    data, exps, bt, lens, qsl, T, g = rows(kv8, 7 * H + len(prev), prev, new, H, D, bs, pad=3)
    # magnitudes from one token to the next: some blocks grow, some keep their exponent
    x = (torch.randn(T, 2 * H, D, generator=g) * torch.pow(2.0, torch.randint(-6, 7, (T, 1, 1), generator=g))).to(torch.bfloat16)
    cos, sin = tables(int(lens.max()) + 1, F, D) if F else (None, None)
    want = ref.append(data, exps, x[:, :H], x[:, H:], bt, lens, qsl, cos, sin)
    up = lambda t: None if t is None else t.to(DEV)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    xd = x.to(DEV)
    kv8.append(c, xd[:, :H], xd[:, H:], up(bt), up(lens), up(qsl), up(cos), up(sin))
    assert torch.equal(c.exps.cpu(), want[1])
    assert same(c.data.cpu(), want[0])
    k, v = kv8.dequantize(c)
    for got, held in zip((k, v), ref.values(*want)):
        assert torch.equal(got.cpu().double(), held)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_append_extremes(kv8, bad):
    """Infinities and NaN become NaN and leave the exponent alone; zeros, subnormals and the largest numbers keep theirs."""
    for D in (64, 128):
        data, exps, bt, lens, qsl, T, g = rows(kv8, 3, [0, 10, 70], [64, 20, 1], 2, D, 64)
        x = torch.randn(T, 4, D, generator=g)
        x[0] = 0.0
        x[3] *= 1e-39
        x[70, :, 5] = 3.0e38
        x[5, 1, 3] = x[80, 2, D - 1] = x[T - 1, 0, 0] = bad
        x[64:84, 3] = bad                                      # a head without a finite value
        x = x.to(torch.bfloat16)
        want = ref.append(data, exps, x[:, :2], x[:, 2:], bt, lens, qsl)
        c = kv8.Cache8(data.to(DEV), exps.to(DEV))
        kv8.append(c, x[:, :2].to(DEV), x[:, 2:].to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV))
        assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])


def test_append_tables_and_positions(kv8):
    """Entries that are no pages, positions past the table and before the first one, positions past the rope tables."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 4, [60, 250, 0, 5], [10, 20, 30, 4], 4, 128, 64, cols=1)
    bt[0, 1], bt[1, 4], bt[2, 0] = -1, 1 << 20, -5
    lens[3] = 2                                                # two of its four tokens would stand before position 0
    x = torch.randn(T, 8, 128, generator=g).to(torch.bfloat16)
    cos, sin = tables(100, 32, 128)
    want = ref.append(data, exps, x[:, :4], x[:, 4:], bt, lens, qsl, cos, sin)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    xd = x.to(DEV)
    kv8.append(c, xd[:, :4], xd[:, 4:], bt.to(DEV), lens.to(DEV), qsl.to(DEV), cos.to(DEV), sin.to(DEV))
    assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])


def check_attend(kv8, data, exps, q, bt, lens, qsl, window=0, scale=None):
    want, far = ref.attend(data, exps, q, bt, lens, qsl, window, scale)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    got = kv8.attend(c, q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV), window=window, scale=scale).cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    worst = float(((got - want).abs()[fine] / far[fine].clamp(min=1e-30)).max())
    assert worst <= 1.0, worst
    return got


ATTENDS = [([0], [1]), ([62], [1]), ([63], [2]), ([127], [1]), ([128], [1]), ([700, 0, 5, 1300], [1, 1, 1, 1]), ([40, 300, 0, 129], [3, 0, 17, 6]),
           ([0, 70], [150, 40]), ([2500], [5]), ([0], [300]), ([513, 64, 9, 200], [129, 0, 200, 1]), ([1000], [65])]


@pytest.mark.parametrize("window", [0, 1, 100, 256])
@pytest.mark.parametrize("prev,new", ATTENDS, ids=str)
@pytest.mark.parametrize("Hq,H,D,bs", [(16, 4, 128, 128), (4, 4, 64, 64), (16, 1, 128, 64), (6, 2, 64, 192)])
def test_attend(kv8, prev, new, Hq, H, D, bs, window):
    data, exps, bt, lens, qsl, T, g = rows(kv8, Hq + len(prev), prev, new, H, D, bs, pad=2)
    q = (torch.randn(T, Hq, D, generator=g) * 2).to(torch.bfloat16)
    got = check_attend(kv8, data, exps, q, bt, lens, qsl, window)
    assert not got[int(qsl[-1]):].any()


def test_attend_sees_nothing_else(kv8):
    """NaN codes behind the rows' ends, before the window and in tokens that only later queries see."""
    for window in (0, 70):
        data, exps, bt, lens, qsl, T, g = rows(kv8, 9, [200, 130, 3], [8, 1, 60], 2, 128, 64)
        K, V = ref.tables(128)
        for r in range(3):
            n, c = int(lens[r]), int(qsl[r + 1] - qsl[r])
            for p in list(range(n, -(-n // 64) * 64)) + ([p for p in range(max(0, n - c - 1 - window))] if window else []):
                data[int(bt[r, p // 64]), :, 0, 0, K[p % 64]] = 0x7F
                data[int(bt[r, p // 64]), :, 0, 1, V[p % 64]] = 0xFF
        # one value and one key of the middle of a chunk: NaN for the queries from there on
        data[int(bt[0, 204 // 64]), 0, 0, 1, V[204 % 64, 7]] = 0x7F
        data[int(bt[2, 0]), 1, 0, 0, K[30, 100]] = 0x7F
        q = torch.randn(T, 8, 128, generator=g).to(torch.bfloat16)
        got = check_attend(kv8, data, exps, q, bt, lens, qsl, window)
        assert not got[:4].isnan().any() and got[4:8, :4, 7].isnan().all() and not got[4:8, :4, :7].isnan().any()


def test_prompt_sees_nothing_else(kv8):
    """The same in prompt chunks, at their causal edge and at the window's."""
    for window, D in ((0, 128), (90, 64)):
        data, exps, bt, lens, qsl, T, g = rows(kv8, 19, [70, 0], [150, 131], 1, D, 64)
        K, V = ref.tables(D)
        for r in range(2):
            n, c = int(lens[r]), int(qsl[r + 1] - qsl[r])
            for p in list(range(n, -(-n // 64) * 64)) + ([p for p in range(max(0, n - c - 1 - window))] if window else []):
                data[int(bt[r, p // 64]), :, 0, 0, K[p % 64]] = 0x7F
                data[int(bt[r, p // 64]), :, 0, 1, V[p % 64]] = 0xFF
        data[int(bt[0, 2]), 0, 0, 1, V[140 % 64, 9]] = 0xFF
        data[int(bt[1, 1]), 0, 0, 0, K[80 % 64, 33]] = 0x7F
        q = torch.randn(T, 4, D, generator=g).to(torch.bfloat16)
        got = check_attend(kv8, data, exps, q, bt, lens, qsl, window)
        assert not got[:70].isnan().any() and got[70, :, 9].isnan().all() and not got[150:230].isnan().any() and got[230].isnan().all()


def test_negative_scale(kv8):
    for new in ([2, 1], [100, 80]):
        data, exps, bt, lens, qsl, T, g = rows(kv8, 6, [200, 10], new, 2, 64, 64)
        q = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16)
        check_attend(kv8, data, exps, q, bt, lens, qsl, scale=-0.1)


def test_attend_all_nan(kv8):
    """A query whose every visible key is NaN has NaN outputs, in each lane group's tokens."""
    for n in (1, 20, 40, 70, 300):
        data, exps, bt, lens, qsl, T, g = rows(kv8, n, [n - 1, 5], [1, 1], 1, 64, 64)
        data[bt[0, :-(-n // 64)].long(), :, :, 0] = 0x7F
        q = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16)
        got = check_attend(kv8, data, exps, q, bt, lens, qsl)
        assert got[0].isnan().all() and not got[1].isnan().any()


@pytest.mark.parametrize("spread", [0, 12, 40])
def test_attend_ranges(kv8, spread):
    """Exponents of the blocks far apart, one dominant key, strong channels of q, a scale of its own, no pages at all."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, spread, [900, 64], [3, 2], 4, 128, 128)
    exps = (exps.int() + torch.randint(-spread, spread // 4 + 1, exps.shape, generator=g)).clamp(27, 247).to(torch.uint8)
    q = torch.randn(T, 16, 128, generator=g)
    q[:, :, 3] *= 30
    q[1, 2] = 0
    q[2] *= 1e-30
    check_attend(kv8, data, exps, q.to(torch.bfloat16), bt, lens, qsl, scale=0.02)
    bt[1] = -1
    got = check_attend(kv8, data, exps, q.to(torch.bfloat16), bt, lens, qsl, scale=0.02)
    assert not got[3:].any()


@pytest.mark.parametrize("prev,new", [([5000], [1]), ([3000, 1, 400, 2047], [1, 2, 1, 1]), ([6000], [40]), ([4000, 700], [33, 100])], ids=str)
@pytest.mark.parametrize("window", [0, 1500])
def test_attend_split(kv8, prev, new, window):
    """Long rows, whose keys several workgroups share, beside short ones, in tables wider than the rows."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 31, prev, new, 2, 128, 64, pad=3, cols=9)
    q = (torch.randn(T, 8, 128, generator=g) * 2).to(torch.bfloat16)
    got = check_attend(kv8, data, exps, q, bt, lens, qsl, window)
    assert not got[int(qsl[-1]):].any()


def test_attend_many_rows(kv8):
    """More rows than a workgroup has threads, some without tokens."""
    g = torch.Generator().manual_seed(1)
    prev = torch.randint(0, 200, (700,), generator=g).tolist()
    new = torch.randint(0, 3, (700,), generator=g).tolist()
    data, exps, bt, lens, qsl, T, g = rows(kv8, 5, prev, new, 1, 64, 64)
    q = torch.randn(T, 2, 64, generator=g).to(torch.bfloat16)
    check_attend(kv8, data, exps, q, bt, lens, qsl)
