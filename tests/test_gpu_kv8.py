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


@pytest.mark.parametrize("R", [64, 70])
@pytest.mark.parametrize("G", [4, 3])
def test_attend_drafts_of_many_rows(kv8, R, G):
    """Tiles of 32 columns: a large step of drafts in tables wider than the rows, some of them empty, one token of NaN values that only
    later queries see, up to 64 rows and beyond."""
    g = torch.Generator().manual_seed(R)
    prev = torch.randint(0, 260, (R,), generator=g).tolist()
    prev[3], prev[R - 2] = 1000, 700
    new = torch.randint(5, 10, (R,), generator=g).tolist()
    new[0] = new[17] = 0
    data, exps, bt, lens, qsl, T, g = rows(kv8, 6, prev, new, 8, 64, 64, pad=2, cols=2)
    assert R * 8 * bt.shape[1] * 64 >= 1 << 19
    bad = prev[3] + 2
    data[int(bt[3, bad // 64]), :, 0, 1, ref.tables(64)[1][bad % 64, 11]] = 0x7F
    q = torch.randn(T, 8 * G, 64, generator=g).to(torch.bfloat16)
    got = check_attend(kv8, data, exps, q, bt, lens, qsl)
    a, b = int(qsl[3]), int(qsl[4])
    assert not got[a:a + 2].isnan().any() and got[a + 2:b, :, 11].isnan().all() and not got[b:].isnan().any()
    if R == 64 and G == 4:
        check_attend(kv8, data, exps, q, bt, lens, qsl, window=1100)


def test_attend_many_long_rows(kv8):
    """More rows than lanes in lists of 128 positions."""
    g = torch.Generator().manual_seed(8)
    prev = torch.randint(0, 150, (300,), generator=g).tolist()
    prev[7], prev[250] = 1500, 1200
    new = torch.randint(0, 3, (300,), generator=g).tolist()
    new[7] = 2
    data, exps, bt, lens, qsl, T, g = rows(kv8, 5, prev, new, 1, 64, 64)
    q = torch.randn(T, 2, 64, generator=g).to(torch.bfloat16)
    check_attend(kv8, data, exps, q, bt, lens, qsl)


SHAPES = [([300, 64], [1, 1]), ([1500, 0], [1, 1]), ([2100, 5], [5, 2]), ([200, 90], [70, 64])]


@pytest.mark.parametrize("prev,new", SHAPES, ids=str)
def test_queries_that_are_no_numbers(kv8, prev, new):
    """An infinity or NaN in one query stays with it; scores far below what exponents reach, on their own, are still a softmax's."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 41, prev, new, 2, 64, 64)
    q = torch.randn(T, 8, 64, generator=g)
    q[0, 1, 3], q[T - 1, 5, 9] = math.nan, math.inf
    q = q.to(torch.bfloat16)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    got = kv8.attend(c, q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV)).cpu().double()
    clean = q.clone()
    clean[0, 1], clean[T - 1, 5] = 0, 0
    want, far = ref.attend(data, exps, clean, bt, lens, qsl)
    rest = torch.ones(T, 8, dtype=torch.bool)
    rest[0, 1] = rest[T - 1, 5] = False
    assert got[0, 1].isnan().all() and got[T - 1, 5].isnan().all()
    assert float(((got - want).abs() / far)[rest].max()) <= 1.0
    # keys of one value, so that all scores of a query are equal: about -2^114, the mean of what it sees
    data[:, :, :, 0] = 0x38
    exps[..., 0] = 247
    q = torch.full((T, 8, 64), -2.0 ** -9)
    check_attend(kv8, data, exps, q.to(torch.bfloat16), bt, lens, qsl, scale=2.0 ** -3)


def test_lengths_and_tables_at_their_ends(kv8):
    """Lengths past the table and before its first position, a table without columns, rows without tokens, no rows, no tokens."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 12, [100, 64, 30, 10], [3, 70, 0, 2], 2, 128, 64, pad=1)
    lens = torch.tensor([400, 150, -7, 1])
    x = torch.randn(T, 4, 128, generator=g).to(torch.bfloat16)
    q = torch.randn(T, 8, 128, generator=g).to(torch.bfloat16)
    want = ref.append(data, exps, x[:, :2], x[:, 2:], bt, lens, qsl)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    up = lambda *a: [t.to(DEV) for t in a]
    kv8.append(c, *up(x[:, :2], x[:, 2:], bt, lens, qsl))
    assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])
    check_attend(kv8, *want, q, bt, lens, qsl)
    none = torch.empty(4, 0, dtype=torch.int32)
    kv8.append(c, *up(x[:, :2], x[:, 2:], none, lens, qsl))
    assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])
    assert not kv8.attend(c, *up(q, none, lens, qsl)).any()
    e = torch.zeros(0, dtype=torch.int64)
    one = torch.zeros(1, dtype=torch.int64)
    kv8.append(c, *up(x[:0, :2], x[:0, 2:], bt[:0], e, one))
    assert kv8.attend(c, *up(q[:0], bt[:0], e, one)).shape == (0, 8, 128)
    assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])


def test_views_of_everything(kv8):
    """Pages apart in a pool, a table and queries that are views, keys that heads share, unaligned values; rows that share pages."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 14, [200, 130, 70], [1, 3, 2], 2, 128, 64)
    bt[1, 0] = bt[0, 0]                                         # a prefix of 64 tokens in common
    wide = torch.full((3, 9), -1, dtype=torch.int32)
    wide[:, 2:2 + bt.shape[1]] = bt
    P = data.shape[0]
    pool, epool = torch.zeros(2 * P, *data.shape[1:], dtype=torch.uint8), torch.zeros(3 * P, *exps.shape[1:], dtype=torch.uint8)
    pool[::2], epool[1::3] = data, exps
    pd, ed = pool.to(DEV), epool.to(DEV)
    c = kv8.Cache8(pd[::2], ed[1::3])
    btd = wide.to(DEV)[:, 2:2 + bt.shape[1]]
    k1 = torch.randn(T, 1, 128, generator=g).to(torch.bfloat16)
    vv = torch.randn(T * 2 * 128 + 3, generator=g).to(torch.bfloat16)
    kd, vd = k1.to(DEV).expand(T, 2, 128), vv.to(DEV)[3:].view(T, 2, 128)
    kv8.append(c, kd, vd, btd, lens.to(DEV), qsl.to(DEV))
    want = ref.append(data, exps, k1.expand(T, 2, 128), vv[3:].view(T, 2, 128), bt, lens, qsl)
    assert torch.equal(ed.cpu()[1::3], want[1]) and same(pd.cpu()[::2], want[0])
    assert not pd.cpu()[1::2].any() and not ed.cpu()[0::3].any() and not ed.cpu()[2::3].any()
    q = torch.randn(8, T, 200, generator=g).to(torch.bfloat16)
    qv = q.to(DEV).transpose(0, 1)[:, :, 5:133]
    for scale in (None, -0.05):
        o = kv8.attend(c, qv, btd, lens.to(DEV), qsl.to(DEV), scale=scale).cpu().double()
        ow, far = ref.attend(*want, q.transpose(0, 1)[:, :, 5:133], bt, lens, qsl, scale=scale)
        assert float(((o - ow).abs() / far).max()) <= 1.0
    k, v = kv8.dequantize(c)
    for got, held in zip((k, v), ref.values(*want)):
        assert torch.equal(got.cpu().double(), held)


def test_offsets_past_32_bits(kv8):
    """Pages 2 GiB apart: bytes past 2^32 are the ones that a row's pages lie at."""
    need = 3 * (1 << 31)
    if torch.cuda.mem_get_info()[0] < need + (1 << 30):
        pytest.skip("not enough memory")
    pool = torch.empty(need, dtype=torch.uint8, device=DEV)
    H, D, U = 2, 64, 1
    dv = pool.as_strided((3, H, U, 2, 64 * D), (1 << 31, U * 2 * 64 * D, 2 * 64 * D, 64 * D, 1))
    data, exps, bt, lens, qsl, T, g = rows(kv8, 15, [100, 10], [2, 1], H, D, 64, spare=0)
    assert data.shape[0] == 3
    dv.copy_(data.to(DEV))
    c = kv8.Cache8(dv, exps.to(DEV))
    x = torch.randn(T, 2 * H, D, generator=g).to(torch.bfloat16)
    xd = x.to(DEV)
    kv8.append(c, xd[:, :H], xd[:, H:], bt.to(DEV), lens.to(DEV), qsl.to(DEV))
    want = ref.append(data, exps, x[:, :H], x[:, H:], bt, lens, qsl)
    assert torch.equal(c.exps.cpu(), want[1]) and same(dv.cpu(), want[0])
    q = torch.randn(T, 8, D, generator=g).to(torch.bfloat16)
    got = kv8.attend(c, q.to(DEV), bt.to(DEV), lens.to(DEV), qsl.to(DEV)).cpu().double()
    ow, far = ref.attend(*want, q, bt, lens, qsl)
    assert float(((got - ow).abs() / far).max()) <= 1.0
    del c, dv, pool
    torch.cuda.empty_cache()


@pytest.mark.parametrize("prev,new", SHAPES + [([700, 600], [200, 129])], ids=str)
def test_recorded_and_on_other_streams(kv8, prev, new):
    """Append and attention recorded into two graphs and replayed in turn on new inputs, with eager work between; the same on two
    streams at once: equal bits."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 16, prev, new, 2, 128, 64, pad=2)
    xs = torch.randn(6, T, 4, 128, generator=g).to(torch.bfloat16).to(DEV)
    qs = torch.randn(6, T, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    btd, ld, qd = bt.to(DEV), lens.to(DEV), qsl.to(DEV)

    def fresh():
        return kv8.Cache8(data.to(DEV), exps.to(DEV))

    def step(c, x, q):
        kv8.append(c, x[:, :2], x[:, 2:], btd, ld, qd)
        return kv8.attend(c, q, btd, ld, qd)

    eager = fresh()
    want = [step(eager, xs[i], qs[i]).clone() for i in range(6)]
    caches, inputs, graphs, outs = [], [], [], []
    for n in range(2):
        c, x, q = fresh(), xs[0].clone(), qs[0].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(c, x, q)
        torch.cuda.current_stream().wait_stream(s)
        c.data.copy_(data)
        c.exps.copy_(exps)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(c, x, q)
        caches.append(c); inputs.append((x, q)); graphs.append(gr); outs.append(out)
    for i in range(6):
        for n in range(2):
            inputs[n][0].copy_(xs[i]); inputs[n][1].copy_(qs[i])
            graphs[n].replay()
        kv8.attend(eager, qs[0], btd, ld, qd)
        torch.cuda.synchronize()
        for n in range(2):
            assert torch.equal(outs[n], want[i]), (i, n)
    # two streams, the cache's work on each in turn with nothing of the other waited for
    a, b = fresh(), fresh()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = {}
    for i in range(6):
        for c, s, key in ((a, sa, "a"), (b, sb, "b")):
            with torch.cuda.stream(s):
                got[key, i] = step(c, xs[i], qs[i])
    torch.cuda.synchronize()
    for i in range(6):
        assert torch.equal(got["a", i], want[i]) and torch.equal(got["b", i], want[i])


def test_calls_that_are_refused(kv8):
    data, exps, bt, lens, qsl, T, g = rows(kv8, 17, [10, 3], [1, 2], 2, 64, 64)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    k = torch.randn(T, 2, 64).to(torch.bfloat16).to(DEV)
    q = torch.randn(T, 4, 64).to(torch.bfloat16).to(DEV)
    btd, ld, qd = bt.to(DEV), lens.to(DEV), qsl.to(DEV)
    cos = torch.ones(9, 16, dtype=torch.bfloat16, device=DEV)
    ok = dict(k=k, v=k, bt=btd, lens=ld, qsl=qd, cos_t=None, sin_t=None)
    ap = lambda **a: kv8.append(c, *{**ok, **a}.values())
    for a in (dict(k=k.float()), dict(v=k.half()), dict(k=k.cpu()), dict(bt=btd.long()), dict(lens=ld.int()), dict(qsl=qd.int()), dict(bt=bt), dict(lens=lens),
              dict(k=k[:2]), dict(v=k[:, :1]), dict(k=k[..., :32]), dict(k=k[0]), dict(bt=btd[:1]), dict(bt=btd[0]), dict(lens=ld[:1]), dict(qsl=qd[None]),
              dict(qsl=qd[:0]), dict(cos_t=cos), dict(cos_t=cos, sin_t=cos[:, :8]), dict(cos_t=cos[:, :12], sin_t=cos[:, :12]), dict(cos_t=cos.float(), sin_t=cos),
              dict(cos_t=cos[:0], sin_t=cos[:0]), dict(cos_t=cos[0], sin_t=cos[0]), dict(bt=btd.repeat(1, 4)[:, ::2]), dict(bt=btd[:0], lens=ld[:0], qsl=qd[:1])):
        with pytest.raises((TypeError, ValueError)):
            ap(**a)
    at = lambda *a, **kw: kv8.attend(c, *a, **kw)
    for a, kw in (((q.float(), btd, ld, qd), {}), ((q[:, :3], btd, ld, qd), {}), ((q[..., :32], btd, ld, qd), {}), ((q[0], btd, ld, qd), {}), ((q[:, :0], btd, ld, qd), {}),
                  ((q.repeat(1, 9, 1), btd, ld, qd), {}), ((q.cpu(), btd, ld, qd), {}), ((q, btd, ld, qd), dict(window=-1)), ((q, btd, ld, qd), dict(scale=0.0)),
                  ((q, btd, ld, qd), dict(scale=math.nan)), ((q, btd[:0], ld[:0], qd[:1]), {})):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            at(*a, **kw)
    assert torch.equal(c.data.cpu(), data) and torch.equal(c.exps.cpu(), exps)
    assert torch.equal(at(q, btd, ld, qd), at(q, btd, ld, qd, window=1 << 70))


@pytest.mark.parametrize("pad,prev", [(3, [700, 64]), (3, [3000, 64]), (200, [3000, 64]), (3, [100] * 70 + [1500])], ids=["direct", "list", "prompt", "rows"])
def test_steps_of_padding(kv8, pad, prev):
    """Rows that all bring nothing, in room for some tokens: zeros, and the cache stays."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 23, prev, [0] * len(prev), 2, 64, 64, pad=pad)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    x = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    kv8.append(c, x[:, :2], x[:, 2:], bt.to(DEV), lens.to(DEV), qsl.to(DEV))
    assert torch.equal(c.data.cpu(), data) and torch.equal(c.exps.cpu(), exps)
    assert not kv8.attend(c, x, bt.to(DEV), lens.to(DEV), qsl.to(DEV)).any()


@pytest.mark.parametrize("prev,new", SHAPES + [([60, 700], [20, 30])], ids=str)
def test_rows_past_the_tokens(kv8, prev, new):
    """Starts of rows past the tokens that are there: the present ones stand where the lengths put them."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 29, prev, new, 2, 64, 64)
    T -= 1
    x = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16)
    q = torch.randn(T, 8, 64, generator=g).to(torch.bfloat16)
    want = ref.append(data, exps, x[:, :2], x[:, 2:], bt, lens, qsl)
    c = kv8.Cache8(data.to(DEV), exps.to(DEV))
    xd = x.to(DEV)
    kv8.append(c, xd[:, :2], xd[:, 2:], bt.to(DEV), lens.to(DEV), qsl.to(DEV))
    assert torch.equal(c.exps.cpu(), want[1]) and same(c.data.cpu(), want[0])
    check_attend(kv8, *want, q, bt, lens, qsl)
