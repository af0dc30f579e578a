"""Attention over the 8-bit cache with scores far from 0: what the weights are relative to has to be what they were taken from."""
import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8 import DEV, SHAPES, kv8, rows

pytestmark = pytest.mark.gpu


# (keys' exponent byte, query): scores of 64 x 2^(byte - 127) x query / 8, up to 1.875 times that with other codes
@pytest.mark.parametrize("byte,x", [(247, -1.25 * 2.0 ** -9), (247, 1.25 * 2.0 ** -9), (160, -1.296875), (160, 1.296875), (145, -1.09375), (150, 1.703125)])
@pytest.mark.parametrize("prev,new", SHAPES + [([1500, 700], [70, 64]), ([30], [300])], ids=str)
def test_large_scores(kv8, prev, new, byte, x):
    """Scores of up to 2^115, queries that are no powers of two: keys that are all the same give the mean of the values, one key ahead
    of all others gives its value. Equal scores have equal weights, so the mean is off by its rounding to bf16 (2^-8 of it) and that
    of equal weights of n values (2^-8) in 32 bits."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 51, prev, new, 2, 64, 64)
    K, V = ref.tables(64)
    data[:, :, :, 0] = 0x38                                                    # 1.0
    exps[..., 0] = byte
    q = torch.full((T, 8, 64), x).to(torch.bfloat16)
    assert float(q[0, 0, 0]) == x
    up = lambda *a: [t.to(DEV) for t in a]
    c = kv8.Cache8(*up(data, exps))
    got = kv8.attend(c, *up(q, bt, lens, qsl)).cpu().double()
    vals = ref.values(data, exps)[1]
    for r in range(len(prev)):
        pos = torch.arange(int(lens[r]))
        v = vals[bt[r].long()[pos // 64], :, pos % 64]                        # (n, 2, 64)
        for j in range(int(qsl[r]), int(qsl[r + 1])):
            see = v[:int(lens[r]) - int(qsl[r + 1]) + j + 1]
            mean, size = (t.repeat_interleave(4, 0) for t in (see.mean(0), see.abs().mean(0)))
            far = 2 ** -8 * mean.abs() + (2 ** -8 + len(see) * 2 ** -23) * size
            assert ((got[j] - mean).abs() <= far).all(), (r, j)
    # one key of each row ahead: less by an eighth where scores are negative, more where they are not
    for r in range(len(prev)):
        for p in range(int(lens[r])):
            data[int(bt[r, p // 64]), :, 0, 0, K[p % 64]] = 0x38 if (p == 0) == (x < 0) else 0x39
    c = kv8.Cache8(*up(data, exps))
    got = kv8.attend(c, *up(q, bt, lens, qsl)).cpu().double()
    for r in range(len(prev)):
        first = vals[int(bt[r, 0]), :, 0].repeat_interleave(4, 0)
        assert (got[int(qsl[r]):int(qsl[r + 1])] == first).all(), r


@pytest.mark.parametrize("window", [0, 1, 130])
@pytest.mark.parametrize("prev,new", SHAPES + [([0, 63, 64], [1, 1, 1]), ([1500, 700], [70, 64]), ([30], [300])], ids=str)
@pytest.mark.parametrize("D", [64, 128])
def test_equal_values_come_back(kv8, prev, new, window, D):
    """Weights that sum to 1 as they are multiplied: where every key holds the same value, that is the output, to the bit (32-bit sums
    of up to 2,048 products are within 2^-12, a quarter of the least half step of bf16, 2^-9). A weight that is rounded in the
    product and not in the sum is off by up to 2^-8 where it dominates."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 61, prev, new, 2, D, 64)
    value = torch.randint(0x30, 0x48, (D,), generator=g).to(torch.uint8)     # 0.5 .. 3.75
    data[:, :, :, 1, ref.tables(D)[1].reshape(-1)] = value.repeat(64)
    exps[..., 1] = 127
    up = lambda *a: [t.to(DEV) for t in a]
    for spread in (0.3, 2.0, 8.0):
        q = (torch.randn(T, 8, D, generator=g) * spread).to(torch.bfloat16)
        got = kv8.attend(kv8.Cache8(*up(data, exps)), *up(q, bt, lens, qsl), window=window).cpu()
        wrong = (got.float() != value.view(torch.float8_e4m3fn).float()).float().mean()
        assert wrong == 0, (spread, float(wrong))


@pytest.mark.parametrize("prev,new", SHAPES + [([0], [1]), ([1500, 700], [70, 64])], ids=str)
@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_scores_of_minus_infinity(kv8, prev, new, scale):
    """A query with an infinity whose scores are all minus infinity has no softmax: NaN, as 0 / 0 is, not the zeros of a query without
    keys; other queries and heads of its tile stay as they are, and so do tokens that are padding."""
    data, exps, bt, lens, qsl, T, g = rows(kv8, 81, prev, new, 2, 64, 64, pad=2)
    data[:, :, :, 0] = data[:, :, :, 0] & 0x7F                                  # no key is negative,
    data[:, :, :, 0] = data[:, :, :, 0].clamp(min=0x10, max=0x7E)               # nor 0, nor NaN
    q = torch.randn(T, 8, 64, generator=g).to(torch.bfloat16)
    up = lambda *a: [t.to(DEV) for t in a]
    c = kv8.Cache8(*up(data, exps))
    plain = kv8.attend(c, *up(q, bt, lens, qsl), scale=scale).cpu()
    bad = float("-inf") if scale > 0 else float("inf")
    last = int(qsl[-1]) - 1
    q[0, 1, 7] = q[last, 6, 0] = q[last + 1, 2, 5] = bad
    got = kv8.attend(c, *up(q, bt, lens, qsl), scale=scale).cpu()
    assert got[0, 1].isnan().all() and got[last, 6].isnan().all()
    plain[0, 1], plain[last, 6] = got[0, 1], got[last, 6]
    assert torch.equal(got.view(torch.int16), plain.view(torch.int16)) and not got[last + 1:].any()
