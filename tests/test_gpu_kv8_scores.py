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
