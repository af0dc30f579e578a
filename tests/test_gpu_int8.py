"""Products in 8-bit integers on the GPU against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def i8(hip):
    import lfm3_kv800_amd.int8_ops as m
    return m


def quantized(x):
    """Codes and scales of bf16 rows as 32-bit arithmetic gives them (the definition's), float64."""
    t = x.float().abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    inv = torch.full_like(t, 127) / t                          # a division (127 / t would be a product with 1 / t)
    return (x.float() * inv).round().double(), (t / 127).double()


def product(x, w, scale, gated):
    """(y, how far a kernel's may be): the integer sums are exact; three roundings of 2^-24 by the scales and the conversion, in
    silu a relative 2^-20 of its exponential's argument and quotient, one of 2^-8 to bf16."""
    q, s = quantized(x)
    y = q @ w.double().T * s * scale.double()
    if not gated:
        return y, 2 ** -8 * y.abs() * (1 + 2 ** -10) + 2.0 ** -133
    g, u = y.chunk(2, 1)
    o = g * torch.sigmoid(g) * u
    return o, (2 ** -8 + 2 ** -18 * (1 + g.abs())) * o.abs() + 2.0 ** -126 * (1 + u.abs())


SIZES = [(1, 2, 8), (1, 64, 128), (3, 70, 136), (32, 32, 2048), (33, 66, 200), (64, 6144, 2048), (65, 130, 264), (127, 34, 8200), (128, 128, 128), (129, 3088, 1000),
         (250, 1000, 384), (256, 2048, 8192), (300, 514, 640), (513, 258, 1032), (4, 100, 2048), (16, 100, 4160), (300, 12900, 264), (200, 70, 4104), (2048, 6160, 136), (1500, 9000, 264)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("R,N,K", SIZES, ids=str)
def test_linear8(i8, R, N, K, gated):
    g = torch.Generator().manual_seed(R + N + K)
    x = torch.randn(R, K, generator=g)
    x[:, ::5] *= 6
    x = x.to(torch.bfloat16)
    w = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
    scale = torch.rand(N, generator=g) * 1e-3 + 1e-4
    want, far = product(x, w, scale, gated)
    got = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV), scale.to(DEV), gated=gated)).cpu().double()
    assert got.shape == (R, N // 2 if gated else N)
    worst = float(((got - want).abs() / far).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("R", [1, 40, 300])
def test_linear8_extremes(i8, R):
    """The largest sums (all codes 127, -128 among the weights), zero rows, subnormal rows, infinities and NaN in one token."""
    K, N = 65536, 96
    x = torch.full((R, K), -2.5)
    w = torch.full((N, K), 127, dtype=torch.int8)
    w[1], w[2, ::2] = -128, -127
    scale = torch.full((N,), 2.0 ** -20)
    x[R // 2] = 0.0
    if R > 4:
        x[1] = 1e-39
        x[2, 77], x[3, 5] = math.inf, math.nan
    x = x.to(torch.bfloat16)
    want, far = product(x, w, scale, False)
    got = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV), scale.to(DEV))).cpu().double()
    for r in range(R):
        if not torch.isfinite(x[r].float()).all():
            assert got[r].isnan().all()
        else:
            assert ((got[r] - want[r]).abs() <= far[r]).all(), r
    assert not got[R // 2].any()


def test_quantize_rows(i8):
    for N, K in ((1, 8), (37, 264), (5, 8192), (3, 20000)):
        g = torch.Generator().manual_seed(K)
        w = (torch.randn(N, K, generator=g) * 0.02).to(torch.bfloat16)
        w[0] = 0
        q, s = quantized(w)
        codes, scale = i8.quantize_rows(w.to(DEV))
        assert torch.equal(codes.cpu().double(), q) and torch.equal(scale.cpu().double(), s[:, 0])
        y = i8.linear8(w.to(DEV), i8.Weight8(w.to(DEV)))
        want, far = product(w, q, s[:, 0], False)
        assert ((y.cpu().double() - want).abs() <= far).all()


def test_views(i8):
    """Rows of a wider product, one row of any stride, unaligned and transposed data."""
    g = torch.Generator().manual_seed(2)
    big = torch.randn(40, 600, generator=g).to(torch.bfloat16)
    w = torch.randint(-127, 128, (100, 256), generator=g).to(torch.int8)
    scale = torch.rand(100, generator=g)
    W = i8.Weight8(w.to(DEV), scale.to(DEV))
    wt = i8.Weight8(w.to(DEV).t().contiguous().t(), scale.to(DEV).repeat_interleave(2)[::2])
    assert torch.equal(W.data, wt.data) and torch.equal(W.scale, wt.scale)
    d = big.to(DEV)
    for x, v in ((big[:, 8:264], d[:, 8:264]), (big[:, 3:259], d[:, 3:259]), (big[5:6, 16:272], d[5:6, 16:272]), (big[::3, :256], d[::3, :256]),
                 (big[:40, :256].t()[:40, :].t(), None)):
        if v is None or v.shape[1] != 256:
            continue
        want, far = product(x, w, scale, False)
        assert ((i8.linear8(v, W).cpu().double() - want).abs() <= far).all()
    t = big[:, :256].t().contiguous().to(DEV).t()
    assert torch.equal(i8.linear8(t, W), i8.linear8(d[:, :256], W))
