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


@pytest.mark.parametrize("R,N,K,gated", [(1, 256, 512, True), (20, 512, 264, False), (256, 512, 2048, False), (1000, 8192, 256, True)], ids=str)
def test_recorded_and_on_other_streams(i8, R, N, K, gated):
    """Two products recorded into two graphs and replayed in turn on new tokens, with eager work between; the same on two streams at
    once: equal bits."""
    g = torch.Generator().manual_seed(R)
    W = i8.Weight8((torch.randn(N, K, generator=g) * 0.05).to(torch.bfloat16).to(DEV), gated=gated)
    xs = torch.randn(5, R, K, generator=g).to(torch.bfloat16).to(DEV)
    want = [i8.linear8(x, W) for x in xs]
    buf, graphs, outs = [xs[0].clone() for _ in range(2)], [], []
    for n in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = i8.linear8(buf[n], W)
        graphs.append(gr); outs.append(out)
    for i in range(5):
        for n in range(2):
            buf[n].copy_(xs[(i + n) % 5])
            graphs[n].replay()
        i8.linear8(xs[0], W)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[(i + 1) % 5]), i
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(5):
        with torch.cuda.stream(streams[i % 2]):
            got.append(i8.linear8(xs[i], W))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_weights_without_numbers(i8):
    """A weight row with an infinity or NaN, or a scale that is none, gives NaN in its channel alone; rows of zeros give zeros."""
    g = torch.Generator().manual_seed(4)
    w = torch.randn(70, 136, generator=g).to(torch.bfloat16)
    w[3, 5], w[40, 0], w[9] = math.inf, math.nan, 0
    x = torch.randn(5, 136, generator=g).to(torch.bfloat16)
    y = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV))).cpu().double()
    q, s = quantized(w[[0, 9, 69]])
    want, far = product(x, q, s[:, 0], False)
    assert y[:, [3, 40]].isnan().all() and ((y[:, [0, 9, 69]] - want).abs() <= far).all() and not y[:, 9].any()
    keep = [n for n in range(70) if n not in (3, 40)]
    assert not y[:, keep].isnan().any()


def test_calls_that_are_refused(i8):
    w, s = torch.ones(64, 64, dtype=torch.int8, device=DEV), torch.ones(64, device=DEV)
    b = torch.ones(64, 64, dtype=torch.bfloat16, device=DEV)
    for a, kw in (((w, s[:63]), {}), ((w, s.double()), {}), ((w, s.cpu()), {}), ((w.cpu(), s.cpu()), {}), ((w.int(), s), {}), ((w,), {}), ((b.float(),), {}), ((b, s), {}),
                  ((w[:, :60], s), {}), ((w[0], s), {}), ((w[:0], s[:0]), {}), ((w[:, :0], s), {}), ((w[:63], s[:63]), dict(gated=True))):
        with pytest.raises((TypeError, ValueError)):
            i8.Weight8(*a, **kw)
    for a in (b.float(), b[:, :60], b[0], b[:0], b[:, :0], w):
        with pytest.raises((TypeError, ValueError)):
            i8.quantize_rows(a)
    W = i8.Weight8(w, s)
    for x in (b.float(), b.cpu(), b[:, :56], b[0], b[None]):
        with pytest.raises((TypeError, ValueError)):
            i8.linear8(x, W)
    assert i8.linear8(b[:0], W).shape == (0, 64)
    assert torch.equal(i8.linear8(b[:1].expand(9, 64), W), i8.linear8(b[:9], W))
