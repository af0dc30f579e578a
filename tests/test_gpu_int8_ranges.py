"""Products in 8-bit integers at the ends of the scales' range."""
import pytest
import torch

from test_gpu_int8 import DEV, i8, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R", [1, 40, 8200])
@pytest.mark.parametrize("u", [1.0, -1e20, 1e30])
def test_gates_far_below_zero(i8, R, u):
    """silu(g) u where the sigmoid leaves the normal numbers of 32 bits and the result does not: g from -200 to 90, u of any size. One
    channel of a token meets one of the weight, so that g and u are the rows' scales by 127. (Bound: as test_linear8's.)"""
    F = 2000
    x = torch.zeros(R, 8)
    x[:, 3] = 1.0
    x = x.to(torch.bfloat16)
    g = torch.linspace(-200, 90, F)
    w = torch.zeros(2 * F, 8, dtype=torch.int8)
    w[:F, 3] = torch.where(g < 0, -127, 127).to(torch.int8)
    w[F:, 3] = 127 if u > 0 else -127
    scale = torch.cat((g.abs(), torch.full((F,), abs(u)))) / 127
    want, far = product(x[:1], w, scale, True)
    assert (want[0, :1000].abs() > 1e-37).any() or u == 1.0
    got = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV), scale.to(DEV), gated=True)).cpu().double()
    y = 127 * scale.double()
    near = (2 ** -8 + 2 ** -18 * (1 + y[:F])) * want.abs() + 2.0 ** -126
    assert torch.equal(got, got[:1].expand(R, F))
    worst = float(((got[:1] - want).abs() / near).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("R,N,K", [(1, 96, 128), (4, 130, 2048), (40, 96, 264), (300, 514, 640), (1500, 9000, 264)], ids=str)
@pytest.mark.parametrize("size,row", [(3e38, 1e-37), (1e38, 1e-41), (2.0 ** 100, 2.0 ** -100), (1e3, 1e-3), (2.0 ** -90, 2.0 ** 90), (1e-30, 1e27)])
def test_scales_far_apart(i8, R, N, K, gated, size, row):
    """Tokens near the largest bf16 and weights whose scales bring the product back, and the other way: the result is in range, and so
    is every product on the way to it. (Bounds: as test_linear8's, a third product by a scale of 1 is exact.)"""
    g = torch.Generator().manual_seed(R + K)
    x = (torch.rand(R, K, generator=g) * 2 - 1).double() * size
    x[:, 0] = size
    x = x.to(torch.bfloat16)
    assert torch.isfinite(x.float()).all()
    w = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
    scale = ((torch.rand(N, generator=g) + 0.5).double() * row / 127).float()
    want, far = product(x, w, scale, gated)
    got = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV), scale.to(DEV), gated=gated)).cpu().double()
    assert torch.isfinite(want.float()).all() and torch.isfinite(got).all()
    worst = float(((got - want).abs() / far).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("R", [1, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(8192, 2048), (8200, 2048), (8200, 2056), (12290, 1000), (16384, 2048), (16386, 2048), (16384, 2056), (8192, 4096), (8192, 4104), (2050, 4096), (34, 2048)], ids=str)
def test_borders_of_rounding_inside(i8, R, N, K, gated):
    """Both sides of where a few tokens are rounded inside their product, on one and on two tiles of the weight a workgroup."""
    g = torch.Generator().manual_seed(R + N + K)
    x = torch.randn(R, K, generator=g).to(torch.bfloat16)
    w = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
    scale = torch.rand(N, generator=g) * 1e-3 + 1e-4
    want, far = product(x, w, scale, gated)
    got = i8.linear8(x.to(DEV), i8.Weight8(w.to(DEV), scale.to(DEV), gated=gated)).cpu().double()
    worst = float(((got - want).abs() / far).max())
    assert worst <= 1.0, worst
