"""decode_chunk's weights of quantized values over the whole range of a softmax: one key far above the others, as the first token
of a text often is, whose value is near zero, so that the output is the others' alone. Tolerance as in test_gpu_chunk.py, whose
11 bits of a weight are meant for every weight that counts, not only for those near the largest."""
import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import check

pytestmark = pytest.mark.gpu


def refill(c, hip, r, K, V):
    """Row r's keys and values (N, 4, 128) in place of those that the cache was made with."""
    P, m, a = c.P, c.nq[r], c.first[r]
    c.K[r], c.V[r] = K, V
    c.sb[r] = hip.quantize_blocks(K[:m * 256].view(m, 256, 4, 128), V[:m * 256].view(m, 256, 4, 128))
    for j in range(m):
        at = int(P.boff[r, j])
        P.qpool.view(-1)[at:at + 51200] = c.sb[r][j]
    pos = torch.arange(a, c.N[r], device=c.dev)
    at = P.eoff[r][pos // P.ebs][:, None, None] + torch.arange(4, device=c.dev)[:, None] * P.e_hs + \
        (pos % P.ebs)[:, None, None] * P.e_ts + torch.arange(128, device=c.dev)
    flat = P.epool.view(-1)
    flat[at] = K[a:]
    flat[at + P.e_v] = V[a:]


@pytest.mark.parametrize("launches", [1, 2])
@pytest.mark.parametrize("new", [3, 7])
@pytest.mark.parametrize("above", [4, 12, 17])           # nats between the first key's score and the others' mean
@pytest.mark.parametrize("size", [1.0, 2 ** -7])         # of the values
def test_a_key_far_above_the_others(hip, launches, new, above, size):
    R, prev = 60, 2100
    c = ref.Cache(hip, [prev] * R, [new] * R, ebs=64, seed=61)
    if launches == 2:
        c.P.nqmax = 8 * torch.cuda.get_device_properties(0).multi_processor_count // R + 1
    g = torch.Generator(device=c.dev).manual_seed(62)
    still = torch.zeros(128, dtype=torch.bool, device=c.dev)   # the dims that do not rotate
    still[32:64] = still[96:] = True
    c.q[..., still] = 2.0
    c.q[..., ~still] *= 0.25
    for r in range(R):
        K = torch.randn(c.N[r], 4, 128, generator=g, device=c.dev) * 0.1
        V = torch.randn(c.N[r], 4, 128, generator=g, device=c.dev) * size
        K[0, :, still] = above * 128 ** 0.5 / (2.0 * 64)
        V[0] = 0.0
        refill(c, hip, r, K.to(torch.bfloat16), V.to(torch.bfloat16))
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"a key {above} above, values of {size}, {new} new")


@pytest.mark.parametrize("new", [3, 7])
def test_value_scales_that_grow_and_shrink(hip, new):
    """Values whose size changes from token to token and block to block by up to 2^14, up and down along the row: a weight's
    bits count from the largest scale so far."""
    R, prev = 60, 2100
    c = ref.Cache(hip, [prev] * R, [new] * R, ebs=64, seed=63)
    g = torch.Generator(device=c.dev).manual_seed(64)
    for r in range(R):
        n = c.N[r]
        K = torch.randn(n, 4, 128, generator=g, device=c.dev)
        V = torch.randn(n, 4, 128, generator=g, device=c.dev)
        t = torch.arange(n, device=c.dev)
        e = (t // 64 % 15 if r % 3 == 0 else 14 - t // 64 % 15 if r % 3 == 1 else (t * 7) % 15).float() - 9
        V *= torch.exp2(e)[:, None, None]
        refill(c, hip, r, K.to(torch.bfloat16), V.to(torch.bfloat16))
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"scales that change, {new} new")
