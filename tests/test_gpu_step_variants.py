"""The operators of a step with several new tokens per row in the variants that large calls take: more tokens per workgroup of the
short conv, one or two waves per tile of a window layer, large pieces of a logits row. References and tolerances as in
test_gpu_chunk.py."""
import random

import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import check, conv_case, poison, run_verify, verify_case

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- short conv
def ragged(total, most, seed):
    """Rows of 0 .. most tokens, `total` of them or a few more."""
    rng, new = random.Random(seed), []
    while sum(new) < total:
        new.append(rng.choice([0, 1, 2, 5, 6, 7, rng.randint(0, most)]))
    return new


@pytest.mark.parametrize("H,total,most", [(2048, 1025, 40), (2048, 6150, 300), (2056, 3100, 50), (8, 12300, 30), (8, 6200, 9),
                                          (8, 1100, 1100), (2048, 12300, 4000)])
def test_conv_of_many_tokens(hip, H, total, most):
    """8 and 16 tokens per workgroup (by tokens x blocks of 2,048 channels: beyond 1,024, 6,144, 12,288), rows that begin
    anywhere in them."""
    from lfm3_kv800_amd import spec_ops as so
    new = ragged(total, most, total + H)
    bcx, w, state, qsl = conv_case(new, H, 5, seed=total)
    q = torch.tensor(qsl, device="cuda")
    out, taps = so.conv_chunk(bcx, w, state, q)
    want, tw = ref.conv(bcx, w, state, qsl)
    assert torch.equal(taps.double(), tw)
    mag = ref.conv(bcx.abs(), w.abs(), state.abs(), qsl)[0]
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + 16 * 2 ** -24 * mag).all()
    assert not out[qsl[-1]:].any() and not taps[qsl[-1]:].any()


# ---------------------------------------------------------------- window and sliding layers
@pytest.mark.parametrize("rows,most,least", [(250, 5, 3), (300, 9, 0)])
@pytest.mark.parametrize("sinks,rot", [(True, True), (False, False)])
def test_window_of_a_large_batch(hip, rows, most, least, sinks, rot):
    """More than 1,024 (tile, KV head) pairs: one wave each, tiles of 8."""
    rng = random.Random(rows)
    new = [rng.randint(least, most) for _ in range(rows)]
    assert sum(new) > rows and 4 * (rows + sum(new) // 8) > 4 * torch.cuda.get_device_properties(0).multi_processor_count
    c = ref.Cache(hip, [rng.choice([0, 1, 3, 4, 250, 255, 256, 259, rng.randint(0, 700)]) for _ in new], new, ebs=40, win=256,
                  sinks=sinks, rot=rot, seed=81)
    want = c.want(hip)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, f"window of {rows} rows")
    r = next(i for i, n in enumerate(new) if n > 2)
    t = sum(new[:r + 1]) - 1                              # the row's last token, whose value is NaN
    poison(c, r, c.N[r] - 1, 1, v=float("nan"))
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    assert torch.isnan(got[t, 4:8]).any(-1).all()
    got[t, 4:8] = want[t, 4:8].to(got.dtype)
    check(got, want, f"window of {rows} rows, a value unseen")


@pytest.mark.parametrize("rows", [1, 40, 150, 300])
@pytest.mark.parametrize("layer", ["window", "slide", "pages"])
def test_one_token_per_row(hip, rows, layer):
    """Layers without sub-blocks whose rows bring one token each, or none: tiles of 4, with four, two and one waves."""
    rng = random.Random(rows)
    new = [1 if rows < 3 or i % 7 else 0 for i in range(rows)]
    prev = [rng.choice([0, 1, 3, 4, 255, 256, 259, rng.randint(0, 700)]) for _ in range(rows)]
    if layer == "pages":
        c = ref.Cache(hip, prev, new, ebs=64, flushed=[0] * rows, seed=82)
    else:
        c = ref.Cache(hip, prev, new, ebs=40, win=256, sinks=layer == "window", rot=layer == "window", seed=82)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"one token of {rows} rows, {layer}")


# ---------------------------------------------------------------- verification
def same(case):
    T, V = case[0].shape
    assert T * -(-V // 2048) > 9216                       # pieces of 8,192
    assert run_verify(*case) == ref.verify(*case)


@pytest.mark.parametrize("V,new", [(65536, [5, 1, 0, 5, 9, 2, 7, 4] * 9), (65536, [300]), (70001, [1] * 270), (24576, [3] * 260),
                                   (8193, [2, 9, 40, 1] * 36)])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_pieces(hip, V, new, probs):
    same(verify_case(new, V, V + len(new), probs, (0.8, 1.0, 0.0, 1.3), pad=3))


@pytest.mark.parametrize("V,new", [(65536, [5, 0, 3] * 35), (20001, [4] * 230)])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_many_small_pieces(hip, V, new, probs):
    case = verify_case(new, V, V + len(new), probs, (0.8, 1.0, 0.0, 1.3), pad=3)
    assert 8000 < case[0].shape[0] * -(-V // 2048) <= 9760     # about the border of the two sizes
    assert run_verify(*case) == ref.verify(*case)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_pieces_borders(hip, probs):
    x, tokens, qsl, temp, u, un, q = verify_case([4] * 240, 20001, 3, probs, (1.0, 0.7))
    for a, b in ((0.0, 0.0), (1 - 2 ** -24, 1 - 2 ** -24), (0.5, 0.0)):
        same((x, tokens, qsl, temp, torch.full_like(u, a), torch.full_like(un, b), q))
    x[:480] = 1.5                                         # equal logits
    temp = torch.tensor([1.0, 0.0, 0.5, float("nan"), float("inf"), -1.0, 1e-30] * 35)[:240]
    tokens[5], tokens[9], tokens[14], tokens[18] = -1, 20001, 1 << 40, 20000
    same((x, tokens, qsl, temp, u, un, q))


@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_pieces_extreme_temperatures(hip, probs):
    temps = (1e-3, 1e-8, 1e-12, 1e-16, 1e-25, 1e-30, 1e-45, 1e3, 1e20, 1e30)
    V = 20001
    x, tokens, qsl, temp, u, un, q = verify_case([4] * 240, V, 12, probs, temps)
    x[::2, 5::V // 3] = x.max(-1, keepdim=True).values[::2]
    x[1::4, 9] = -torch.finfo(torch.bfloat16).max
    near = torch.randint(0, 3, (960,), generator=torch.Generator().manual_seed(5)) * (V // 3) + 5
    tokens = torch.where(torch.rand(960, generator=torch.Generator().manual_seed(6)) < 0.4, near, tokens)
    same((x, tokens, qsl, temp, u, un, q))


@pytest.mark.parametrize("probs", [False, True])
def test_verify_large_pieces_infinities_and_nan(hip, probs):
    V = 60001
    x, tokens, qsl, temp, u, un, q = verify_case([5] * 64, V, 4, probs, (1.0, 0.7))
    x[:, 100:50000] = float("-inf")                       # whole pieces without a token
    x[5:10, :50] = torch.finfo(torch.bfloat16).min
    x[10:15, 40000] = float("inf")
    x[12, 30000] = float("nan")
    x[16, V - 1] = float("nan")
    x[21] = float("-inf")
    x[25:30, :V - 3] = float("-inf")                      # the last three alone
    if probs:
        q[30:35, 55000:] = float("nan")
        q[35:40] = 2.0                                    # above p everywhere
    same((x, tokens, qsl, temp, u, un, q))


def test_verify_large_pieces_strides(hip):
    from lfm3_kv800_amd import spec_ops as so
    V, new = 20001, [3] * 320
    x, tokens, qsl, temp, u, un, q = verify_case(new, V, 9, True, (1.0, 0.0))
    want = ref.verify(x, tokens, qsl, temp, u, un, q)
    d = [t.cuda() for t in (tokens, torch.tensor(qsl), temp, u, un)]
    for at, width in ((1, V + 2), (8, V + 15), (5, V + 5)):
        wide = torch.full((960, width), float("nan"), dtype=torch.bfloat16).cuda()
        wide[:, at:at + V] = x.cuda()
        qw = torch.full((960, width + 4), float("nan")).cuda()
        qw[:, 4:4 + V] = q.cuda()
        out, count = so.verify_drafts(wide[:, at:at + V], *d, qw[:, 4:4 + V])
        assert (out.tolist(), count.tolist()) == want, at
