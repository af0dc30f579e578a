"""PagedAttention8's room for steps that are recorded once and replayed: as many as the caches hold, the next one refused before anything
moves on."""
import pytest
import torch

from lfm3_kv800_amd import model as M


def attention(steps):
    return M.PagedAttention8([5, 9], steps, "cpu", bs=64)


class Untouched:
    """A model that no step may reach."""
    def step(self, *a, **k):
        pytest.fail("a step ran")

    greedy = step


def test_freeze_refuses_steps_without_room():
    attn = attention(3)                                    # room for 4: nmax counts one more
    left = attn.nmax - 9
    with pytest.raises(ValueError, match="positions"):
        attn.freeze(left + 1)
    assert attn.lens_dev is None and attn.lens.tolist() == [5, 9]
    attn.freeze(left)
    assert attn.lens_dev.tolist() == [5, 9]


def test_recorded_loop_refuses_before_its_first_step():
    attn = attention(3)
    left = attn.nmax - 9
    with pytest.raises(ValueError, match="positions"):
        M.decode_loop(Untouched(), attn, torch.zeros(2, dtype=torch.int64), left + 1, graph=True)
    with pytest.raises(ValueError, match="positions"):
        M.DecodeGraph(Untouched(), attn, torch.zeros(2, dtype=torch.int64), left)      # its first step is one more
    assert attn.lens.tolist() == [5, 9] and attn.lens_dev is None


def build(steps):
    attn = M.PagedAttention8([70, 126], steps, "cuda", seed=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    bank = torch.randn(2, 200, 4, 128, generator=g, device="cuda").to(torch.bfloat16)
    attn.fill(lambda l, r, p0, p1: (bank[0, p0:p1], bank[1, p0:p1]))
    return M.Lfm3Decoder(M.Lfm3Config(layers=5, vocab=512), attn, 2, "cuda", seed=3), attn


@pytest.mark.gpu
@pytest.mark.parametrize("provided", [0, 4])
def test_loops_to_the_last_position(hip, provided):
    """The recorded loop takes the last position that the caches hold, as the eager one does, and neither takes one more."""
    tok = torch.tensor([3, 4], device="cuda")
    model, attn = build(provided)
    steps = attn.nmax - 126
    want = M.decode_loop(model, attn, tok, steps)
    with pytest.raises(ValueError):
        attn.begin_step()
    model, attn = build(provided)
    with pytest.raises(ValueError):
        M.decode_loop(model, attn, tok, steps + 1, graph=True)
    assert torch.equal(M.decode_loop(model, attn, tok, steps, graph=True), want)
    assert attn.lens.tolist() == [70 + steps, 126 + steps]
    with pytest.raises(ValueError):
        attn.begin_step()
    attn.thaw()
    with pytest.raises(ValueError):
        attn.begin_step()
