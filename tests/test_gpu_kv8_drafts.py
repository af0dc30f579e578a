"""Drafts that are taken back from the 8-bit cache: what they leave of their block's other tokens, and the tokens of a loop with them."""
import pytest
import torch

import kv8_reference as ref
from test_gpu_kv8 import DEV, kv8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("larger", [0, 1, 3, 7])
def test_what_a_draft_leaves(kv8, larger):
    """40 tokens, a draft 2^larger times as large, taken back, 20 more tokens: magnitudes from 2^-6 of the grown exponent on are held as
    without the draft, smaller ones within half a step of the least code there, 2^-10 of it."""
    g = torch.Generator().manual_seed(larger)
    x = torch.randn(61, 4, 64, generator=g).clamp(-3.4, 3.4).to(torch.bfloat16)
    x[0, :, 0] = 3.4375                                                   # the largest of every head's keys and values
    draft = x[:1] * 2.0 ** larger
    i64 = lambda *a: torch.tensor(a, dtype=torch.int64, device=DEV)
    bt = torch.zeros(1, 1, dtype=torch.int32, device=DEV)

    def held(drafts):
        c = kv8.Cache8.empty(1, 2, 64, 64, DEV)
        put = lambda t, n: kv8.append(c, t[:, :2].to(DEV), t[:, 2:].to(DEV), bt, i64(n), i64(0, len(t)))
        put(x[:40], 40)
        if drafts:
            put(draft, 41)
        put(x[40:60], 60)
        return c.exps.cpu(), [t.cpu().double()[0, :, :60] for t in kv8.dequantize(c)]

    (e0, plain), (e1, after) = held(False), held(True)
    assert (e1.int() - e0.int() == larger).all()
    top = 2.0 ** (int(e1[0, 0, 0, 0]) - 127)
    for a, b in zip(plain, after):
        fine = a.abs() >= 2.0 ** -6 * top
        assert torch.equal(a[fine], b[fine])
        assert ((a - b).abs()[~fine] <= 2.0 ** -10 * top * (1 + 2.0 ** -8)).all()


def test_tokens_of_a_loop_with_drafts(hip):
    """Tokens of speculative_loop over the 8-bit cache, a row whose drafts are the one-token loop's and one whose drafts are random, are
    the one-token loop's choices up to near-ties: fed the same tokens, its logit of each is within what its sub-layers' roundings
    leave (a relative 6e-2 of the logits, as test_model_follows_plain_forms, here at five times their spread and for both of the
    compared logits). bf16 products: of 8-bit ones a rounding may move a code by a whole step, which that figure does not hold."""
    from lfm3_kv800_amd import model as M
    from test_gpu_model8 import build
    lens0, n, most = [700, 65], 6, 3
    start = torch.tensor([11, 22], device=DEV)
    make = lambda: build(lens0, n * (most + 1) + 2, int8=False)
    truth = M.decode_loop(*make(), start, n * (most + 1) + 1)                  # (steps, 2)
    g = torch.Generator(device=DEV).manual_seed(1)

    def draft(last, lens):
        at = (lens[0] - lens0[0]) + torch.arange(most, device=DEV)
        d = torch.randint(0, 8192, (2, most), generator=g, device=DEV)
        d[0] = truth[at.clamp(max=truth.shape[0] - 1), 0]
        return d, torch.full((2,), most, dtype=torch.int32, device=DEV), None

    rows, kept = M.speculative_loop(*make(), start, n, draft, most)
    print("kept", kept.tolist(), "one-token", truth[:, 0].tolist(), "with drafts", rows[0].tolist(), flush=True)
    assert [len(r) for r in rows] == kept.sum(0).tolist()
    model, attn = make()
    tok, worst = start, 0.0
    for i in range(max(len(r) for r in rows)):
        logits = model.step(tok, attn.begin_step())
        for r, got in enumerate(rows):
            if i < len(got):
                short = float(logits[r].max() - logits[r, got[i]]) / float(logits[r].std())
                worst = max(worst, short)
                assert short <= 2 * 5 * 6e-2, (i, r, short)
        tok = torch.stack([r[min(i, len(r) - 1)] for r in rows])
    print("furthest below the largest logit, in their spread", round(worst, 3), flush=True)
