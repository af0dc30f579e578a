"""Steps with several new tokens per row through the layers and the engine loop: chunk_step_meta, the layers' chunk step and
speculative_loop against the one-token decode of the same model, whose every step is held to the oracle elsewhere."""
import pytest
import torch

import chunk_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def say(*a):
    print("[speculative]", *a, flush=True)


def build(lens0, steps, layers=8, seed=3):
    from lfm3_kv800_amd import model as M
    g = torch.Generator(device=DEV).manual_seed(seed)
    noise = (torch.randn(2, max(lens0) + 64, 4, 128, generator=g, device=DEV)).to(torch.bfloat16)
    attn = M.PagedAttention800(lens0, steps, DEV, seed=seed)
    attn.fill(lambda l, r, p0, p1: tuple(noise[i, p0 + (r + l) % 64:p1 + (r + l) % 64] for i in range(2)))
    model = M.Lfm3Decoder(M.Lfm3Config(layers=layers, vocab=8192), attn, len(lens0), DEV, seed=seed + 1)
    model.randomize_conv_states(seed + 2)
    return model, attn


@pytest.mark.parametrize("lens0", [[1405, 700, 380, 3], [1406, 640, 1919, 383]])
def test_chunks_follow_the_decode(hip, lens0):
    """The one-token decode's tokens as drafts, some of them replaced: logits agree with the decode's at every position up to
    the layers' bf16 rounding, a true draft is kept and a replaced one is not, unless the two logits are tied
    within the models' own difference; the states and caches behind a rejection are those of the kept tokens. Rows cross
    flush boundaries (384, 1408, 1920). Where a token inside a chunk is the one that makes a block eligible, the decode reads
    that block quantized and the chunk, as extend rows do, its exact rows: from there on the row's values are others, and it
    is compared no further."""
    from lfm3_kv800_amd import model as M, spec_ops as so
    most, steps = 4, 6
    R, n = len(lens0), steps * (most + 1)
    model, attn = build(lens0, n)
    first = torch.tensor([5, 6, 7, 8], device=DEV)
    states = [L["state"].clone() for L in model.layers if L["type"] == M.CONV]
    true, want = [first], []
    for _ in range(n):
        want.append(model.step(true[-1], attn.begin_step()))
        true.append(want[-1].argmax(-1))
    true, want = torch.stack(true, 1), torch.stack(want, 1)        # (R, n + 1) tokens; (R, n, vocab) logits behind them

    chunked, attn2 = build(lens0, n)
    for L, s in zip((L for L in chunked.layers if L["type"] == M.CONV), states):
        assert torch.equal(L["state"], s)
    rng = torch.Generator().manual_seed(1)
    at = torch.zeros(R, dtype=torch.int64)                          # tokens taken so far
    last, worst, kept_all, compared, alike = first, 0.0, [], 0, [True] * R
    for step in range(steps):
        nd = torch.tensor([(step + r) % (most + 1) for r in range(R)])
        bad = torch.rand(R, most, generator=rng) < 0.25
        drafts = torch.stack([true[r, at[r] + 1:at[r] + 1 + most] for r in range(R)])
        drafts = torch.where(bad.to(DEV), (drafts + 17) % 8192, drafts)
        ql = (nd + 1).to(torch.int32).to(DEV)
        lens = (torch.tensor(lens0) + at).to(DEV) + ql
        m = attn2.begin_chunk(lens, ql, R * (most + 1), most + 1, lens.cpu())
        i = (torch.arange(R * (most + 1), device=DEV) - m.qsl[m.row]).clamp(max=most)
        tok = torch.cat((last[:, None], drafts), 1)[m.row, i]
        logits = chunked.chunk(tok, m)
        out, kept = so.verify_drafts(logits, tok, m.qsl, torch.zeros(R, device=DEV), torch.rand(R * (most + 1), device=DEV),
                                     torch.rand(R, device=DEV))
        qsl, kept_l = m.qsl.tolist(), kept.tolist()
        for r in range(R):
            for i in range(qsl[r + 1] - qsl[r]):
                prev = lens0[r] + int(at[r])
                if ref.nq(prev + i + 1) != ref.nq(prev + 1):
                    alike[r] = False
                if bad[r, :i].any() or not alike[r]:
                    break                                          # behind a replaced draft the decode knows nothing
                compared += 1
                a, b = logits[qsl[r] + i].float(), want[r, at[r] + i]
                d = float((a - b).norm() / b.norm())
                worst = max(worst, d)
                assert d < 1e-1, (step, r, i, d)
                tie = 2 * float((a - b).abs().max())
                top = float(b.max())
                if i < qsl[r + 1] - qsl[r] - 1:
                    x = int(tok[qsl[r] + i + 1])
                    if kept_l[r] > i + 1:
                        assert top - float(b[x]) <= tie
                    elif kept_l[r] == i + 1:
                        second = float(b.topk(2).values[1])
                        assert bool(bad[r, i]) or top - second <= tie
        took = [qsl[r] + k - 1 for r, k in enumerate(kept_l)]
        new = out[torch.tensor(took, device=DEV)]
        # go on from the decode's own tokens: what it took is the truth, or tied with it
        for r in range(R):
            good = 1
            while good < (kept_l[r] if alike[r] else qsl[r + 1] - qsl[r]) and not bad[r, good - 1]:
                good += 1
            kept_l[r] = good
        chunked.commit(torch.tensor(kept_l, dtype=torch.int32, device=DEV))
        at += torch.tensor(kept_l)
        last = torch.stack([true[r, at[r]] for r in range(R)])
        kept_all.append(kept_l)
        assert new.shape == (R,)
    say("logits' worst rel-L2", f"{worst:.2e}", "kept", kept_all)
    assert sum(map(sum, kept_all)) > R * steps and compared > R * steps // 2


@pytest.mark.parametrize("sampled", [False, True])
def test_speculative_loop(hip, sampled):
    """The loop runs, keeps drafts that the model proposes itself, and its lengths, counts and tokens agree; greedy tokens are
    those of the one-token loop up to the first tie (a token whose logit there is within the models' difference)."""
    from lfm3_kv800_amd import model as M
    lens0, most, steps = [500, 129, 1020], 3, 5
    R = len(lens0)
    n = steps * (most + 1)
    model, attn = build(lens0, n)
    first = torch.tensor([1, 2, 3], device=DEV)
    true = [first] + list(M.decode_loop(model, attn, first, n))
    true = torch.stack(true, 1)
    model, attn = build(lens0, n)
    start = attn.lens.to(DEV)

    def draft(last, lens):
        i = (lens - start)[:, None] + 1 + torch.arange(most, device=DEV)
        d = true.gather(1, i.clamp(max=n))
        if not sampled:
            return d, torch.full((R,), most, dtype=torch.int32, device=DEV), None
        q = torch.full((R, most, 8192), 0.1 / 8192, device=DEV)
        q.scatter_(2, d[..., None], 0.9 + 0.1 / 8192)
        return d, torch.tensor([most, 0, 1], dtype=torch.int32, device=DEV), q

    temp = torch.tensor([1e-3, 0.8, 0.0], device=DEV) if sampled else None
    rows, counts = M.speculative_loop(model, attn, first, steps, draft, most, temp, torch.Generator(device=DEV).manual_seed(4))
    assert counts.shape == (steps, R) and [len(t) for t in rows] == counts.sum(0).tolist()
    assert attn.lens.tolist() == [a + b for a, b in zip(lens0, counts.sum(0).tolist())]
    assert int(counts.min()) >= 1 and int(counts.max()) <= most + 1
    say("counts", counts.tolist())
    if sampled:
        assert counts[:, 1].tolist() == [1] * steps
    else:
        same = [int((t == true[r, 1:1 + len(t)]).long().cumprod(0).sum()) for r, t in enumerate(rows)]
        say("as the one-token loop for", same, "of", [len(t) for t in rows])
        assert sum(same) > R * steps                                # more than one token a step: drafts are kept


def test_a_whole_step_in_a_graph(hip):
    """Metadata, layers, verification, commit and lengths in one captured step, replayed: each replay does what the eager step
    does from the same state."""
    from lfm3_kv800_amd import spec_ops as so
    lens0, most, steps = [900, 300], 2, 5
    R, T, n = 2, 6, 15
    first = torch.tensor([3, 4], device=DEV)

    def step(model, attn, s):
        ql = torch.full((R,), most + 1, dtype=torch.int32, device=DEV)
        m = attn.begin_chunk(s["lens"] + ql, ql, T, most + 1, torch.tensor(lens0) + n)
        tok = torch.cat((s["last"][:, None], s["last"][:, None] + 1, s["last"][:, None] + 2), 1).flatten() % 8192
        logits = model.chunk(tok, m)
        out, kept = so.verify_drafts(logits, tok, m.qsl, s["temp"], s["u"], s["un"])
        model.commit(kept)
        s["lens"] += kept
        s["last"].copy_(out[m.qsl[:-1] + kept - 1])
        s["out"].copy_(out)

    def state():
        g = torch.Generator(device=DEV).manual_seed(2)
        return {"lens": torch.tensor(lens0, device=DEV), "last": first.clone(), "temp": torch.full((R,), 30.0, device=DEV),
                "u": torch.rand(T, device=DEV, generator=g), "un": torch.rand(R, device=DEV, generator=g),
                "out": torch.zeros(T, dtype=torch.int64, device=DEV)}
    want, s = [], state()
    model, attn = build(lens0, n)
    for _ in range(steps):
        step(model, attn, s)
        want.append((s["out"].tolist(), s["lens"].tolist()))
    model, attn = build(lens0, n)
    s = state()
    step(model, attn, s)                                            # eager: tables, library handles
    assert (s["out"].tolist(), s["lens"].tolist()) == want[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(model, attn, s)
    other, oattn = build([40, 50], 8)
    for k in range(1, steps):
        g.replay()
        other.step(first, oattn.begin_step())                       # eager work of another model in between
        torch.cuda.synchronize()
        assert (s["out"].tolist(), s["lens"].tolist()) == want[k], k


def test_chunk_step_refusals(hip):
    from lfm3_kv800_amd import model as M, vllm_cache as vc
    model, attn = build([100, 20], 8)
    ql = torch.ones(2, dtype=torch.int32, device=DEV)
    lens = attn.lens.to(DEV) + 1
    with pytest.raises(ValueError):
        attn.begin_chunk(lens, ql, 4, 2, torch.tensor([200, 30]))          # past the caches
    with pytest.raises(ValueError):
        vc.chunk_step_meta(attn.qbt, lens, ql, vc.QBLOCK, 4, 0, [101, 21])
    with pytest.raises(ValueError):
        vc.chunk_step_meta(attn.qbt, lens, ql, vc.QBLOCK, 4, 1, [101])
    with pytest.raises(ValueError):
        M.speculative_loop(model, attn, torch.tensor([1, 2], device=DEV), 1, None, 128)
    rows, counts = M.speculative_loop(model, attn, torch.tensor([1, 2], device=DEV), 0, None, 3)
    assert [len(t) for t in rows] == [0, 0] and counts.shape == (0, 2)


def test_speculative_loop_without_drafts(hip):
    """most = 0, with and without (empty) distributions: the one-token loop. Draft counts past `most` count as `most`."""
    from lfm3_kv800_amd import model as M
    first = torch.tensor([1, 2], device=DEV)
    empty = torch.zeros(2, 0, dtype=torch.int64, device=DEV)
    runs = []
    for probs in (None, torch.zeros(2, 0, 8192, device=DEV)):
        model, attn = build([300, 20], 8)
        rows, counts = M.speculative_loop(model, attn, first, 4, lambda last, lens: (empty, torch.full((2,), 7, device=DEV), probs), 0)
        assert counts.tolist() == [[1, 1]] * 4 and attn.lens.tolist() == [304, 24]
        runs.append(torch.stack(rows).tolist())
    assert runs[0] == runs[1]
