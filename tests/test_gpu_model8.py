"""The engine loop in 8 bits: PagedAttention8's steps (prompts, drafts that are taken back, single tokens) against plain 64-bit forms
of the cache and the attention, the model with int8 weights against the same model on plain forms of its 8-bit operators, recorded
steps against eager ones."""
import pytest
import torch

import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def say(*a):
    print("[model8]", *a, flush=True)


def noise(n, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(2, n, 4, 128, generator=g, device=DEV).to(torch.bfloat16)


def rows_from(bank):
    return lambda l, r, p0, p1: tuple(bank[i, p0 + (r + l) % 64:p1 + (r + l) % 64] for i in range(2))


def test_steps_together(hip):
    """A full and a sliding layer through a history (the sliding ring goes round), prompt chunks, drafts, a retreat and single
    tokens: every step's cache bytes and outputs."""
    from lfm3_kv800_amd import model as M
    lens0, R = [2600, 40], 2
    attn = M.PagedAttention8(lens0, 500, DEV, seed=1)
    attn.kind = {l: attn.kind[l] for l in (2, 4)}
    assert attn.kind == {2: M.FULL, 4: M.SLIDE} and attn.ring < attn.bt[M.SLIDE].shape[1]
    cpu = {l: (attn.layers[l].data.cpu(), attn.layers[l].exps.cpu()) for l in attn.kind}
    bts = {t: b.cpu() for t, b in attn.bt.items()}
    tabs = {M.FULL: tuple(t.cpu() for t in attn.tables[M.FULL]), M.SLIDE: tuple(t.cpu() for t in attn.tables[M.SLIDE])}
    bank = noise(2800, 3)
    history = rows_from(bank)
    attn.fill(history)
    for c0 in (0, 2048):
        n = [min(x, c0 + 2048) for x in lens0]
        new = [max(0, x - c0) for x in n]
        qsl = torch.tensor([0, new[0], new[0] + new[1]])
        for l, t in attn.kind.items():
            K, V = (torch.cat([history(l, r, c0, c0 + c)[i].cpu() for r, c in enumerate(new) if c]) for i in (0, 1))
            cpu[l] = ref.append(*cpu[l], K, V, bts[t], torch.tensor(n), qsl, *(tabs[t] if t == M.FULL else (None, None)))
    lens = torch.tensor(lens0)
    g = torch.Generator().manual_seed(5)
    # (tokens a row, tokens taken back afterwards)
    for new, back in (([70, 33], [0, 0]), ([5, 3], [3, 1]), ([2, 5], [1, 4]), ([1, 1], [0, 0]), ([1, 200], [0, 0]), ([1, 1], [0, 0])):
        ql = torch.tensor(new)
        lens = lens + ql
        T = int(ql.sum()) + 2
        q, k, v = (torch.randn(T, h, 128, generator=g).to(torch.bfloat16) for h in (16, 4, 4))
        k = (k.float() * torch.pow(2.0, torch.randint(-2, 3, (T, 1, 1), generator=g))).to(torch.bfloat16)
        m = attn.begin_chunk(lens.to(DEV), ql.to(torch.int32).to(DEV), T, max(new), lens)
        for l, t in attn.kind.items():
            out = attn.attend(l, q.to(DEV), k.to(DEV), None, v.to(DEV)).cpu().double()
            qsl = m.qsl.cpu()
            cpu[l] = ref.append(*cpu[l], k, v, bts[t], lens, qsl, *tabs[t])
            assert torch.equal(attn.layers[l].exps.cpu(), cpu[l][1]) and torch.equal(attn.layers[l].data.cpu(), cpu[l][0]), (l, new)
            want, far = ref.attend(*cpu[l], q, bts[t], lens, qsl, window=256 if t == M.SLIDE else 0)
            worst = float(((out - want).abs() / far.clamp(min=1e-30)).max())
            say("layer", l, "new", new, "worst error over its bound", round(worst, 3))
            assert worst <= 1.0
        lens = lens - torch.tensor(back)


def build(lens0, steps, layers=8, int8=True, seed=3):
    from lfm3_kv800_amd import model as M
    attn = M.PagedAttention8(lens0, steps, DEV, seed=seed)
    attn.fill(rows_from(noise(max(lens0) + 64, seed)))
    model = M.Lfm3Decoder(M.Lfm3Config(layers=layers, vocab=8192), attn, len(lens0), DEV, seed=seed + 1, int8=int8)
    model.randomize_conv_states(seed + 2)
    return model, attn


def test_model_follows_plain_forms(hip, monkeypatch):
    """Logits of the 8-bit model, single tokens and a chunk, against the same model whose products, appends and attention are the
    plain forms. Every sub-layer's output may differ by a few bf16 roundings (2^-8 each): the 16 sub-layers' four each add up, as their
    squares do, to 8 x 2^-8 = 3 %, twice that with the LM head's and the tokens' rounding to 8 bits behind each difference."""
    from lfm3_kv800_amd import int8_ops as i8, kv8, model as M
    lens0, steps, n = [700, 65, 3], 3, 5

    class Kept(i8.Weight8):
        def __init__(self, w, scale=None, gated=False):
            self.codes, self.rows = i8.quantize_rows(w)
            super().__init__(self.codes, self.rows, gated)

    def linear8(x, w):
        t = x.float().abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
        y = ((x.float() * (torch.full_like(t, 127) / t)).round() @ w.codes.float().T.contiguous()) * (t / 127) * w.rows
        if w.gated:
            a, b = y.chunk(2, 1)
            y = a * torch.sigmoid(a) * b
        return y.to(torch.bfloat16)

    def append(c, k, v, bt, lens, qsl, cos=None, sin=None):
        d, e = ref.append(c.data.cpu(), c.exps.cpu(), k.cpu(), v.cpu(), bt.cpu(), lens.cpu(), qsl.cpu(), cos.cpu(), sin.cpu())
        c.data.copy_(d)
        c.exps.copy_(e)

    def attend(c, q, bt, lens, qsl, window=0, scale=None):
        return ref.attend(c.data.cpu(), c.exps.cpu(), q.cpu(), bt.cpu(), lens.cpu(), qsl.cpu(), window)[0].to(torch.bfloat16).to(DEV)

    got = []
    model, attn = build(lens0, steps + n)
    tok = torch.tensor([5, 6, 7], device=DEV)
    toks = []
    for s in range(steps):
        toks.append(tok)
        got.append(model.step(tok, attn.begin_step()))
        tok = got[-1].argmax(-1)
    more = torch.randint(0, 8192, (3 * n,), generator=torch.Generator().manual_seed(2)).to(DEV)
    lens = torch.tensor(lens0) + steps + n

    def chunk(model, attn):            # five more tokens a row at once
        m = attn.begin_chunk(lens.to(DEV), torch.full((3,), n, dtype=torch.int32, device=DEV), 3 * n, n, lens)
        return model.chunk(more, m).float()

    got.append(chunk(model, attn))
    monkeypatch.setattr(M.i8, "Weight8", Kept)
    plain, pattn = build(lens0, steps + n)
    monkeypatch.setattr(M.i8, "linear8", linear8)
    monkeypatch.setattr(M.kv8, "append", append)
    monkeypatch.setattr(M.kv8, "attend", attend)
    for s in range(steps + 1):
        want = plain.step(toks[s], pattn.begin_step()) if s < steps else chunk(plain, pattn)
        rel = float((got[s] - want).norm() / want.norm())
        say("step", s, "logits rel-L2", rel)
        assert torch.isfinite(got[s]).all() and rel < 6e-2


def test_replays_match_eager(hip):
    """Steps replayed from one recorded step against the same steps from the host, with eager work in between: equal bits."""
    from lfm3_kv800_amd import model as M, model_ops as mo
    lens0, steps = [1405, 126, 63], 5
    tok0 = torch.tensor([11, 22, 33], device=DEV)
    model, attn = build(lens0, steps)
    want, tok = [], tok0
    for s in range(steps):
        logits = model.step(tok, attn.begin_step(), fp32=False)
        tok = mo.argmax(logits)
        want.append((tok.clone(), logits.clone()))
    model, attn = build(lens0, steps)
    dg = M.DecodeGraph(model, attn, tok0, steps - 1)
    got = [(dg.tokens.clone(), dg.first_logits.clone())]
    junk = torch.randn(512, 512, device=DEV)
    for s in range(1, steps):
        dg.step()
        got.append((dg.tokens.clone(), dg.logits.clone()))
        junk = (junk @ junk.t()).tanh()
        torch.cuda.synchronize()
    for s, ((tw, lw), (tg, lg)) in enumerate(zip(want, got)):
        assert torch.equal(tw, tg) and torch.equal(lw, lg), s


def test_loops_run(hip):
    """A whole prompt, then the loop with drafts and the recorded loop on the same caches."""
    from lfm3_kv800_amd import model as M
    model, attn = build([1, 1], 400)
    n = torch.tensor([300, 77])
    toks = torch.randint(0, 8192, (int(n.sum()),), generator=torch.Generator().manual_seed(4)).to(DEV)
    lens = torch.tensor([1, 1]) + n
    m = attn.begin_chunk(lens.to(DEV), n.to(torch.int32).to(DEV), len(toks), 300, lens)
    logits = model.chunk(toks, m)
    model.commit(n.to(torch.int32).to(DEV))
    attn.lens = lens
    last = logits[m.qsl[1:] - 1].float().argmax(-1)
    assert torch.isfinite(logits.float()).all()

    def draft(last, lens):
        return torch.randint(0, 8192, (2, 3), device=DEV), torch.tensor([3, 1], dtype=torch.int32, device=DEV), None

    rows, kept = M.speculative_loop(model, attn, last, 4, draft, 3)
    assert [len(r) for r in rows] == kept.sum(0).tolist() and bool((kept >= 1).all()) and bool((kept <= torch.tensor([4, 2], device=DEV)).all())
    assert attn.lens.tolist() == (lens + kept.sum(0).cpu()).tolist()
    out = M.decode_loop(model, attn, torch.stack([r[-1] for r in rows]), 4, graph=True)
    assert out.shape == (4, 2) and bool(((out >= 0) & (out < 8192)).all())
    with pytest.raises(ValueError):
        attn.begin_chunk(lens.to(DEV), torch.ones(2, dtype=torch.int32, device=DEV), 2, 1, torch.tensor([10 ** 6, 1]))
    with pytest.raises(ValueError):
        attn.begin_chunk(lens.to(DEV), torch.ones(2, dtype=torch.int32, device=DEV), 2, 4096, lens)
