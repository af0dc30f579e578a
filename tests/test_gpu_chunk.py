"""Operators of a step whose rows bring several new tokens each, on the GPU, against the references in 64 bits of
chunk_reference.py: attention over the paged cache, slots and block tables, short conv, verification of drafts.

Attention's tolerance, per (token, head) vector of 128: its own rounding to bf16 is at most 2^-8 of every element, so of the
vector's length; weights of quantized blocks are rounded to 11 bits (2^-12 of each, in the root of the sum of their squares,
as the vector's length itself), which is 2^-12 of it, doubled for the scales' spread and the 16-bit weights of exact rows;
the fp32 sums are far below. A rotated key within an fp32 ulp of a bf16 boundary may fall on its other side: 2^-8 of one of
128 elements of some keys, below 2^-11 of the vector. In all 2^-8 + 2^-11 + 2^-11."""
import pytest
import torch

import chunk_reference as ref

pytestmark = pytest.mark.gpu
VEC = 2 ** -8 + 2 ** -10


def check(got, want, what):
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    d = (got.double() - want).norm(dim=-1)
    bound = VEC * want.norm(dim=-1) + 1e-30
    worst = float((d / bound).max()) if d.numel() else 0.0
    print(f"[chunk] {what}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, (what, worst)


ROWS = {   # history and new tokens of the rows
    "one": ([5], [1]),
    "first": ([0], [1]),
    "edges": ([0, 1, 127, 128, 383, 384, 385, 639, 640], [4, 1, 3, 4, 2, 1, 4, 4, 3]),
    "empty rows": ([0, 500, 7, 900, 0, 40], [0, 3, 0, 4, 2, 0]),
    "odd": ([700, 1500, 33, 2050], [7, 5, 13, 6]),
    "chunk": ([390, 0, 1029], [33, 65, 17]),
    "more rows than a wave": ([(37 * i) % 900 for i in range(130)], [(i * 7) % 6 for i in range(130)]),
}


@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("ebs,token_major", [(64, False), (24, True)])
def test_quantized(hip, rows, ebs, token_major):
    c = ref.Cache(hip, *ROWS[rows], ebs=ebs, token_major=token_major, seed=len(rows))
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"quantized {rows} ebs {ebs}")


@pytest.mark.parametrize("rows", ["one", "edges", "empty rows", "more rows than a wave", "rows of one wave each"])
def test_quantized_in_two_launches(hip, rows):
    """Tiles of 4 under a bound on the blocks that allows long lists: the two parts have a launch each."""
    prev, new = ROWS.get(rows) or ([(53 * i) % 1100 for i in range(300)], [i % 5 for i in range(300)])
    c = ref.Cache(hip, prev, new, ebs=40, seed=len(rows))
    c.P.nqmax = 8 * torch.cuda.get_device_properties(0).multi_processor_count // len(prev) + 1
    want = c.want(hip)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, f"two launches {rows}")
    r = next(i for i, n in enumerate(new) if n)
    t = sum(new[:r + 1]) - 1                             # the row's last token, whose value is NaN
    poison(c, r, c.N[r] - 1, 2, v=float("nan"))
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    assert torch.isnan(got[t, 8:12]).any(-1).all()
    got[t, 8:12] = want[t, 8:12].to(got.dtype)
    check(got, want, f"two launches {rows}, a value unseen")


@pytest.mark.parametrize("rows", ["odd", "chunk", "edges"])
def test_quantized_part_first(hip, rows):
    """One launch in which the exact part's workgroups come last: a bound that allows more than three entries a workgroup, but
    not the lists that get a launch of their own."""
    c = ref.Cache(hip, *ROWS[rows], ebs=40, seed=len(rows))
    c.P.nqmax = 8 * torch.cuda.get_device_properties(0).multi_processor_count // len(c.N)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"quantized part first {rows}")
    small = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    assert torch.equal(small, hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin))


@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("sinks,rot", [(True, True), (False, False)])
def test_window(hip, rows, sinks, rot):
    prev, new = ROWS[rows]
    prev = prev + [254, 255, 256, 257, 258, 259, 260, 300]
    c = ref.Cache(hip, prev, new + [4, 4, 4, 4, 4, 9, 1, 20], ebs=40, win=256, sinks=sinks, rot=rot, seed=7)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), f"window {rows} sinks {sinks}")


def test_long_window_chunk(hip):
    c = ref.Cache(hip, [0, 700], [900, 301], ebs=128, win=256, sinks=True, seed=3)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), "long chunk over a window")


def test_exact_pages_alone(hip):
    """No sub-blocks at all (nqmax 0): every position from the pages, without a window."""
    c = ref.Cache(hip, [900, 0, 130], [3, 2, 9], flushed=[0, 0, 0], seed=4)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), "exact pages alone")


def test_fewer_and_more_blocks_than_the_rule(hip):
    """Blocks that reach into the new tokens are masked by position; fewer leave the rest to the pages."""
    c = ref.Cache(hip, [600, 1000, 700], [300, 30, 5], flushed=[3, 1, 0], seed=5)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), "blocks past the queries")


def test_long_context(hip):
    c = ref.Cache(hip, [32768, 9000], [5, 3], ebs=128, seed=6)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip), "long context")


def test_padding_strides_and_repeat(hip):
    """Padded tokens give zeros whatever stands in q; q and the tables may be strided views; two calls agree bit for bit."""
    c = ref.Cache(hip, [700, 90], [3, 4], seed=8)
    T = c.q.shape[0]
    wide = torch.full((T + 5, 16, 160), float("nan"), dtype=torch.bfloat16, device=c.dev)
    wide[:T, :, :128] = c.q
    c.P.boff = torch.cat([c.P.boff, c.P.boff], 1)[:, :c.P.boff.shape[1]]
    c.P.eoff = torch.cat([c.P.eoff, c.P.eoff], 1)[:, :c.P.eoff.shape[1]]
    got = hip.decode_chunk(c.P, wide[..., :128], c.qsl, c.cos, c.sin)
    check(got[:T], c.want(hip), "padded")
    assert not got[T:].any()
    assert torch.equal(got, hip.decode_chunk(c.P, wide[..., :128], c.qsl, c.cos, c.sin))
    w = ref.Cache(hip, [700, 90], [3, 4], win=256, sinks=True, seed=8)
    q = torch.cat([w.q, torch.full_like(w.q[:2], float("inf"))])
    got = hip.decode_chunk(w.P, q, w.qsl, w.cos, w.sin)
    check(got[:7], w.want(hip), "padded window")
    assert not got[7:].any()


def test_bad_offsets_are_skipped(hip):
    """Blocks and pages outside their pools, and positions past the tables, are left out."""
    c = ref.Cache(hip, [1500, 800], [4, 4], ebs=64, seed=9)
    c.P.boff[0, 2] = -7
    c.P.boff[1, 1] = c.P.qpool.numel() - 51199
    c.P.eoff[0, 1280 // 64 + 1] = -1
    c.P.eoff[1, 512 // 64] = c.P.epool.numel() - 100
    gone = {0: lambda p: ((p >= 512) & (p < 768)) | ((p >= 1344) & (p < 1408)),
            1: lambda p: ((p >= 256) & (p < 512)) | ((p >= 512) & (p < 576))}
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip, lambda r, p: gone[r](p)), "bad offsets")
    short = 1400
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos[:short], c.sin[:short])
    check(got, c.want(hip, lambda r, p: gone[r](p) | (p >= short)), "short rope table")


def poison(c, r, pos, what, k=None, v=None):
    """Exact position `pos` of row r, head `what`: its key and value set to k and v."""
    at = int(c.P.eoff[r, pos // c.P.ebs]) + what * c.P.e_hs + (pos % c.P.ebs) * c.P.e_ts
    flat = c.P.epool.view(-1)
    if k is not None:
        flat[at:at + 128] = k
    if v is not None:
        flat[at + c.P.e_v:at + c.P.e_v + 128:3] = v


@pytest.mark.parametrize("win", [0, 256])
@pytest.mark.parametrize("new", [[1, 3, 4, 2], [1, 9, 12, 35]])
def test_values_that_a_query_does_not_see(hip, win, new):
    """NaN and infinities at positions behind a query, or before its window, do not reach it; queries that see them give NaN or
    infinities in the heads that read them, and nowhere else."""
    c = ref.Cache(hip, [700, 390, 1000, 513], new, ebs=40, win=win, seed=21)
    want, at = c.want(hip), 0
    bad = torch.zeros(sum(new), 16, dtype=torch.bool)
    for r, n in enumerate(new):
        hits = [(c.N[r] - 1, 0, float("nan"), None), (c.N[r] - 1, 1, None, float("inf")), (c.N[r] - n // 2 - 1, 2, None, float("nan")),
                (c.N[r] - 1, 3, float("inf"), float("-inf"))]
        if win:
            hits += [(c.first[r], 0, None, float("inf")), (c.first[r] + n // 2, 2, float("nan"), float("nan"))]
        for pos, h, k, v in hits:
            poison(c, r, pos, h, k, v)
            for i in range(n):
                q = c.prev[r] + i
                if pos <= q and (not win or pos > q - win):
                    bad[at + i, 4 * h:4 * h + 4] = True
        at += n
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    seen = ~torch.isfinite(got).all(-1).cpu()
    assert torch.equal(seen, bad)
    check(got[~bad.to(got.device)], want[~bad.to(got.device)], f"values unseen, window {win}")


def test_scales_that_a_query_does_not_see(hip):
    """Sub-blocks that reach into the new tokens, with NaN scales there."""
    c = ref.Cache(hip, [250, 700], [12, 70], flushed=[1, 3], seed=22)
    want = c.want(hip)
    nan = 0x7F
    VLO, VSC = 256 * 128 + 256 * 64, 256 * 128 + 256 * 64 + 512
    bad = torch.zeros(82, 16, dtype=torch.bool)
    for r, j, t, h, o in ((0, 0, 254, 1, VSC), (1, 2, 740 - 512, 0, VLO), (1, 2, 767 - 512, 3, VSC)):
        block = int(c.P.boff[r, j])
        c.P.qpool.view(-1)[block + o + 2 * t + h // 2] = nan
        first = [0, 12][r]
        for i in range([12, 70][r]):
            if j * 256 + t <= c.prev[r] + i:
                bad[first + i, 8 * (h // 2):8 * (h // 2) + 8] = True
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    assert torch.equal(~torch.isfinite(got).all(-1).cpu(), bad)
    check(got[~bad.to(got.device)], want[~bad.to(got.device)], "scales unseen")


def test_a_query_without_keys(hip):
    c = ref.Cache(hip, [40, 300], [2, 2], seed=10)
    c.P.eoff[0] = -1
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    assert not got[:2].any()
    check(got, c.want(hip, lambda r, p: torch.full_like(p, r == 0, dtype=torch.bool)), "a row without keys")


def test_attention_of_one_token_is_the_decode(hip):
    c = ref.Cache(hip, [700, 1500, 60, 2000], [1, 1, 1, 1], seed=11)
    a = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin).double()
    b = hip.decode(c.P, c.q, c.cos, c.sin).double()
    assert float((a - b).norm(dim=-1).div(b.norm(dim=-1)).max()) <= 2 * VEC


def test_attention_in_a_graph_and_on_another_stream(hip):
    """A captured call on a stream of its own follows new queries and lengths; eager calls in between do not disturb it."""
    c = ref.Cache(hip, [700, 300, 1400], [4, 2, 3], seed=12)
    other = ref.Cache(hip, [100, 900], [3, 4], seed=13)
    st = torch.cuda.Stream()
    hip.rope_pairs(c.cos, c.sin)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        out = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    base = c.q.clone()
    for i in range(3):
        c.q.copy_(base * (1 + i))
        g.replay()
        check(hip.decode_chunk(other.P, other.q, other.qsl, other.cos, other.sin), other.want(hip), "beside a graph")
        torch.cuda.synchronize()
        check(out, c.want(hip), f"replay {i}")
    with torch.cuda.stream(st):
        got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    st.synchronize()
    check(got, c.want(hip), "another stream")


def test_graphs_keep_their_rope_tables(hip):
    """A call captured before its pair table exists makes it on every replay; one captured after keeps the table that it found,
    however many others are made since."""
    c = ref.Cache(hip, [700, 1400], [4, 3], seed=31)
    want = c.want(hip)
    hip.rope_pairs(torch.ones_like(c.cos), c.sin)
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
        graphs.append((g, out))
        hip.rope_pairs(c.cos, c.sin)
    kept = [hip.rope_pairs(torch.rand_like(c.cos), c.sin) for _ in range(12)]
    c.cos.add_(0)                                       # another version: the cached table is made anew
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, "eager after the captures")
    for k in range(3):
        for g, out in graphs:
            out.zero_()
            g.replay()
            kept.append(torch.full((c.cos.shape[0], 32), 0x7FC07FC0, dtype=torch.int32, device=c.dev))
            torch.cuda.synchronize()
            check(out, want, f"replay {k}")


def test_rope_table_of_another_stream(hip):
    """The table is made on one stream behind other work and used on a second at once."""
    c = ref.Cache(hip, [700, 1400], [4, 3], seed=32)
    want, cos = c.want(hip), torch.zeros_like(c.cos)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        x = torch.randn(4096, 4096, device=c.dev)
        for _ in range(20):
            x = x @ x * 1e-2
        cos.copy_(c.cos)
        hip.rope_pairs(cos, c.sin)
        ready = torch.cuda.Event()
        ready.record()
    with torch.cuda.stream(b):
        got = hip.decode_chunk(c.P, c.q, c.qsl, cos, c.sin)
    torch.cuda.synchronize()
    check(got, want, "a table of another stream")


def test_offsets_past_32_bits(hip):
    """Pages and sub-blocks that lie behind the first 2^32 bytes and 2^31 elements of their pools."""
    c = ref.Cache(hip, [700, 1100], [4, 6], ebs=64, seed=33)
    want = c.want(hip)
    old, far = c.P.epool, (1 << 31) + 8 * 1024
    big = torch.empty(far + old.numel(), dtype=torch.bfloat16, device=c.dev)
    big[far:] = old.flatten()
    c.P.epool, c.P.eoff = big, c.P.eoff + far
    oldq, farq = c.P.qpool, (1 << 32) + 51200
    bigq = torch.empty(farq + oldq.numel(), dtype=torch.uint8, device=c.dev)
    bigq[farq:] = oldq.flatten()
    c.P.qpool, c.P.boff = bigq, torch.where(c.P.boff < (1 << 50), c.P.boff + farq, c.P.boff)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, "far offsets")
    w = ref.Cache(hip, [700, 1100], [4, 6], ebs=64, win=256, seed=33)
    want = w.want(hip)
    big[far:far + w.P.epool.numel()] = w.P.epool.flatten()
    w.P.epool, w.P.eoff = big, w.P.eoff + far
    check(hip.decode_chunk(w.P, w.q, w.qsl, w.cos, w.sin), want, "far offsets of a window")


def test_sinks_outside_their_buffers(hip):
    c = ref.Cache(hip, [700, 400], [4, 6], win=256, sinks=True, seed=34)
    c.P.skoff = c.P.skoff.clone()
    c.P.skoff[1] = c.P.sk.numel() - 3 * 512
    got = hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    check(got[:4], c.want(hip)[:4], "sinks in place")
    c.P.skoff[1] = -1
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip, lambda r, p: (p < 4) & (r == 1)), "sinks outside")


def test_strided_lengths_are_refused(hip):
    c = ref.Cache(hip, [700, 90], [3, 4], seed=35)
    for name in ("N", "NQ"):
        keep = getattr(c.P, name)
        setattr(c.P, name, torch.stack([keep, keep], 1)[:, 0])
        with pytest.raises(ValueError):
            hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
        setattr(c.P, name, keep)
    w = ref.Cache(hip, [700, 90], [3, 4], win=256, sinks=True, seed=35)
    w.P.svoff = torch.stack([w.P.svoff, w.P.svoff], 1)[:, 0]
    with pytest.raises(ValueError):
        hip.decode_chunk(w.P, w.q, w.qsl, w.cos, w.sin)


def test_attention_of_nothing(hip):
    c = ref.Cache(hip, [300, 10], [2, 3], seed=14)
    empty = hip.decode_chunk(c.P, c.q[:0], torch.zeros(3, dtype=torch.int64, device=c.dev), c.cos, c.sin)
    assert empty.shape == (0, 16, 128)
    none = hip.decode_chunk(c.P, c.q, torch.zeros(3, dtype=torch.int64, device=c.dev), c.cos, c.sin)
    assert none.shape == c.q.shape and not none.any()


def test_attention_refusals(hip):
    c = ref.Cache(hip, [700, 90], [3, 4], seed=15)
    call = lambda P=c.P, q=c.q, qsl=c.qsl, cos=c.cos, sin=c.sin: hip.decode_chunk(P, q, qsl, cos, sin)
    import copy

    def changed(**k):
        P = copy.copy(c.P)
        for n, v in k.items():
            setattr(P, n, v)
        return P
    for bad, err in ((dict(q=c.q.float()), TypeError), (dict(q=c.q[:, :8]), ValueError), (dict(qsl=c.qsl.int()), TypeError),
                     (dict(qsl=c.qsl.cpu()), ValueError), (dict(cos=None), ValueError), (dict(cos=None, sin=None), ValueError),
                     (dict(sin=c.sin[:5]), ValueError), (dict(qsl=c.qsl.repeat(3)), ValueError),
                     (dict(P=changed(eoff=c.P.eoff[:1])), ValueError),
                     (dict(P=changed(boff=c.P.boff[:1])), ValueError),
                     (dict(P=changed(N=c.P.N.long())), TypeError),
                     (dict(P=changed(e_ts=12)), RuntimeError),
                     (dict(P=changed(ebs=0)), RuntimeError)):
        with pytest.raises(err):
            call(**bad)


# ---------------------------------------------------------------- slots and block tables
TABLES = {
    "one": ([1], [1], 64), "none new": ([0, 5, 0], [0, 0, 0], 64), "pages' ends": ([64, 65, 128, 1, 63], [64, 2, 1, 1, 63], 64),
    "clamped": ([3, 10, 7], [5, -2, 7], 16), "odd page": ([100, 1, 250], [7, 1, 250], 24),
    "257 rows": ([1 + (i * 37) % 500 for i in range(257)], [(i * 5) % 9 for i in range(257)], 64),
    "1000 rows": ([1 + (i * 91) % 3000 for i in range(1000)], [1 + (i * 3) % 4 for i in range(1000)], 128),
    "long": ([5000, 20, 3333], [5000, 20, 2000], 128),
}


@pytest.mark.parametrize("name", list(TABLES))
@pytest.mark.parametrize("grow", [False, True])
def test_chunk_meta(hip, name, grow):
    lens, ql, ebs = TABLES[name]
    import random
    rng = random.Random(len(name))
    R, width = len(lens), max(-(-n // ebs) for n in lens) + 1
    ids = rng.sample(range(R * width * 2), R * width * 2)
    T = sum(min(max(c, 0), n) for n, c in zip(lens, ql))
    held = [min(-(-(n - min(max(c, 0), n)) // ebs) + rng.randint(0, 1), width) for n, c in zip(lens, ql)] if grow else None
    need = sum(max(0, -(-n // ebs) - h) for n, h in zip(lens, held)) if grow else 0
    dev = torch.device("cuda", 0)
    up = lambda x, t: torch.tensor(x, dtype=t, device=dev)
    for tokens, nfree in ((T, need + 3), (T + 70, need), (max(T - 2, 0), max(need - 2, 0)), (T, 0)):
        bt = [[ids[r * width + p] if not grow or p < held[r] else -1 for p in range(width)] for r in range(R)]
        wide = torch.full((R, width + 2), -9, dtype=torch.int32, device=dev)   # a table wider than its pages in use
        wide[:, :width] = up(bt, torch.int32)
        free = ids[R * width:R * width + 2 + nfree]
        m = hip.chunk_meta(wide[:, :width], up(lens, torch.int64), up(ql, torch.int32), ebs, tokens,
                           **(dict(held=up(held, torch.int32), free=up(free, torch.int32), taken=up([2], torch.int64)) if grow else {}))
        qsl, slot, pos, row, after, taken = ref.tables(bt, lens, ql, ebs, tokens, held, free, 2)
        assert m.qsl.tolist() == qsl and m.pos.tolist() == pos and m.row.tolist() == row
        assert m.slot.tolist() == slot and m.lens32.tolist() == lens
        assert wide[:, :width].tolist() == bt and (wide[:, width:] == -9).all()
        if grow:
            assert m.held.tolist() == after and m.taken.tolist() == [taken]
        else:
            assert m.held is None and m.taken is None


def test_chunk_meta_past_the_table(hip):
    """Positions whose page the table lacks get no slot."""
    dev = torch.device("cuda", 0)
    bt = torch.tensor([[5, -1], [7, 8]], dtype=torch.int32, device=dev)
    m = hip.chunk_meta(bt, torch.tensor([20, 40], device=dev), torch.tensor([8, 12], dtype=torch.int32, device=dev), 16, 22)
    assert m.slot.tolist() == [5 * 16 + 12 + i for i in range(4)] + [-1] * 4 + [8 * 16 + 12 + i for i in range(4)] + [-1] * 10
    assert m.pos.tolist() == list(range(12, 20)) + list(range(28, 40)) + [-1, -1]


def test_chunk_meta_without_rows_and_refusals(hip):
    dev = torch.device("cuda", 0)
    i32, i64 = torch.int32, torch.int64
    z = lambda *s, t=i32: torch.zeros(*s, dtype=t, device=dev)
    m = hip.chunk_meta(z(0, 4), z(0, t=i64), z(0), 64, 3)
    assert m.qsl.tolist() == [0] and m.slot.tolist() == [-1] * 3 and m.row.tolist() == [0] * 3
    for args, kw, err in (((z(2, 4, t=i64), z(2, t=i64), z(2), 64, 3), {}, TypeError), ((z(2, 4), z(2), z(2), 64, 3), {}, TypeError),
                          ((z(2, 4), z(3, t=i64), z(2), 64, 3), {}, ValueError), ((z(2, 4), z(2, t=i64), z(2), 0, 3), {}, ValueError),
                          ((z(2, 4), z(2, t=i64), z(2), 64, -1), {}, ValueError), ((z(2, 4), z(2, t=i64), z(2).cpu(), 64, 3), {}, ValueError),
                          ((z(2, 4), z(2, t=i64), z(2), 64, 3), dict(held=z(2)), ValueError),
                          ((z(1, 4).expand(2, 4), z(2, t=i64), z(2), 64, 3), dict(held=z(2), free=z(5), taken=z(1, t=i64)), ValueError),
                          ((z(4, 2).T, z(2, t=i64), z(2), 64, 3), {}, ValueError)):
        with pytest.raises(err):
            hip.chunk_meta(*args, **kw)


# ---------------------------------------------------------------- short conv
CONV = {"one": [1], "rows": [1, 5, 0, 7, 3], "empty": [0, 0, 2], "tile ends": [15, 1, 16, 33, 0, 2], "long": [300, 0, 41],
        "more than a wave": [i % 4 for i in range(150)]}


def conv_case(new, H, pad, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    qsl = [0]
    for c in new:
        qsl.append(qsl[-1] + c)
    return r(qsl[-1] + pad, 3 * H), r(H, 7), r(len(new), H, 6), qsl


@pytest.mark.parametrize("new", list(CONV))
@pytest.mark.parametrize("H,pad", [(2048, 0), (8, 3), (2056, 1), (4096, 2)])
def test_conv_chunk(hip, new, H, pad):
    """Out: 7 products and sums in fp32 (each within 2^-24 of the running magnitude), then one rounding to bf16."""
    from lfm3_kv800_amd import spec_ops as so
    bcx, w, state, qsl = conv_case(CONV[new], H, pad)
    q = torch.tensor(qsl, device="cuda")
    before = state.clone()
    out, taps = so.conv_chunk(bcx, w, state, q)
    want, tw = ref.conv(bcx, w, state, qsl)
    assert torch.equal(state, before) and torch.equal(taps.double(), tw)
    a = bcx[:, H:2 * H].double().abs()
    mag = ref.conv(torch.cat([bcx[:, :H].abs(), bcx[:, H:2 * H].abs(), bcx[:, 2 * H:].abs()], 1), w.abs(), state.abs(), qsl)[0]
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + 16 * 2 ** -24 * mag).all(), a.shape
    assert not out[qsl[-1]:].any()
    # the state: the last 6 of it and the kept taps
    kept = torch.tensor([(3 * i + 1) % (c + 3) - 1 for i, c in enumerate(CONV[new])], dtype=torch.int32, device="cuda")
    so.conv_commit(state, taps, q, kept)
    for r, c in enumerate(CONV[new]):
        n = min(max(int(kept[r]), 0), c)
        line = torch.cat([before[r].T, taps[qsl[r]:qsl[r] + n]])
        assert torch.equal(state[r], line[-6:].T)


def test_conv_in_pieces_and_step(hip):
    """A row's tokens in one call or in pieces, each committed: the same bits. One token: conv_step up to its roundings (a
    product, the sum and the output, 2^-8 each of at most the sum of magnitudes; here one more)."""
    from lfm3_kv800_amd import model_ops as mo, spec_ops as so
    bcx, w, state, _ = conv_case([40], 2048, 0, seed=5)
    first = state.clone()
    whole, _ = so.conv_chunk(bcx, w, state, torch.tensor([0, 40], device="cuda"))
    at = 0
    for n in (1, 3, 16, 2, 18):
        q = torch.tensor([0, n], device="cuda")
        out, taps = so.conv_chunk(bcx[at:at + n], w, state, q)
        assert torch.equal(out, whole[at:at + n])
        so.conv_commit(state, taps, q, torch.tensor([n], dtype=torch.int32, device="cuda"))
        at += n
    mag = ref.conv(bcx[:1].abs(), w.abs(), first.abs(), [0, 1])[0]   # of the state before conv_step moves it on
    one = mo.conv_step(bcx[:1], w, first)
    assert ((one.double() - whole[:1].double()).abs() <= 2 ** -6 * mag).all()


def test_conv_strides_and_refusals(hip):
    from lfm3_kv800_amd import spec_ops as so
    bcx, w, state, qsl = conv_case([3, 2], 16, 0)
    q = torch.tensor(qsl, device="cuda")
    want = so.conv_chunk(bcx, w, state, q)[0]
    for extra in (8, 5):                       # rows of a wider product, aligned or not
        wide = torch.full((5, 48 + extra), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, :48] = bcx
        assert torch.equal(so.conv_chunk(wide, w, state, q)[0], want)
    assert torch.equal(so.conv_chunk(bcx.T.contiguous().T, w, state, q)[0], want)
    assert so.conv_chunk(bcx[:0], w, state, torch.zeros(3, dtype=torch.int64, device="cuda"))[0].shape == (0, 16)
    kept = torch.ones(2, dtype=torch.int32, device="cuda")
    for f, err in ((lambda: so.conv_chunk(bcx.float(), w, state, q), TypeError), (lambda: so.conv_chunk(bcx, w[:8], state, q), ValueError),
                   (lambda: so.conv_chunk(bcx, w, state[:, :, :5], q), ValueError), (lambda: so.conv_chunk(bcx, w, state[:1], q), ValueError),
                   (lambda: so.conv_chunk(bcx, w, state.transpose(0, 1), q), ValueError), (lambda: so.conv_chunk(bcx, w, state, q.int()), TypeError),
                   (lambda: so.conv_chunk(bcx[:, :40], w, state, q), ValueError), (lambda: so.conv_commit(state, want, q, kept.long()), TypeError),
                   (lambda: so.conv_commit(state, want[:, :8], q, kept), ValueError), (lambda: so.conv_commit(state, want, q, kept[:1]), ValueError)):
        with pytest.raises(err):
            f()


# ---------------------------------------------------------------- verification
def verify_case(new, V, seed, probs, temps, pad=0):
    g = torch.Generator().manual_seed(seed)
    T, R = sum(new) + pad, len(new)
    x = torch.randn(T, V, generator=g) * 2
    x.scatter_(1, torch.randint(0, V, (T, 4), generator=g), 9 + 2 * torch.rand(T, 4, generator=g))
    x = x.to(torch.bfloat16)
    qsl = [0]
    for c in new:
        qsl.append(qsl[-1] + c)
    q = torch.softmax(x.float() + 0.6 * torch.randn(T, V, generator=g), -1) if probs else None
    near = x.float().argmax(-1)
    drawn = torch.multinomial(q if probs else torch.softmax(x.float(), -1), 1, generator=g)[:, 0] if T else near
    tokens = torch.roll(torch.where(torch.rand(T, generator=g) < 0.4, near, drawn), 1)
    temp = torch.tensor([temps[i % len(temps)] for i in range(R)], dtype=torch.float32)
    return x, tokens, qsl, temp, torch.rand(T, generator=g), torch.rand(R, generator=g), q


def run_verify(x, tokens, qsl, temp, u, u_next, q):
    from lfm3_kv800_amd import spec_ops as so
    d = lambda t: None if t is None else t.cuda()
    out, count = so.verify_drafts(d(x), d(tokens), torch.tensor(qsl, device="cuda"), d(temp), d(u), d(u_next), d(q))
    return out.tolist(), count.tolist()


@pytest.mark.parametrize("V", [1, 7, 500, 8192, 8193, 20001])
@pytest.mark.parametrize("probs", [False, True])
def test_verify(hip, V, probs):
    for seed, new in enumerate(([1], [5, 1, 0, 3, 4], [2, 9, 40, 1], [1 + i % 4 for i in range(90)])):
        if V > 9000 and len(new) > 10:
            continue
        case = verify_case(new, V, 10 * seed + V, probs, (0.8, 1.0, 0.0, 1.3), pad=3 * (seed % 2))
        assert run_verify(*case) == ref.verify(case[0], case[1], case[2], *case[3:]), (V, probs, new)


def test_verify_borders(hip):
    """u at 0 and just below 1, equal logits, drafts outside the vocabulary, temperatures that are no positive number."""
    x, tokens, qsl, temp, u, un, q = verify_case([4, 4, 4, 4, 4, 4, 4], 300, 3, True, (1.0,))
    for k, (a, b) in enumerate(((0.0, 0.0), (1 - 2 ** -24, 1 - 2 ** -24), (0.5, 0.0))):
        u, un = torch.full_like(u, a), torch.full_like(un, b)
        for qq in (q, None):
            assert run_verify(x, tokens, qsl, temp, u, un, qq) == ref.verify(x, tokens, qsl, temp, u, un, qq), k
    x[:14] = 1.5
    temp = torch.tensor([1.0, 0.0, 0.5, float("nan"), float("inf"), -1.0, 1e-30])
    tokens[5], tokens[9], tokens[14] = -1, 300, 1 << 40
    assert run_verify(x, tokens, qsl, temp, u, un, None) == ref.verify(x, tokens, qsl, temp, u, un, None)
    assert run_verify(x, tokens, qsl, temp, u, un, q) == ref.verify(x, tokens, qsl, temp, u, un, q)


@pytest.mark.parametrize("V", [700, 9000])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_extreme_temperatures(hip, V, probs):
    """Down to the smallest numbers a row goes by its largest logits (several equal ones share), up to 1e30 all count alike."""
    temps = (1e-3, 1e-8, 1e-12, 1e-16, 1e-25, 1e-30, 1e-45, 1e3, 1e20, 1e30)
    x, tokens, qsl, temp, u, un, q = verify_case([4] * 40, V, 12, probs, temps)
    x[::2, 5::V // 3] = x.max(-1, keepdim=True).values[::2]
    x[1::4, 9] = -torch.finfo(torch.bfloat16).max
    near = torch.randint(0, 3, (160,), generator=torch.Generator().manual_seed(5)) * (V // 3) + 5
    tokens = torch.where(torch.rand(160, generator=torch.Generator().manual_seed(6)) < 0.4, near, tokens)
    case = (x, tokens, qsl, temp, u, un, q)
    assert run_verify(*case) == ref.verify(*case)


def test_verify_infinities_and_nan(hip):
    """Masked tokens (-inf, the lowest bf16) are never taken; a row whose largest logit is not finite goes by its index."""
    x, tokens, qsl, temp, u, un, q = verify_case([5] * 8, 9000, 4, True, (1.0, 0.7))
    x[:, 100:8900] = float("-inf")
    x[5:10, :50] = torch.finfo(torch.bfloat16).min
    x[10:15, 4000] = float("inf")
    x[12, 3000] = float("nan")
    x[16, 8999] = float("nan")
    x[21] = float("-inf")
    for qq in (q, None):
        assert run_verify(x, tokens, qsl, temp, u, un, qq) == ref.verify(x, tokens, qsl, temp, u, un, qq)
    same = torch.softmax(x.double() / 1.0, -1).float().nan_to_num(0.0)
    big = torch.full_like(same, 2.0)                       # a q above p everywhere: nothing is left but p itself
    for qq in (same, big):
        out, count = run_verify(x[25:], tokens[25:], [0, 5, 10, 15], temp[:3], u[25:], un[:3], qq[25:])
        want = ref.verify(x[25:], tokens[25:], [0, 5, 10, 15], temp[:3], u[25:], un[:3], qq[25:])
        assert count == want[1] and (qq is same or out == want[0])


def test_verify_strides_graph_and_refusals(hip):
    from lfm3_kv800_amd import spec_ops as so
    x, tokens, qsl, temp, u, un, q = verify_case([3, 5, 2], 1001, 9, True, (1.0, 0.0))
    want = ref.verify(x, tokens, qsl, temp, u, un, q)
    wide = torch.full((10, 1200), float("nan"), dtype=torch.bfloat16).cuda()
    wide[:, 100:1101] = x.cuda()
    qw = torch.full((10, 1300), float("nan")).cuda()
    qw[:, 3:1004] = q.cuda()
    d = [t.cuda() for t in (tokens, torch.tensor(qsl), temp, u, un)]
    out, count = so.verify_drafts(wide[:, 100:1101], *d, qw[:, 3:1004])
    assert (out.tolist(), count.tolist()) == want
    out, count = so.verify_drafts(wide[:, 100:1101].T.contiguous().T, *d, qw[:, 3:1004].T.contiguous().T)
    assert (out.tolist(), count.tolist()) == want
    g, X = torch.cuda.CUDAGraph(), x.cuda()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out, count = so.verify_drafts(X, *d, qw[:, 3:1004])
    for i in range(3):
        X.copy_(x * (1 + 0.25 * i))
        g.replay()
        torch.cuda.synchronize()
        assert (out.tolist(), count.tolist()) == ref.verify(X.cpu(), tokens, qsl, temp, u, un, q), i
    out, count = so.verify_drafts(X[:0], d[0][:0], torch.zeros(4, dtype=torch.int64, device="cuda"), d[2], d[3][:0], d[4])
    assert out.shape == (0,) and count.tolist() == [0, 0, 0]
    ok = [X, *d]
    for i, bad, err in ((0, X.float(), TypeError), (0, X[0], ValueError), (1, d[0][:3], ValueError), (1, d[0].int(), TypeError),
                        (2, d[1].cpu(), ValueError), (3, d[2].double(), TypeError), (4, d[3][:2], ValueError), (5, d[4][:1], ValueError)):
        with pytest.raises(err):
            so.verify_drafts(*[bad if k == i else t for k, t in enumerate(ok)])
    with pytest.raises(ValueError):
        so.verify_drafts(*ok, q.cuda()[:, :50])


def test_step_operators_on_another_stream(hip):
    """Tables, conv and verification on a stream of their own, from inputs that it made."""
    from lfm3_kv800_amd import spec_ops as so
    st = torch.cuda.Stream()
    g = torch.Generator().manual_seed(41)
    lens, ql = [70, 5, 300], [3, 0, 5]
    bcx, w = torch.randn(8, 3 * 64, generator=g).to(torch.bfloat16), torch.randn(64, 7, generator=g).to(torch.bfloat16)
    state, logits = torch.randn(3, 64, 6, generator=g).to(torch.bfloat16), torch.randn(8, 777, generator=g).to(torch.bfloat16)
    tok, u, un = torch.randint(0, 777, (8,), generator=g), torch.rand(8, generator=g), torch.rand(3, generator=g)
    temp = torch.tensor([1.0, 0.0, 0.7])
    kept = torch.tensor([2, 0, 5], dtype=torch.int32)

    def run():
        d = "cuda"
        bt = torch.arange(3 * 20, dtype=torch.int32, device=d).view(3, 20)
        m = hip.chunk_meta(bt, torch.tensor(lens, device=d), torch.tensor(ql, dtype=torch.int32, device=d), 16, 8)
        s = state.to(d)
        out, taps = so.conv_chunk(bcx.to(d), w.to(d), s, m.qsl)
        so.conv_commit(s, taps, m.qsl, kept.to(d))
        ids, n = so.verify_drafts(logits.to(d), tok.to(d), m.qsl, temp.to(d), u.to(d), un.to(d))
        return m.qsl, m.slot, m.pos, out, s, ids, n
    here = run()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        there = run()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(here, there))
    want = ref.verify(logits, tok, here[0].tolist(), temp, u, un)
    assert there[5].tolist() == want[0] and there[6].tolist() == want[1]
