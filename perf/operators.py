"""Operators of a decode step that brings several new tokens per row (drafted tokens to verify, short prompt chunks).

A server of the 800h caches runs such a step as: the rows' slots, positions and pages from their lengths on the GPU
(tables), the attention of the new tokens over each layer's paged cache (attend), the short-conv layers with a state that
follows only the tokens that are kept (conv), and the choice of the kept tokens (verify). Here each is timed alone, in its
plain form (`own` false: elementary torch operations) or through the package's entry points (`own` true).

Formulas. Row r has history and c_r new tokens, n_r positions in all; its queries stand at n_r - c_r + i.
  attend   keys k(p) = bf16(code * scale + lo) in flushed blocks, bf16 rows elsewhere; the model rotates the dim pairs
           (d, d + 64), d < 32, and holds the rotated key in bf16; values (bit * scale + lo) H, H the normalized 128-point
           Hadamard matrix, or bf16 rows; softmax(q . k / sqrt(128)) v over p <= query position, in window layers
           p > position - 256 or p < 4 (sinks). Query head h reads KV head h / 4.
  conv     tap = bf16(B x) (the state's type); out = C sum_k w_k tap_(t - 6 + k) over the state and the row's taps; the state
           becomes the last 6 taps after the kept tokens.
  verify   p = softmax(logits / temperature); the draft token d that follows logits row t is kept while u_t q_t(d) < p_t(d);
           at the first that is not, a token of max(p - q, 0) is taken, else one of the last row's p: the first index whose
           running sum exceeds u_next times the whole. q is the drafts' distribution, or all on d. Temperature 0: the
           largest logit.
  tables   positions, slots (page * tokens per page + offset) and row numbers of the new tokens, their prefix sums, and the
           pages that the rows need next, taken from a list of free ones in row order."""
import math
import random

import torch

own = False

DEV = "cuda"
BLK, LAG, SUB, WIN, NSINK = 256, 128, 51200, 256, 4
HIDDEN, TAPS, VOCAB = 2048, 7, 65536


def listed():
    return [
        # one user, four drafted tokens over a long context: all latency
        {"name": "attend_1x16384_5", "op": "attend", "layer": "quant", "rows": 1, "lo": 16384, "hi": 16384, "new": 5,
         "ragged": False, "ebs": 128},
        # 64 users at 32K tokens, three drafted tokens each
        {"name": "attend_64x32768_4", "op": "attend", "layer": "quant", "rows": 64, "lo": 32760, "hi": 32760, "new": 4,
         "ragged": False, "ebs": 64},
        # a serving batch of ragged contexts whose rows bring one to eight tokens
        {"name": "attend_192_ragged_8", "op": "attend", "layer": "quant", "rows": 192, "lo": 1024, "hi": 16384, "new": 8,
         "ragged": True, "ebs": 128},
        # short prompt chunks of an odd length behind 4K tokens
        {"name": "attend_16x4096_33", "op": "attend", "layer": "quant", "rows": 16, "lo": 3900, "hi": 4200, "new": 33,
         "ragged": True, "ebs": 128},
        # the largest batch on a window + sinks layer
        {"name": "window_398_5", "op": "attend", "layer": "window", "rows": 398, "lo": 1024, "hi": 32768, "new": 5,
         "ragged": True, "ebs": 128},
        # a native sliding layer, chunks of 16
        {"name": "slide_64_16", "op": "attend", "layer": "slide", "rows": 64, "lo": 100, "hi": 4096, "new": 16,
         "ragged": False, "ebs": 64},
        # tables of one user's step, and of the largest batch
        {"name": "tables_1_5", "op": "tables", "rows": 1, "lo": 1000, "hi": 1000, "new": 5, "ebs": 128, "pad": 3},
        {"name": "tables_398_8", "op": "tables", "rows": 398, "lo": 1024, "hi": 32768, "new": 8, "ebs": 128, "pad": 0},
        # the short-conv layer of a verified batch, and of prompt chunks
        {"name": "conv_64_5", "op": "conv", "rows": 64, "new": 5, "ragged": True},
        {"name": "conv_8x2048", "op": "conv", "rows": 8, "new": 2048, "ragged": False},
        # one user's four drafts without a draft distribution, and a batch whose drafts come with theirs
        {"name": "verify_1_4", "op": "verify", "rows": 1, "drafts": 4, "ragged": False, "vocab": VOCAB, "probs": False,
         "greedy": 0.0},
        {"name": "verify_256_4", "op": "verify", "rows": 256, "drafts": 4, "ragged": True, "vocab": VOCAB, "probs": True,
         "greedy": 0.2},
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "tables", "conv", "verify", "verify"])
    if op == "attend":
        layer = rng.choice(["quant", "quant", "window", "slide"])
        hi = _log(rng, 2, 32768)
        most = 64 * 32768 // hi if layer == "quant" else 398
        new = _log(rng, 1, 40)
        rows = _log(rng, 1, min(398, most))
        if rows * hi * new > 64 * 32768 * 4 and layer == "quant":   # no more work than the largest listed
            new = max(1, 64 * 32768 * 4 // (rows * hi))
        if layer != "quant":
            rows = max(1, min(rows, 398 * 5 // new))
        return {"op": op, "layer": layer, "rows": rows, "lo": _log(rng, max(1, hi // 32), hi), "hi": hi, "new": new,
                "ragged": rng.random() < 0.7, "ebs": rng.choice([64, 128, 256])}
    if op == "tables":
        hi = _log(rng, 2, 32768)
        return {"op": op, "rows": _log(rng, 1, 1024), "lo": _log(rng, 1, hi), "hi": hi, "new": _log(rng, 1, 64),
                "ebs": rng.choice([64, 128, 1280]), "pad": rng.choice([0, 1, 17])}
    if op == "conv":
        new = _log(rng, 1, 2048)
        return {"op": op, "rows": _log(rng, 1, max(1, min(398, 8 * 2048 // new))), "new": new,
                "ragged": rng.random() < 0.7}
    return {"op": op, "rows": _log(rng, 1, 256), "drafts": rng.randint(1, 4), "ragged": rng.random() < 0.7,
            "vocab": rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), "probs": rng.random() < 0.5,
            "greedy": rng.choice([0.0, 0.3])}


# ---------------------------------------------------------------- sizes (from the case alone)
def _sizes(case):
    """(history lengths, new tokens) of the rows."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    most = case["new"] if "new" in case else case["drafts"] + 1
    least = 1 if case.get("ragged", True) else most
    prev = [rng.randint(case["lo"], case["hi"]) if "lo" in case else 0 for _ in range(case["rows"])]
    return prev, [rng.randint(least, most) for _ in range(case["rows"])]


def _starts(new):
    at = [0]
    for c in new:
        at.append(at[-1] + c)
    return at


def _nq(n):
    return max(n - LAG, 0) // BLK


# ---------------------------------------------------------------- inputs
def _gen(seed, tag):
    return torch.Generator(device=DEV).manual_seed(seed * 1009 + tag)


def _up(x, dtype=torch.int64):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale).to(torch.bfloat16)


def _blocks(seed, m):
    """(m, 51200) sub-blocks with what unit-variance keys and values give: of a 2-bit code the middle values 1 and 2
    are common and 0 and 3 come once in 16; scales near those of 256 normal keys and of 256 rotated values."""
    g, out = _gen(seed, 6), torch.empty(max(m, 1), SUB, dtype=torch.uint8, device=DEV)
    for a in range(0, out.shape[0], 2048):
        o = out[a:a + 2048]
        rnd = lambda n: torch.randint(-(1 << 63), (1 << 63) - 1, (o.shape[0], n // 8), generator=g, device=DEV).view(torch.uint8)
        f8 = lambda mean: (torch.randn(o.shape[0], 512, generator=g, device=DEV) * 0.15 + mean).to(torch.float8_e4m3fn).view(torch.uint8)
        high = rnd(32768) & 0xAA
        o[:, :32768] = high | (((~high >> 1) & 0x55) ^ (rnd(32768) & rnd(32768) & rnd(32768) & rnd(32768) & 0x55))
        o[:, 32768:49152] = rnd(16384)
        for at, mean in ((49152, -2.8), (49664, 5.6), (50176, -2.8), (50688, 1.87)):
            o[:, at:at + 512] = f8(mean)
    return out


def _rope(n):
    inv = 1.0 / (1e6 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 128))
    fr = torch.arange(n, dtype=torch.float64)[:, None] * inv[None]
    return fr.cos().to(torch.bfloat16).to(DEV), fr.sin().to(torch.bfloat16).to(DEV)


def _pages(seed, first, last, ebs):
    """(R, P) page numbers, shuffled, of the rows' positions [first[r], last[r]), and how many there are. Entries that
    no position reaches hold the row's nearest page."""
    held = [(a // ebs, -(-b // ebs)) for a, b in zip(first, last)]
    total = sum(b - a for a, b in held)
    perm, at, table, width = random.Random(seed).sample(range(total), total), 0, [], max(b for _, b in held)
    for a, b in held:
        mine, at = perm[at:at + b - a], at + b - a
        table.append([mine[min(max(j - a, 0), b - a - 1)] for j in range(width)])
    return table, total


def _attend_state(case, seed):
    prev, new = _sizes(case)
    R, ebs, quant = case["rows"], case["ebs"], case["layer"] == "quant"
    nq = [_nq(p) if quant else 0 for p in prev]
    first = [c * BLK if quant else max(0, p - (WIN - 1)) for p, c in zip(prev, nq)]
    last = [p + c for p, c in zip(prev, new)]
    table, pages = _pages(seed, first, last, ebs)
    perm, at, boff = random.Random(seed + 1).sample(range(sum(nq)), sum(nq)), 0, []
    for c in nq:
        boff.append([x * SUB for x in perm[at:at + c]] + [0] * (max(nq + [1]) - c))
        at += c
    T = sum(new)
    s = {"prev": prev, "new": new, "nq": nq, "first": first}
    s["q"] = _normal(_gen(seed, 1), T, 16, 128, scale=2.0)
    s["qsl"], s["N"], s["NQ"] = _up(_starts(new)), _up(last, torch.int32), _up(nq, torch.int32)
    s["epool"] = _normal(_gen(seed, 3), pages, 4, ebs, 256)   # [page, KV head, token, K | V]
    s["eoff"] = _up(table) * (4 * ebs * 256)
    s["qpool"], s["boff"] = _blocks(seed, sum(nq)), _up(boff)
    if case["layer"] == "window":
        s["sk"], s["sv"] = (_normal(_gen(seed, t), R, NSINK, 4, 128) for t in (4, 5))
        s["soff"] = torch.arange(R, device=DEV) * (NSINK * 512)
    if case["layer"] != "slide":   # sliding layers hold rotated keys
        s["cos"], s["sin"] = _rope(max(last) + 64)
    return s


def _tables_state(case, seed):
    prev, new = _sizes(case)
    ebs, R, rng = case["ebs"], case["rows"], random.Random(seed)
    held = [-(-p // ebs) for p in prev]
    need = [-(-(p + c) // ebs) for p, c in zip(prev, new)]
    ids = rng.sample(range(sum(need) + 64), sum(need) + 64)
    at, table, width = 0, [], max(need) + 2
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    return {"bt": _up(table, torch.int32), "lens": _up([p + c for p, c in zip(prev, new)]),
            "qlens": _up(new, torch.int32), "held": _up(held, torch.int32), "free": _up(ids, torch.int32),
            "taken": _up([at]), "tokens": sum(new) + case["pad"]}


def _conv_state(case, seed):
    _, new = _sizes(case)
    g, T, R = _gen(seed, 1), sum(new), case["rows"]
    rng = random.Random(seed)
    return {"bcx": _normal(g, T, 3 * HIDDEN), "w": _normal(g, HIDDEN, TAPS, scale=0.3),
            "state": _normal(g, R, HIDDEN, TAPS - 1), "qsl": _up(_starts(new)),
            "kept": _up([rng.randint(1, c) for c in new], torch.int32)}


def _verify_state(case, seed):
    """Target logits with a few likely tokens per row; drafts from a distribution near the target's."""
    _, new = _sizes(case)
    g, T, V, R = _gen(seed, 1), sum(new), case["vocab"], case["rows"]
    rng = random.Random(seed)
    temp = _up([0.0 if rng.random() < case["greedy"] else rng.uniform(0.6, 1.2) for _ in range(R)], torch.float32)
    row = torch.repeat_interleave(torch.arange(R, device=DEV), _up(new))
    logits = torch.randn(T, V, generator=g, device=DEV).mul_(2.2)
    logits.scatter_(1, torch.randint(0, V, (T, 8), generator=g, device=DEV), 12.0 + 2 * torch.rand(T, 8, generator=g, device=DEV))
    t = torch.where(temp > 0, temp, 1.0)[row, None]
    q = torch.softmax((logits + 0.7 * torch.randn(T, V, generator=g, device=DEV)) / t, -1)
    e = torch.empty(T, V, device=DEV).exponential_(generator=g)
    drafted = (q / e).argmax(-1)                             # one token of each row of q
    best = logits.argmax(-1)
    drafted = torch.where((temp[row] == 0) & (torch.rand(T, generator=g, device=DEV) < 0.8), best, drafted)
    tokens = torch.roll(drafted, 1)                          # token t + 1 is drawn from distribution t
    return {"logits": logits.to(torch.bfloat16), "tokens": tokens, "qsl": _up(_starts(new)), "temp": temp,
            "u": torch.rand(T, generator=g, device=DEV), "u_next": torch.rand(R, generator=g, device=DEV),
            "q": q if case["probs"] else None}


def prepare(case, seed):
    s = {"attend": _attend_state, "tables": _tables_state, "conv": _conv_state, "verify": _verify_state}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"attend": _attend, "tables": _tables, "conv": _conv, "verify": _verify}[op](s)


def _own(s, op):
    from lfm3_kv800_amd import kv800, kv800_hip, spec_ops
    if op == "attend":
        e, win = s["epool"], s["case"]["layer"] != "quant"
        sk, so = s.get("sk"), s.get("soff")
        P = kv800.Paged(qpool=s["qpool"], boff=s["boff"], epool=e, eoff=s["eoff"], ebs=e.shape[2], e_hs=e.stride(1),
                        e_ts=e.stride(2), e_v=128, sk=sk, sv=s.get("sv"), skoff=so, svoff=so, N=s["N"], NQ=s["NQ"],
                        nqmax=max(s["nq"]), win=WIN if win else 0)
        return kv800_hip.decode_chunk(P, s["q"], s["qsl"], s.get("cos"), s.get("sin"))
    if op == "tables":
        m = kv800_hip.chunk_meta(s["bt"], s["lens"], s["qlens"], s["case"]["ebs"], s["tokens"], held=s["held"],
                                 free=s["free"], taken=s["taken"])
        return {"qsl": m.qsl, "slot": m.slot, "pos": m.pos, "row": m.row, "held": m.held, "taken": m.taken, "bt": s["bt"]}
    if op == "conv":
        out, taps = spec_ops.conv_chunk(s["bcx"], s["w"], s["state"], s["qsl"])
        spec_ops.conv_commit(s["state"], taps, s["qsl"], s["kept"])
        return {"out": out, "taps": taps, "state": s["state"]}
    out, count = spec_ops.verify_drafts(s["logits"], s["tokens"], s["qsl"], s["temp"], s["u"], s["u_next"], s["q"])
    return {"tokens": out, "count": count}


# ---------------------------------------------------------------- plain forms
def _f8(b):
    return b.contiguous().view(torch.float8_e4m3fn).float()


def _hadamard(dtype):
    """The normalized 128-point Hadamard matrix: (-1)^popcount(i & j) / sqrt(128)."""
    h = torch.ones(1, 1, dtype=dtype, device=DEV)
    two = torch.tensor([[1, 1], [1, -1]], dtype=dtype, device=DEV)
    h = torch.kron(two, torch.kron(two, torch.kron(two, torch.kron(two, torch.kron(two, torch.kron(two, torch.kron(two, h)))))))
    return h / math.sqrt(128)


def _rotated(k, pos, cos, sin):
    """Keys (..., 4, 128) at positions pos (...), rotated and held in bf16 as the model holds them."""
    c, s = cos[pos].float()[..., None, :], sin[pos].float()[..., None, :]
    a, b, x, y = k[..., :32], k[..., 32:64], k[..., 64:96], k[..., 96:]
    return torch.cat([a * c - x * s, b, x * c + a * s, y], -1).to(torch.bfloat16).float()


def _attend(s):
    R, C, nq, dev = len(s["new"]), max(s["new"]), s["nq"], DEV
    qsl, N = s["qsl"], s["N"].long()
    ar = lambda n: torch.arange(n, device=dev)
    new = qsl[1:] - qsl[:-1]
    at = (qsl[:-1, None] + ar(C)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[at].view(R, C, 4, 4, 128).permute(0, 2, 1, 3, 4).reshape(R, 4, 4 * C, 128) / math.sqrt(128)
    qpos = ((N - new)[:, None] + ar(C)).repeat_interleave(4, 1)                                 # (R, 4 C)
    # exact rows, from position `lo` of each row on, behind the sinks
    win = s["case"]["layer"] != "quant"
    lo = (N - new - (WIN - 1)).clamp(min=0) if win else s["NQ"].long() * BLK
    E = max(p + c - f for p, c, f in zip(s["prev"], s["new"], s["first"]))
    pos = lo[:, None] + ar(E)
    ebs, pool = s["epool"].shape[2], s["epool"].view(-1, 128)
    page = s["eoff"].gather(1, (pos // ebs).clamp(max=s["eoff"].shape[1] - 1))
    vec = (page[..., None] // 128 + (ar(4) * ebs + (pos % ebs)[..., None]) * 2).clamp(max=pool.shape[0] - 2)   # K's 128-vector
    K, V = pool[vec].float(), pool[vec + 1].float()                                             # (R, E, 4, 128)
    kpos = torch.where(pos < N[:, None], pos, 1 << 30)
    if "sk" in s:
        K, V = torch.cat([s["sk"].float(), K], 1), torch.cat([s["sv"].float(), V], 1)
        sinks = torch.where(ar(NSINK) < lo[:, None], ar(NSINK), 1 << 30)
        kpos = torch.cat([sinks, kpos], 1)
    if "cos" in s:
        K = _rotated(K, kpos.clamp(max=s["cos"].shape[0] - 1), s["cos"], s["sin"])
    x = q @ K.permute(0, 2, 3, 1).contiguous()                                                  # (R, 4, 4 C, E)
    keep = kpos[:, None] <= qpos[..., None]
    if win:
        near = kpos[:, None] > qpos[..., None] - WIN
        keep = keep & ((near | (kpos[:, None] < NSINK)) if "sk" in s else near)
    x = x.masked_fill(~keep[:, None], -math.inf)
    V = V.permute(0, 2, 1, 3).contiguous()
    M = sum(nq)
    if M == 0:
        o = torch.softmax(x, -1) @ V
    else:   # flushed blocks, one after the other over all rows
        row = torch.repeat_interleave(ar(R), s["NQ"].long(), output_size=M)
        j = ar(M) - (s["NQ"].long().cumsum(0) - s["NQ"])[row]
        sb = s["qpool"][s["boff"][row, j] // SUB]
        kc = sb[:, :32768].view(M, BLK, 4, 32)
        k = torch.cat([kc & 3, (kc >> 2) & 3, (kc >> 4) & 3, kc >> 6], -1).float()
        k = k * _f8(sb[:, 50688:]).view(M, 1, 4, 128) + _f8(sb[:, 50176:50688]).view(M, 1, 4, 128)
        k = _rotated(k.to(torch.bfloat16).float(), j[:, None] * BLK + ar(BLK), s["cos"], s["sin"])
        y = q[row] @ k.permute(0, 2, 3, 1).contiguous()                                         # (M, 4, 4 C, 256)
        del k
        wide = torch.full((R, max(nq)) + y.shape[1:], -math.inf, device=dev)
        wide[row, j] = y
        del y
        top = torch.maximum(wide.amax((1, 4)), x.amax(-1))
        x = torch.exp(x - top[..., None])
        wide = torch.exp(wide - top[:, None, ..., None])
        total = wide.sum((1, 4)) + x.sum(-1)
        vb = sb[:, 32768:49152].view(M, BLK, 4, 1, 16)
        v = ((vb >> torch.arange(8, dtype=torch.uint8, device=dev)[:, None]) & 1).view(M, BLK, 4, 128).float()
        pair = lambda b: _f8(b).view(M, BLK, 2, 1).repeat_interleave(2, 2)
        v = v * pair(sb[:, 49664:50176]) + pair(sb[:, 49152:49664])
        part = wide[row, j] @ v.permute(0, 2, 1, 3).contiguous()                                # (M, 4, 4 C, 128)
        acc = torch.zeros((R, max(nq)) + part.shape[1:], device=dev)
        acc[row, j] = part
        o = (acc.sum(1) @ _hadamard(torch.float32) + x @ V) / total[..., None]
    o = o.view(R, 4, C, 4, 128).permute(0, 2, 1, 3, 4).reshape(R * C, 16, 128)
    T = s["q"].shape[0]
    row = torch.repeat_interleave(ar(R), new, output_size=T)
    return o[row * C + ar(T) - qsl[row]].to(torch.bfloat16)


def _tables(s):
    ebs, bt, held, T = s["case"]["ebs"], s["bt"], s["held"].long(), s["tokens"]
    R, width = bt.shape
    n, c = s["lens"], s["qlens"].long()
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    qsl = torch.cat([zero, c.cumsum(0)])
    grow = ((n + ebs - 1) // ebs - held).clamp(min=0)
    at = s["taken"] + grow.cumsum(0) - grow
    col = torch.arange(width, device=DEV)
    fresh = (col >= held[:, None]) & (col < (held + grow)[:, None])
    new = s["free"][(at[:, None] + col - held[:, None]).clamp(0, s["free"].shape[0] - 1)]
    bt.copy_(torch.where(fresh, new, bt))
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(qsl[1:], t, right=True)
    live = row < R
    row = torch.where(live, row, 0)
    pos = (n - c)[row] + t - qsl[row]
    slot = bt[row, (pos // ebs).clamp(0, width - 1)].long() * ebs + pos % ebs
    return {"qsl": qsl, "slot": torch.where(live, slot, -1), "pos": torch.where(live, pos, -1), "row": row,
            "held": (held + grow).to(torch.int32), "taken": s["taken"] + grow.sum(), "bt": bt}


def _conv(s):
    T, R, qsl, state = s["bcx"].shape[0], s["state"].shape[0], s["qsl"], s["state"]
    b, c, x = s["bcx"].float().split(HIDDEN, 1)
    taps = (b * x).to(torch.bfloat16)
    t = torch.arange(T, device=DEV)
    row = torch.repeat_interleave(torch.arange(R, device=DEV), qsl[1:] - qsl[:-1], output_size=T)
    # every row's state and taps one after the other; row r's taps begin at qsl[r] + 6 (r + 1)
    line = torch.empty(T + 6 * R, HIDDEN, device=DEV)
    line[t + 6 * (row + 1)] = taps.float()
    line[(qsl[:-1] + 6 * torch.arange(R, device=DEV))[:, None] + torch.arange(6, device=DEV)] = state.float().transpose(1, 2)
    window = line[(t + 6 * row)[:, None] + torch.arange(TAPS, device=DEV)]                       # (T, 7, H)
    out = (c * (window * s["w"].float().T).sum(1)).to(torch.bfloat16)
    last = (qsl[:-1] + 6 * torch.arange(R, device=DEV) + s["kept"])[:, None] + torch.arange(6, device=DEV)
    state.copy_(line[last].transpose(1, 2))
    return {"out": out, "taps": taps, "state": state}


def _verify(s):
    x, tokens, qsl, V = s["logits"].double(), s["tokens"], s["qsl"], s["logits"].shape[1]
    T, R = x.shape[0], qsl.shape[0] - 1
    t = torch.arange(T, device=DEV)
    row = torch.repeat_interleave(torch.arange(R, device=DEV), qsl[1:] - qsl[:-1], output_size=T)
    temp = s["temp"].double()[row]
    best = s["logits"].float().argmax(-1)
    e = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(temp > 0, temp, 1.0)[:, None])
    p = e / e.sum(-1, keepdim=True)
    del e, x
    d = tokens[(t + 1).clamp(max=T - 1)]                     # the draft behind each row of logits
    pd = p.gather(1, d[:, None])[:, 0]
    qd = s["q"].double().gather(1, d[:, None])[:, 0] if s["q"] is not None else torch.ones_like(pd)
    kept = torch.where(temp > 0, s["u"].double() * qd < pd, best == d)
    last = t == qsl[1:][row] - 1
    stop = torch.where(kept & ~last, T, t)                   # where a row's kept tokens end: at a rejection or its last row
    first = torch.full((R,), T, device=DEV).scatter_reduce(0, row, stop, "amin")
    # the token after them
    ps, ds = p[first], d[first]
    full = last[first]
    if s["q"] is not None:
        w = (ps - s["q"][first].double()).clamp(min=0)
    else:
        w = ps.scatter(1, ds[:, None], 0.0)
    w = torch.where(full[:, None], ps, w)
    run_ = w.cumsum(-1)
    hit = (run_ <= s["u_next"].double()[:, None] * run_[:, -1:]).sum(-1)
    nxt = torch.where(s["temp"] > 0, hit, best[first])
    out = torch.where(t < first[row], d, torch.where(t == first[row], nxt[row], -1))
    return {"tokens": out, "count": (first - qsl[:-1] + 1).to(torch.int32)}


# ---------------------------------------------------------------- work
def work(case):
    op = case["op"]
    prev, new = _sizes(case)
    R, T = case["rows"], sum(new)
    if op == "attend":
        if case["layer"] == "quant":
            b = sum(_nq(p) * SUB + (p + c - _nq(p) * BLK) * 2048 for p, c in zip(prev, new))
            pairs = sum(c * p + c * (c + 1) // 2 for p, c in zip(prev, new))
        else:
            ns = NSINK if case["layer"] == "window" else 0
            b = sum((min(p, WIN - 1 + ns) + c) * 2048 for p, c in zip(prev, new))
            pairs = sum(min(p + i + 1, WIN + ns) for p, c in zip(prev, new) for i in range(c))
        return {"bytes": b + T * 8192, "flops": pairs * 4 * 16 * 128}
    if op == "tables":
        need = sum(-(-(p + c) // case["ebs"]) - -(-p // case["ebs"]) for p, c in zip(prev, new))
        return {"bytes": R * 24 + (T + case["pad"]) * 28 + need * 8, "flops": 0}
    if op == "conv":
        return {"bytes": T * HIDDEN * 10 + R * HIDDEN * 24 + HIDDEN * 14, "flops": T * HIDDEN * 16}
    V = case["vocab"]
    return {"bytes": T * V * 2 + (R * V * 4 if case["probs"] else 0), "flops": T * V * 12}


# ---------------------------------------------------------------- the same in 64 bits, row by row
def _dequantized(sb, H):
    """(m, 51200) -> keys in bf16 values and rotated-back values, (256 m, 4, 128) float64."""
    m = sb.shape[0]
    byte = sb[:, :32768].reshape(m * BLK, 4, 32).long()
    code = torch.stack([(byte >> (2 * i)) % 4 for i in range(4)], 2).reshape(m, BLK, 4, 128).double()
    k = code * _f8(sb[:, 50688:]).double().view(m, 1, 4, 128) + _f8(sb[:, 50176:50688]).double().view(m, 1, 4, 128)
    byte = sb[:, 32768:49152].reshape(m * BLK, 4, 16).long()
    bit = torch.stack([(byte >> i) % 2 for i in range(8)], 2).reshape(m * BLK, 2, 2, 128).double()
    sc, lo = (_f8(sb[:, a:a + 512]).double().reshape(m * BLK, 2, 1, 1) for a in (49664, 49152))
    return k.to(torch.bfloat16).double().reshape(-1, 4, 128), (bit * sc + lo).reshape(-1, 4, 128) @ H


def exact(case, seed):
    op = case["op"]
    if op in ("tables", "verify"):
        return None
    s = prepare(case, seed)
    if op == "conv":
        b, c, x = s["bcx"].double().split(HIDDEN, 1)
        taps = (b * x).to(torch.bfloat16).double()
        out, qsl, w = torch.empty(taps.shape, dtype=torch.float64, device=DEV), s["qsl"].tolist(), s["w"].double()
        state = torch.empty(s["state"].shape, dtype=torch.float64, device=DEV)
        for r, a in enumerate(s["kept"].tolist()):
            i, j = qsl[r], qsl[r + 1]
            line = torch.cat([s["state"][r].double().T, taps[i:j]])
            out[i:j] = c[i:j] * sum(w[:, k] * line[k:k + j - i] for k in range(TAPS))
            state[r] = line[a:a + 6].T
        return {"out": out, "taps": taps, "state": state}
    H, e, out, at = _hadamard(torch.float64), s["epool"], [], _starts(s["new"])
    ebs, win = e.shape[2], case["layer"] != "quant"
    for r, (p, c) in enumerate(zip(s["prev"], s["new"])):
        pos = torch.arange(s["first"][r], p + c, device=DEV)
        page = s["eoff"][r][pos // ebs] // e.stride(0)
        kv = e[page, :, pos % ebs].double()                                                     # (t, 4, 256)
        K, V = kv[..., :128], kv[..., 128:]
        ns = min(NSINK, s["first"][r]) if case["layer"] == "window" else 0
        if ns:
            K, V = torch.cat([s["sk"][r, :ns].double(), K]), torch.cat([s["sv"][r, :ns].double(), V])
            pos = torch.cat([torch.arange(ns, device=DEV), pos])
        if s["nq"][r]:
            k, v = _dequantized(s["qpool"][s["boff"][r, :s["nq"][r]] // SUB], H)
            K, V, pos = torch.cat([k, K]), torch.cat([v, V]), torch.arange(p + c, device=DEV)
        if "cos" in s:
            cs, sn = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
            turned = K.clone()
            turned[..., :32] = K[..., :32] * cs - K[..., 64:96] * sn
            turned[..., 64:96] = K[..., 64:96] * cs + K[..., :32] * sn
            K = turned.to(torch.bfloat16).double()
        qpos = torch.arange(p, p + c, device=DEV)[:, None]
        keep = pos <= qpos
        if win:
            keep &= (pos > qpos - WIN) | (pos < (NSINK if case["layer"] == "window" else 0))
        o = torch.empty(c, 16, 128, dtype=torch.float64, device=DEV)
        for h in range(16):
            x = s["q"][at[r]:at[r + 1], h].double() @ K[:, h // 4].T.contiguous() / math.sqrt(128)
            o[:, h] = torch.softmax(x.masked_fill(~keep, -math.inf), -1) @ V[:, h // 4].contiguous()
        out.append(o)
    return torch.cat(out)
