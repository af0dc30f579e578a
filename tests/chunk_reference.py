"""References in 64 bits for the operators of a step with several new tokens per row, and the caches that their tests use."""
import math

import torch

BLK, LAG, WIN, NSINK = 256, 128, 256, 4


def nq(n):
    return max(n - LAG, 0) // BLK


def rope(n, dev):
    inv = 1.0 / (1e6 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 128))
    fr = torch.arange(n, dtype=torch.float64)[:, None] * inv[None]
    return fr.cos().to(torch.bfloat16).to(dev), fr.sin().to(torch.bfloat16).to(dev)


def rotate(K, pos, cos, sin):
    """(t, 4, 128) keys rotated on the pairs (d, d + 64), d < 32, rounded to bf16; float64."""
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    out = K.clone()
    out[..., :32] = K[..., :32] * c - K[..., 64:96] * s
    out[..., 64:96] = K[..., 64:96] * c + K[..., :32] * s
    return out.to(torch.bfloat16).double()


def attend(q, K, V, kpos, qpos, win=0, nsink=0):
    """q (c, 16, 128), K / V (t, 4, 128) float64 -> (c, 16, 128); a query without keys gives zeros."""
    keep = kpos[None] <= qpos[:, None]
    if win:
        keep &= (kpos[None] > qpos[:, None] - win) | (kpos[None] < nsink)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for h in range(16):
        x = q[:, h].double() @ K[:, h // 4].T.contiguous() / math.sqrt(128)
        p = torch.softmax(x.masked_fill(~keep, -math.inf), -1).nan_to_num(0.0)
        out[:, h] = p @ V[:, h // 4].contiguous()
    return out


class Cache:
    """A paged cache of rows with prev[r] history positions and new[r] new ones, all of them in the exact pages (permuted,
    of `ebs` tokens, heads before tokens or after), the first flushed[r] sub-blocks quantized. Exact positions that nothing may
    read hold NaN, so do the first positions' pages of a window layer; sinks lie in buffers of their own."""

    def __init__(self, kh, prev, new, ebs=64, flushed=None, win=0, sinks=False, token_major=False, seed=0, rot=True):
        dev = torch.device("cuda", 0)
        g = torch.Generator().manual_seed(seed)
        self.prev, self.new, self.win, self.dev, self.rot = prev, new, win, dev, rot
        R = len(prev)
        self.N = [p + c for p, c in zip(prev, new)]
        self.nq = [0] * R if win else [nq(p) for p in prev] if flushed is None else flushed
        rnd = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k).to(torch.bfloat16)
        off = 3 * torch.randn(1, 4, 128, generator=g)                       # per-channel offsets, as trained keys have
        self.K = [(torch.randn(n, 4, 128, generator=g) + off).to(torch.bfloat16).to(dev) for n in self.N]
        self.V = [rnd(n, 4, 128).to(dev) for n in self.N]
        per = max(-(-max(self.N + [1]) // ebs), 1)
        perm = torch.randperm(R * per, generator=g).view(R, per)
        shape = (R * per, ebs, 4, 256) if token_major else (R * per, 4, ebs, 256)
        pool = torch.full(shape, float("nan"), dtype=torch.bfloat16, device=dev)
        e_hs, e_ts = (256, 1024) if token_major else (ebs * 256, 256)
        self.first = [max(0, p - (win - 1)) if win else m * BLK for p, m in zip(prev, self.nq)]
        for r in range(R):
            for p in range(self.first[r] // ebs, -(-self.N[r] // ebs)):
                a, b = max(p * ebs, self.first[r]), min((p + 1) * ebs, self.N[r])
                page = pool[perm[r, p]] if token_major else pool[perm[r, p]].transpose(0, 1)    # (ebs, 4, 256)
                page[a - p * ebs:b - p * ebs, :, :128] = self.K[r][a:b]
                page[a - p * ebs:b - p * ebs, :, 128:] = self.V[r][a:b]
        cap = max(self.nq + [1])
        self.sb = [kh.quantize_blocks(self.K[r][:m * BLK].view(m, BLK, 4, 128), self.V[r][:m * BLK].view(m, BLK, 4, 128))
                   if m else torch.zeros(0, 51200, dtype=torch.uint8, device=dev) for r, m in enumerate(self.nq)]
        total = sum(self.nq)
        where = torch.randperm(max(total, 1), generator=g).tolist()
        qpool = torch.full((max(total, 1), 51200), 0xFF, dtype=torch.uint8, device=dev)
        boff = torch.full((R, cap), 1 << 60, dtype=torch.int64)             # what lies behind a row's blocks is never followed
        at = 0
        for r, m in enumerate(self.nq):
            for j in range(m):
                qpool[where[at]] = self.sb[r][j]
                boff[r, j] = where[at] * 51200
                at += 1
        from lfm3_kv800_amd import kv800
        self.cos, self.sin = rope(max(self.N + [1]) + 8, dev) if rot else (None, None)
        self.sinks = sinks
        sk = sv = so = None
        if sinks:
            sk, sv = rnd(R, NSINK, 4, 128).to(dev), rnd(R, NSINK, 4, 128).to(dev)
            so = torch.arange(R, dtype=torch.int64, device=dev) * (NSINK * 512)
        self.q = rnd(sum(new), 16, 128, k=2.0).to(dev)
        self.qsl = torch.tensor([0] + torch.tensor(new, dtype=torch.int64).cumsum(0).tolist(), dtype=torch.int64, device=dev)
        self.P = kv800.Paged(qpool=qpool, boff=boff.to(dev), epool=pool, eoff=(perm * (ebs * 1024)).to(dev), ebs=ebs, e_hs=e_hs,
                             e_ts=e_ts, e_v=128, sk=sk, sv=sv, skoff=so, svoff=so,
                             N=torch.tensor(self.N, dtype=torch.int32, device=dev),
                             NQ=torch.tensor(self.nq, dtype=torch.int32, device=dev), nqmax=max(self.nq + [0]), win=win)

    def row(self, kh, r):
        """Row r's keys, values and positions as the layer holds them."""
        pos = torch.arange(self.first[r], self.N[r], device=self.dev)
        K, V = self.K[r][self.first[r]:].double(), self.V[r][self.first[r]:].double()
        ns = min(NSINK, self.first[r]) if self.sinks else 0
        if ns:
            K, V = torch.cat([self.P.sk[r, :ns].double(), K]), torch.cat([self.P.sv[r, :ns].double(), V])
            pos = torch.cat([torch.arange(ns, device=self.dev), pos])
        if self.nq[r]:
            k, v = kh.dequantize_blocks(self.sb[r])
            K, V = torch.cat([k.double().view(-1, 4, 128), K]), torch.cat([v.double().view(-1, 4, 128), V])
            pos = torch.cat([torch.arange(self.nq[r] * BLK, device=self.dev), pos])
        if self.rot:
            K = rotate(K, pos, self.cos, self.sin)
        return K, V, pos

    def want(self, kh, drop=None):
        """(T, 16, 128) float64; drop(r, pos) -> positions that the cache cannot give."""
        out, at = torch.zeros(sum(self.new), 16, 128, dtype=torch.float64, device=self.dev), 0
        for r, c in enumerate(self.new):
            if c:
                K, V, pos = self.row(kh, r)
                if drop is not None:
                    keep = ~drop(r, pos)
                    K, V, pos = K[keep], V[keep], pos[keep]
                out[at:at + c] = attend(self.q[at:at + c], K, V, pos, torch.arange(self.prev[r], self.N[r], device=self.dev),
                                        self.win, NSINK if self.sinks else 0)
            at += c
        return out


def tables(bt, lens, qlens, ebs, tokens, held=None, free=None, taken=0):
    """chunk_meta on host lists; bt is a list of lists and grows in place."""
    qsl, slot, pos, row, after = [0], [], [], [], []
    width = len(bt[0]) if bt else 0
    for r, (n, c) in enumerate(zip(lens, qlens)):
        c = min(max(c, 0), n)
        have = width
        if held is not None:
            have = held[r]
            while have < min(-(-n // ebs), width) and taken < len(free):
                bt[r][have] = free[taken]
                have, taken = have + 1, taken + 1
            want = max(0, min(-(-n // ebs), width) - have)
            after.append(have)
            assert want == 0 or taken == len(free)
        for p in range(n - c, n):
            pg = p // ebs
            page = bt[r][pg] if pg < have else -1
            slot.append(page * ebs + p % ebs if page >= 0 else -1)
            pos.append(p)
            row.append(r)
        qsl.append(len(slot))
    pad = max(0, tokens - len(slot))
    return ([min(x, tokens) for x in qsl], (slot + [-1] * pad)[:tokens], (pos + [-1] * pad)[:tokens], (row + [0] * pad)[:tokens],
            after, taken)


def verify(logits, tokens, qsl, temp, u, u_next, q=None):
    """verify_drafts on the host in 64 bits: (T,) tokens, (R,) counts."""
    T, V = logits.shape
    x = logits.double().cpu()
    out, count = [-1] * T, []
    for r in range(len(qsl) - 1):
        a, b = qsl[r], qsl[r + 1]
        n = 0
        for t in range(a, b):
            row, d, last = x[t], int(tokens[t + 1]) if t + 1 < b else None, t + 1 == b
            nan = torch.isnan(row).nonzero()
            top = int(nan[0]) if len(nan) else int((row == row.max()).nonzero()[0])
            tp, ok = float(temp[r]), not len(nan) and math.isfinite(float(row.max()))
            n += 1
            if not (0 < tp <= float(torch.tensor(1e30))) or not ok:     # the fp32 number nearest 1e30
                keep, nxt = not last and d == top, top
            else:
                e = torch.exp((row - row.max()) / tp)
                p = e / e.sum()
                qd = 1.0 if q is None else float(q[t, d]) if not last and 0 <= d < V else 0.0
                keep = not last and 0 <= d < V and float(u[t]) * qd < float(p[d])
                w = p
                if not last:
                    if q is not None:
                        w = (p - q[t].double().cpu()).clamp(min=0).nan_to_num(0.0)
                    elif 0 <= d < V:
                        w = p.clone()
                        w[d] = 0
                    if not float(w.sum()) > 0:
                        w = p
                c = w.cumsum(0)
                over = (c > float(u_next[r]) * float(c[-1])).nonzero()
                nxt = int(over[0]) if len(over) else int(w.nonzero()[-1])
            out[t] = d if keep else nxt
            if not keep:
                break
        count.append(n)
    return out, count


def conv(bcx, w, state, qsl):
    """conv_chunk in 64 bits: outputs and taps (T, H)."""
    H = state.shape[1]
    b, c, x = bcx[:, :H].double(), bcx[:, H:2 * H].double(), bcx[:, 2 * H:3 * H].double()
    taps = (b * x).to(torch.bfloat16).double()
    out = torch.zeros_like(taps)
    keep = torch.zeros_like(taps)
    for r in range(len(qsl) - 1):
        i, j = qsl[r], qsl[r + 1]
        line = torch.cat([state[r].double().T, taps[i:j]])
        keep[i:j] = taps[i:j]
        for k in range(7):
            out[i:j] += w[:, k].double() * line[k:k + j - i]
        out[i:j] *= c[i:j]
    return out, keep
