"""Plain 64-bit forms of the paged 8-bit cache's operators (CPU, one row after the other), for the tests: the block layout, the
append with its exponents, the attention and how far a kernel may be from it."""
import math

import torch

BLK, LO, HI = 64, -100, 120


def place(t, d, D):
    """Byte of channel d of token t of a block in its keys and in its values."""
    g, a, i = t // 16, t // 4 % 4, t % 4
    return (d // 16) * BLK * 16 + (16 * a + 4 * g + i) * 16 + d % 16, (t // 16 * D + d) * 16 + t % 16


def tables(D):
    t, d = torch.arange(BLK)[:, None], torch.arange(D)[None]
    return place(t, d, D)                                                                       # (64, D) each


def values(data, exps):
    """(keys, values) (pages, H, tokens, D) float64 of a cache on the CPU; NaN where a code is."""
    P, H, U, _, n = data.shape
    D = n // BLK
    out = []
    for i, at in enumerate(tables(D)):
        codes = data[:, :, :, i][..., at.reshape(-1)].contiguous().view(torch.float8_e4m3fn).double().view(P, H, U, BLK, D)
        e = (exps[..., i].long() - 127).clamp(LO, HI).double()
        out.append((codes * torch.pow(2.0, e)[..., None, None]).view(P, H, U * BLK, D))
    return out


def rotate(k, pos, cos, sin):
    """Keys (n, H, D) float64 at positions (n,), rotated and rounded to 32 bits."""
    F, h = cos.shape[1], k.shape[-1] // 2
    p = pos.clamp(0, cos.shape[0] - 1)
    c, s = cos[p].double()[:, None], sin[p].double()[:, None]
    y = k.clone()
    y[..., :F] = k[..., :F] * c - k[..., h:h + F] * s
    y[..., h:h + F] = k[..., h:h + F] * c + k[..., :F] * s
    return y.float().double()


def encode(x, e):
    """float64 x -> e4m3 bytes at exponent e."""
    y = (x * 2.0 ** -e).float()
    return torch.where(torch.isfinite(y), y, math.nan).to(torch.float8_e4m3fn).view(torch.uint8)


def append(data, exps, k, v, bt, lens, qsl, cos=None, sin=None):
    """The cache (data, exps: CPU tensors) after the step, as new tensors."""
    data, exps = data.clone(), exps.clone()
    P, H, U, _, n = data.shape
    D, bs = n // BLK, U * BLK
    at = tables(D)
    for r in range(len(lens)):
        a, b = int(qsl[r]), min(int(qsl[r + 1]), k.shape[0])
        N, c = int(lens[r]), int(qsl[r + 1]) - int(qsl[r])
        pos = torch.arange(N - c, N - c + b - a)
        x = [k[a:b].double(), v[a:b].double()]
        if cos is not None and b > a:
            x[0] = rotate(x[0], pos, cos, sin)
        for blk in sorted({int(p) // BLK for p in pos if p >= 0}):
            if blk * BLK // bs >= bt.shape[1]:
                continue
            page, u = int(bt[r, blk * BLK // bs]), blk % U
            if not 0 <= page < P:
                continue
            here = (pos >= 0) & (pos // BLK == blk)
            t = pos[here] % BLK
            first = int(t.min())
            for i in range(2):
                for h in range(H):
                    y = x[i][here, h]
                    fin = y[torch.isfinite(y)].abs()
                    top = float(fin.max()) if fin.numel() else 0.0
                    e = LO
                    if top > 0:
                        m, ex = math.frexp(top / 448)
                        e = min(max(ex - (m == 0.5), LO), HI)
                    old = min(max(int(exps[page, h, u, i]) - 127, LO), HI)
                    if first > 0 and old > e:
                        e = old
                    codes = data[page, h, u, i]
                    if first > 0 and e > old:
                        w = at[i][:first].reshape(-1)
                        codes[w] = encode(codes[w].view(torch.float8_e4m3fn).double() * 2.0 ** (old - e), 0)
                    codes[at[i][t].reshape(-1)] = encode(y, e).reshape(-1)
                    exps[page, h, u, i] = e + 127
    return data, exps


def attend(data, exps, q, bt, lens, qsl, window=0, scale=None):
    """(outputs, how far a kernel's may be) (T, heads, D) float64. A kernel may round a weight and the output by 2^-8 (bf16);
    scores may be off by 2^-20 of the sum of |q k| (32-bit sums of exact products)."""
    K, V = values(data, exps)
    P, H, bs, D = K.shape
    T, Hq, G = q.shape[0], q.shape[1], q.shape[1] // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, far = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    for r in range(len(lens)):
        a, b, N = int(qsl[r]), int(qsl[r + 1]), int(lens[r])
        n = min(N, bt.shape[1] * bs)
        pos = torch.arange(max(n, 0))
        page = bt[r].long()[pos // bs] if len(pos) else pos
        ok = (page >= 0) & (page < P)
        pos, page = pos[ok], page[ok]
        kr, vr = K[page, :, pos % bs], V[page, :, pos % bs]
        for j in range(a, min(b, T)):
            qp = N - (b - a) + j - a
            see = (pos <= qp) & ((pos > qp - window) if window else torch.ones_like(pos, dtype=torch.bool))
            if not see.any():
                continue
            for h in range(Hq):
                x, kk, vv = q[j, h].double(), kr[see, h // G], vr[see, h // G]
                s = kk @ x * scale
                p = torch.softmax(s, 0)
                out[j, h] = p @ vv
                ds = abs(scale) * 2 ** -20 * float((kk.abs() @ x.abs()).max())
                far[j, h] = (2 ** -8 + 2 * ds) * (p @ vv.abs()) + 2 ** -8 * out[j, h].abs() + 1e-30
    return out, far
