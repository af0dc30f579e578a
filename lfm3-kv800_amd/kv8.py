"""Paged 8-bit cache of keys and values (include/kv8_hip.h, in libkv800_hip.so): appending a step's tokens with the position
rotation on the way, attention over it, reading it back.

Between the exact bf16 pages and the 800h format: e4m3 codes with a power of two for each block of 64 tokens of a KV head, keys
and values apart. A step's tokens lie row after row; qsl (R + 1,) int64 holds the rows' starts and lens (R,) int64 their lengths
with the new tokens, both on the device (kv800_hip.chunk_meta makes them for steps of any shape). Like kv800_hip, there is no
fallback: without the library or a GPU the first call raises ImportError. Launches go on the current stream of the tensors'
device; workspaces are torch allocations of the call."""
import ctypes
import math

import torch

from . import kv800_hip
from .kv800_hip import _need, _on, _raw_stream

BLK = 64                 # tokens per block
_VP, _I64, _I32, _F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float


class _Cache(ctypes.Structure):
    """kv8_cache_t (include/kv8_hip.h)."""
    _fields_ = [("data", _VP), ("exps", _VP), ("pages", _I64), ("kv_heads", _I64), ("blocks", _I64), ("dim", _I64),
                ("page_stride", _I64), ("exp_stride", _I64)]


_CP = ctypes.POINTER(_Cache)
SIGNATURES = {
    "kv8_hip_append": (_I32, [_CP, _VP, _I64, _I64, _VP, _I64, _I64, _VP, _I64, _I64, _VP, _VP, _I64, _I64, _VP, _VP, _I64, _I64,
                              _VP]),
    "kv8_hip_dequantize": (_I32, [_CP, _VP, _VP, _VP]),
    "kv8_hip_attend_workspace": (_I64, [_CP, _I64, _I64, _I64, _I64, _I64]),
    "kv8_hip_attend": (_I32, [_CP, _VP, _I64, _VP, _I64, _I64, _VP, _VP, _I64, _I64, _I64, _F32, _VP, _VP, _I64, _VP]),
}
_BOUND = {}


def _lib():
    L = kv800_hip.ops()
    if id(L) not in _BOUND:
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _BOUND.clear()
        _BOUND[id(L)] = True
    return L


class Cache8:
    """A layer's cache: data (pages, kv heads, blocks, 2, 64 D) uint8, the e4m3 codes of each block's keys and values in operand
    order, and exps (pages, kv heads, blocks, 2) uint8, their exponent bytes (value = code 2^(byte - 127)); D 64 or 128, a page
    holds 64 blocks tokens. The pages of both may lie apart (stride(0)); within a page they are contiguous."""

    def __init__(self, data, exps):
        if data.dtype != torch.uint8 or data.dim() != 5 or data.shape[3] != 2 or data.shape[4] not in (64 * BLK, 128 * BLK):
            raise ValueError(f"data must be (pages, heads, blocks, 2, 64 D) uint8 with D 64 or 128, got {data.dtype} {tuple(data.shape)}")
        _need(exps, "exps", torch.uint8, data.device)
        if exps.shape != data.shape[:4]:
            raise ValueError(f"exps must be {tuple(data.shape[:4])}, got {tuple(exps.shape)}")
        P, H, U, _, n = data.shape
        if not (P and H and U):
            raise ValueError("a cache needs pages, heads and blocks")
        for t, name in ((data, "data"), (exps, "exps")):
            if not t[0].is_contiguous() or (P > 1 and t.stride(0) < t[0].numel()):
                raise ValueError(f"{name}: a page must be contiguous, and pages may not overlap")
        ps = data.stride(0) if P > 1 else H * U * 2 * n
        es = exps.stride(0) if P > 1 else H * U * 2
        if ps % 16 or data.data_ptr() % 16 or es % 2 or exps.data_ptr() % 2:
            raise ValueError("data must be 16-byte aligned, its pages a multiple of 16 bytes apart; exps 2-byte aligned, an even number apart")
        self.data, self.exps = data, exps
        self.pages, self.heads, self.blocks, self.dim = P, H, U, n // BLK
        self.bs, self.dev, self.on_gpu = U * BLK, data.device, data.is_cuda
        self._c = _Cache(data.data_ptr(), exps.data_ptr(), P, H, U, self.dim, ps, es)
        self._p = ctypes.byref(self._c)

    @classmethod
    def empty(cls, pages, heads, bs, dim, device):
        """A cache of `pages` pages of bs tokens (a multiple of 64) of `heads` KV heads of `dim` channels."""
        if bs < BLK or bs % BLK or dim not in (64, 128):
            raise ValueError("bs must be a multiple of 64 and dim 64 or 128")
        return cls(torch.zeros(pages, heads, bs // BLK, 2, BLK * dim, dtype=torch.uint8, device=device),
                   torch.full((pages, heads, bs // BLK, 2), 127, dtype=torch.uint8, device=device))


def _dev(cache):
    """The cache's GPU. (A cache of host tensors may be described, not worked on.)"""
    if not cache.on_gpu:
        raise ValueError(f"the cache must be on a GPU, got {cache.dev}")
    return cache.dev


def _step(cache, T, bt, lens, qsl):
    dev, i64 = cache.dev, torch.int64
    if not (bt.dtype is torch.int32 and lens.dtype is i64 and qsl.dtype is i64 and bt.device == dev and lens.device == dev and qsl.device == dev):
        _need(bt, "bt", torch.int32, dev); _need(lens, "lens", i64, dev); _need(qsl, "qsl", i64, dev)
    if qsl.dim() != 1 or qsl.shape[0] < 1:
        raise ValueError("qsl must be (R + 1,)")
    R = qsl.shape[0] - 1
    if lens.shape != (R,) or bt.dim() != 2 or bt.shape[0] != R:
        raise ValueError(f"lens must be ({R},) and bt ({R}, pages), got {tuple(lens.shape)}, {tuple(bt.shape)}")
    if bt.shape[1] > 1 and R and bt.stride(1) != 1:
        raise ValueError("bt must have contiguous rows")
    if T and not R:
        raise ValueError("tokens without rows")
    return R, lens.contiguous(), qsl.contiguous()


def _kv(x, name, cache, T):
    """x with channels side by side and aligned rows, and its token and head strides."""
    if x.dtype is not torch.bfloat16 or x.device != cache.dev:
        _need(x, name, torch.bfloat16, cache.dev)
    if x.shape != (T, cache.heads, cache.dim):
        raise ValueError(f"{name} must be ({T}, {cache.heads}, {cache.dim}), got {tuple(x.shape)}")
    ts, hs, one = x.stride()
    if T <= 1:
        ts = 0                                           # of a single one torch's stride may be anything
    if cache.heads == 1:
        hs = 0
    if one != 1 or ts % 8 or hs % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        ts, hs = cache.heads * cache.dim, cache.dim
    return x, ts, hs


def append(cache, k, v, bt, lens, qsl, cos_t=None, sin_t=None):
    """Append a step's tokens to the rows' blocks (kv8_hip_append): k, v (T, kv heads, D) bf16, views of one product among them;
    bt (R, pages) int32 block table, lens, qsl (above); cos_t / sin_t (P, F) bf16: the key pairs (f, f + D / 2), f < F, are
    rotated by the angles of their positions in fp32 (F a multiple of 8; None: keys as they come). Tokens [qsl[R], T) are padding,
    tokens whose position the table has no page for are dropped. A block's exponent never falls while the row's earlier tokens are
    in it: a larger token has their codes rounded again."""
    L = _lib()
    dev = _dev(cache)
    if k.dim() != 3:
        raise ValueError(f"k must be (T, heads, D), got {tuple(k.shape)}")
    T = k.shape[0]
    R, lens, qsl = _step(cache, T, bt, lens, qsl)
    k, kt, kh = _kv(k, "k", cache, T)
    v, vt, vh = _kv(v, "v", cache, T)
    rows = F = 0
    if (cos_t is None) != (sin_t is None):
        raise ValueError("cos_t and sin_t go together")
    if cos_t is not None:
        if not (cos_t.dtype is torch.bfloat16 and sin_t.dtype is torch.bfloat16 and cos_t.device == dev and sin_t.device == dev):
            _need(cos_t, "cos_t", torch.bfloat16, dev); _need(sin_t, "sin_t", torch.bfloat16, dev)
        if cos_t.dim() != 2 or cos_t.shape != sin_t.shape or not cos_t.shape[0] or cos_t.shape[1] % 8 or not 0 < cos_t.shape[1] <= cache.dim // 2:
            raise ValueError(f"cos_t / sin_t must be (P, F) with F a multiple of 8 up to {cache.dim // 2}, got {tuple(cos_t.shape)}, {tuple(sin_t.shape)}")
        rows, F = cos_t.shape
        cos_t, sin_t = _whole(cos_t), _whole(sin_t)
    if T == 0 or R == 0 or bt.shape[1] == 0:
        return
    with _on(dev):
        kv800_hip._check(L.kv8_hip_append(cache._p, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, bt.data_ptr(),
                                          bt.stride(0) if R > 1 else bt.shape[1], bt.shape[1], lens.data_ptr(), qsl.data_ptr(), R, T,
                                          cos_t.data_ptr() if F else None, sin_t.data_ptr() if F else None, rows, F,
                                          _raw_stream(dev)))


def dequantize(cache):
    """(k, v) (pages, kv heads, page tokens, D) bf16: what the cache stands for (kv8_hip_dequantize)."""
    L = _lib()
    dev = _dev(cache)
    k, v = torch.empty(2, cache.pages, cache.heads, cache.bs, cache.dim, dtype=torch.bfloat16, device=dev).unbind(0)
    with _on(dev):
        kv800_hip._check(L.kv8_hip_dequantize(cache._p, k.data_ptr(), v.data_ptr(), _raw_stream(dev)))
    return k, v


def attend(cache, q, bt, lens, qsl, window=0, scale=None):
    """Attention of a step's tokens over the cache, which holds them already (kv8_hip_attend): q (T, heads, D) bf16, query head h
    on KV head h / (heads / kv heads), up to 16 query heads a KV head; a query sees the positions up to its own and, with a
    window, the last `window` of them. scale: 1 / sqrt(D) if None. Returns (T, heads, D) bf16; zeros for queries without keys and
    for the padding. How it runs goes by T, R and the table's width: a prompt beside single tokens over long rows is quicker in a call
    of its own (its rows of q, bt and lens, and their starts)."""
    L = _lib()
    dev = _dev(cache)
    _need(q, "q", torch.bfloat16, dev)
    if q.dim() != 3 or q.shape[2] != cache.dim or not q.shape[1] or q.shape[1] % cache.heads or q.shape[1] > 16 * cache.heads:
        raise ValueError(f"q must be (T, heads, {cache.dim}) with heads a multiple of {cache.heads} up to {16 * cache.heads}, got {tuple(q.shape)}")
    T, heads = q.shape[:2]
    R, lens, qsl = _step(cache, T, bt, lens, qsl)
    window = min(int(window), 1 << 40)
    if window < 0:
        raise ValueError("window must be >= 0")
    scale = 1.0 / math.sqrt(cache.dim) if scale is None else float(scale)
    out = torch.empty(T, heads, cache.dim, dtype=torch.bfloat16, device=dev)
    if T == 0:
        return out
    q = _whole(q)
    cols = bt.shape[1]
    with _on(dev):
        wsb = int(L.kv8_hip_attend_workspace(cache._p, heads, R, T, cols, window))
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        kv800_hip._check(L.kv8_hip_attend(cache._p, q.data_ptr(), heads, bt.data_ptr(), bt.stride(0) if R > 1 else cols, cols,
                                          lens.data_ptr(), qsl.data_ptr(), R, T, window, scale, out.data_ptr(), ws.data_ptr() if wsb else None, wsb,
                                          _raw_stream(dev)))
    return out


def _whole(x):
    """x contiguous and 16-byte aligned."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x
