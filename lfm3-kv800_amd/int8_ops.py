"""ctypes binding of the engine loop's products in 8-bit integers (include/lfm3_int8.h, in libkv800_hip.so): weights with a scale for
each output channel, activations with one for each token, taken in the call.

Like kv800_hip, there is no fallback: without the library or a GPU the first call raises ImportError. Launches go on the current
stream of the tensors' device; workspaces are torch allocations of the call."""
import ctypes

import torch

from . import kv800_hip
from .kv800_hip import _need, _on, _raw_stream

_VP, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
SIGNATURES = {
    "lfm3_hip_int8_layout": (_I32, [_VP, _I64, _VP, _I64, _I64, _I32, _VP, _VP, _VP]),
    "lfm3_hip_int8_quantize": (_I32, [_VP, _I64, _I64, _I64, _VP, _VP, _VP]),
    "lfm3_hip_linear8_workspace": (_I64, [_I64, _I64, _I64, _I32]),
    "lfm3_hip_linear8": (_I32, [_VP, _I64, _VP, _VP, _I64, _I64, _I64, _I32, _VP, _I64, _VP, _I64, _VP]),
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


def _rows16(x):
    """x (2-D bf16) with rows that the kernels can read (16-byte aligned, channels side by side), and their stride."""
    R, K = x.shape
    ld = x.stride(0) if R > 1 else K                # of a single row torch's stride may be anything
    if x.stride(1) != 1 or ld % 8 or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format), K
    return x, ld


def quantize_rows(w):
    """(codes (N, K) int8, scale (N,) fp32) of a bf16 matrix: with t = max(max |w|, 2^-100) of a row, scale = t / 127 and codes
    round(w (127 / t)), all in fp32 (lfm3_hip_int8_quantize)."""
    L = _lib()
    if w.device.type != "cuda":
        raise ValueError(f"w must be on a GPU, got {w.device}")
    _need(w, "w", torch.bfloat16, w.device)
    if w.dim() != 2 or not w.shape[0] or not w.shape[1] or w.shape[1] % 8 or w.shape[1] > 65536:
        raise ValueError(f"w must be (N, K) with K a multiple of 8 up to 65536, got {tuple(w.shape)}")
    w, ld = _rows16(w)
    N, K = w.shape
    codes = torch.empty(N, K, dtype=torch.int8, device=w.device)
    scale = torch.empty(N, dtype=torch.float32, device=w.device)
    with _on(w.device):
        kv800_hip._check(L.lfm3_hip_int8_quantize(w.data_ptr(), ld, N, K, codes.data_ptr(), scale.data_ptr(), _raw_stream(w.device)))
    return codes, scale


class Weight8:
    """A weight of linear8: w (N, K) int8 with scale (N,) fp32 of its rows, or bf16 without (quantize_rows then), K a multiple of 8
    up to 65,536, laid out once in operand order. gated: w is [g | u] (2 F, K) and linear8 returns silu(g) u, (R, F). n, k: its shape;
    width: that of the product."""

    def __init__(self, w, scale=None, gated=False):
        L = _lib()
        if w.dim() != 2 or not w.shape[0] or not w.shape[1] or w.shape[1] % 8 or w.shape[1] > 65536 or w.shape[0] >= 1 << 24:
            raise ValueError(f"w must be (N, K) with K a multiple of 8 up to 65536, got {tuple(w.shape)}")
        self.gated = bool(gated)
        if self.gated and w.shape[0] % 2:
            raise ValueError(f"a gated weight has an even number of rows, got {w.shape[0]}")
        dev = w.device
        if dev.type != "cuda":
            raise ValueError(f"w must be on a GPU, got {dev}")
        if scale is None:
            w, scale = quantize_rows(w)
        _need(w, "w", torch.int8, dev); _need(scale, "scale", torch.float32, dev)
        N, K = self.n, self.k = w.shape
        if scale.shape != (N,):
            raise ValueError(f"scale must be ({N},), got {tuple(scale.shape)}")
        w, scale = w.contiguous(), scale.contiguous()
        self.width = N // 2 if self.gated else N
        npad = 2 * (-(-(N // 2) // 32) * 32) if self.gated else -(-N // 64) * 64
        self.data = torch.empty(npad * (-(-K // 128) * 128), dtype=torch.int8, device=dev)
        self.scale = torch.empty(npad, dtype=torch.float32, device=dev)
        self._ws = {}                                 # workspace bytes by the number of tokens
        with _on(dev):
            kv800_hip._check(L.lfm3_hip_int8_layout(w.data_ptr(), K, scale.data_ptr(), N, K, int(self.gated), self.data.data_ptr(),
                                                    self.scale.data_ptr(), _raw_stream(dev)))


def linear8(x, weight):
    """x (R, K) bf16 times a Weight8, (R, weight.width) bf16 (lfm3_hip_linear8): x is rounded to 8 bits with a scale for each token,
    the sums are exact, scales and (gated) silu(g) u in fp32, one rounding. A token with an infinity or NaN gives NaN."""
    L = _lib()
    dev = weight.data.device
    _need(x, "x", torch.bfloat16, dev)
    if x.dim() != 2 or x.shape[1] != weight.k:
        raise ValueError(f"x must be (R, {weight.k}), got {tuple(x.shape)}")
    R = x.shape[0]
    out = torch.empty(R, weight.width, dtype=torch.bfloat16, device=dev)
    if R == 0:
        return out
    x, ld = _rows16(x)
    wsb = weight._ws.get(R)
    if wsb is None:
        wsb = weight._ws[R] = int(L.lfm3_hip_linear8_workspace(R, weight.n, weight.k, int(weight.gated)))
    with _on(dev):
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        kv800_hip._check(L.lfm3_hip_linear8(x.data_ptr(), ld, weight.data.data_ptr(), weight.scale.data_ptr(), R, weight.n, weight.k,
                                            int(weight.gated), out.data_ptr(), weight.width, ws.data_ptr() if wsb else None, wsb, _raw_stream(dev)))
    return out
