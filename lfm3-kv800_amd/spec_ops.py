"""ctypes binding of the model-side operators of a step whose rows bring several new tokens each (include/lfm3_spec.h, in
libkv800_hip.so): the short conv over a row's new tokens, its state moved on over the kept ones, the verification of drafts.

A step's tokens lie row after row; qsl (R + 1,) int64 on the device holds the rows' starts (kv800_hip.chunk_meta). Like
kv800_hip, there is no fallback: without the library or a GPU the first call raises ImportError. Launches go on the current
stream of the tensors' device; workspaces are torch allocations of the call."""
import ctypes

import torch

from . import kv800_hip
from .kv800_hip import _need, _on, _raw_stream

_VP, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
SIGNATURES = {
    "lfm3_hip_conv_chunk": (_I32, [_VP, _I64, _VP, _VP, _VP, _I64, _I64, _I64, _VP, _VP, _VP]),
    "lfm3_hip_conv_commit": (_I32, [_VP, _VP, _VP, _VP, _I64, _I64, _I64, _VP]),
    "lfm3_hip_verify_workspace": (_I64, [_I64, _I64, _I64]),
    "lfm3_hip_verify_drafts": (_I32, [_VP, _I64, _VP, _VP, _VP, _VP, _VP, _VP, _I64, _I64, _I64, _I64, _VP, _VP, _VP, _I64,
                                      _VP]),
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


def _rows(qsl, dev):
    _need(qsl, "qsl", torch.int64, dev)
    if qsl.dim() != 1 or qsl.shape[0] < 1:
        raise ValueError("qsl must be (R + 1,)")
    return qsl.contiguous(), qsl.shape[0] - 1


def _state(state, R, dev):
    _need(state, "state", torch.bfloat16, dev)
    if state.dim() != 3 or state.shape[0] != R or state.shape[2] != 6 or state.shape[1] % 8 or not state.is_contiguous():
        raise ValueError(f"state must be a contiguous ({R}, H, 6) with H a multiple of 8, got {tuple(state.shape)}")


def conv_chunk(bcx, conv_w, state, qsl):
    """Short conv over each row's new tokens (lfm3_hip_conv_chunk): bcx (T, >= 3H) bf16 rows [B | C | x], conv_w (H, 7),
    state (R, H, 6), read only. Returns (out (T, H), taps (T, H)) bf16: the conv outputs, and bf16(B x) of every token, from
    which conv_commit moves the state on."""
    L = _lib()
    dev = bcx.device
    qsl, R = _rows(qsl, dev)
    _need(bcx, "bcx", torch.bfloat16, dev); _need(conv_w, "conv_w", torch.bfloat16, dev)
    _state(state, R, dev)
    H = state.shape[1]
    if bcx.dim() != 2 or bcx.shape[1] < 3 * H or tuple(conv_w.shape) != (H, 7):
        raise ValueError(f"bcx must be (T, >= {3 * H}) and conv_w ({H}, 7), got {tuple(bcx.shape)}, {tuple(conv_w.shape)}")
    T = bcx.shape[0]
    ld = bcx.stride(0) if T > 1 else 3 * H        # of a single row torch's stride may be anything
    if H and (bcx.stride(1) != 1 or ld % 8 or ld < 3 * H or bcx.data_ptr() % 16):
        bcx, ld = bcx[:, :3 * H].clone(memory_format=torch.contiguous_format), 3 * H
    out = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    taps = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    if T == 0 or R == 0 or H == 0:
        return out.zero_(), taps.zero_()
    conv_w = _whole(conv_w)
    with _on(dev):
        kv800_hip._check(L.lfm3_hip_conv_chunk(bcx.data_ptr(), ld, conv_w.data_ptr(), state.data_ptr(), qsl.data_ptr(),
                                               R, T, H, out.data_ptr(), taps.data_ptr(), _raw_stream(dev)))
    return out, taps


def conv_commit(state, taps, qsl, kept):
    """state (R, H, 6) moved on, in place, over the first kept[r] ((R,) int32) of each row's new tokens, whose taps
    conv_chunk returned (lfm3_hip_conv_commit)."""
    L = _lib()
    dev = state.device
    qsl, R = _rows(qsl, dev)
    _state(state, R, dev)
    _need(taps, "taps", torch.bfloat16, dev); _need(kept, "kept", torch.int32, dev)
    H = state.shape[1]
    if taps.dim() != 2 or taps.shape[1] != H or kept.shape != (R,):
        raise ValueError(f"taps must be (T, {H}) and kept ({R},), got {tuple(taps.shape)}, {tuple(kept.shape)}")
    if R == 0 or H == 0 or taps.shape[0] == 0:
        return
    taps, kept = _whole(taps), kept.contiguous()
    with _on(dev):
        kv800_hip._check(L.lfm3_hip_conv_commit(state.data_ptr(), taps.data_ptr(), qsl.data_ptr(), kept.data_ptr(), R,
                                                taps.shape[0], H, _raw_stream(dev)))


def verify_drafts(logits, tokens, qsl, temperature, u, u_next, draft_probs=None):
    """Which drafts of a step are kept, and the token behind them (lfm3_hip_verify_drafts). logits (T, V) bf16: the target's
    behind every token; tokens (T,) int64: the step's tokens, each row's drafts behind its first one; temperature (R,) fp32 (0:
    greedy); u (T,) and u_next (R,) fp32 in [0, 1): u[t] decides on the draft that logits row t judges, u_next[r] picks
    the token behind; draft_probs (T, V) fp32: row t the distribution that token t + 1 was drawn from (None: drafts without
    one, all of it on the draft). Returns (tokens (T,) int64, count (R,) int32): row r's kept drafts and the token
    behind them at qsl[r] .., count[r] of them, -1 elsewhere."""
    L = _lib()
    dev = logits.device
    qsl, R = _rows(qsl, dev)
    _need(logits, "logits", torch.bfloat16, dev); _need(tokens, "tokens", torch.int64, dev)
    for t, name in ((temperature, "temperature"), (u, "u"), (u_next, "u_next")):
        _need(t, name, torch.float32, dev)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be (T, V), got {tuple(logits.shape)}")
    T, V = logits.shape
    if tokens.shape != (T,) or u.shape != (T,) or temperature.shape != (R,) or u_next.shape != (R,):
        raise ValueError(f"tokens and u must be ({T},), temperature and u_next ({R},)")
    if draft_probs is not None:
        _need(draft_probs, "draft_probs", torch.float32, dev)
        if draft_probs.shape != (T, V):
            raise ValueError(f"draft_probs must be ({T}, {V}), got {tuple(draft_probs.shape)}")
        draft_probs, ldq = _row_major(draft_probs)
    logits, ld = _row_major(logits)
    out = torch.empty(T, dtype=torch.int64, device=dev)
    count = torch.empty(R, dtype=torch.int32, device=dev)
    if R == 0 or T == 0:
        return out.fill_(-1), count.zero_()
    wsb = int(L.lfm3_hip_verify_workspace(R, T, V))
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
    tokens, temperature, u, u_next = tokens.contiguous(), temperature.contiguous(), u.contiguous(), u_next.contiguous()
    with _on(dev):
        kv800_hip._check(L.lfm3_hip_verify_drafts(
            logits.data_ptr(), ld, tokens.data_ptr(), qsl.data_ptr(), temperature.data_ptr(), u.data_ptr(),
            u_next.data_ptr(), None if draft_probs is None else draft_probs.data_ptr(),
            0 if draft_probs is None else ldq, R, T, V, out.data_ptr(), count.data_ptr(), ws.data_ptr(), wsb,
            _raw_stream(dev)))
    return out, count


def _row_major(x):
    """x with contiguous rows that do not overlap, and their stride (a size of one may have any stride in torch, and counts as
    contiguous with it)."""
    T, V = x.shape
    ld = x.stride(0) if T > 1 else V
    return (x, ld) if (V == 1 or x.stride(1) == 1) and ld >= V else (x.clone(memory_format=torch.contiguous_format), V)


def _whole(x):
    """x contiguous and 16-byte aligned."""
    x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x
