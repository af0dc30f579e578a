"""The C entries and argument checks of the paged 8-bit cache (CPU, no GPU calls): exported, bound, bad arguments rejected on the
host before any launch."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import lfm3_kv800_amd.kv800_hip as kh
import lfm3_kv800_amd.kv8 as kv8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20          # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not os.path.isfile(kh.LIB):
        pytest.fail(f"{kh.LIB} not built: run __graft_entry__.build()")
    L = kh.load_library()
    for name, (res, args) in kv8.SIGNATURES.items():
        getattr(L, name).restype, getattr(L, name).argtypes = res, args
    return L


def test_header_exported_and_bound(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "kv8_hip.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(kv8_hip_\w+)\s*\(", src)))
    out = subprocess.run(["nm", "-D", "--defined-only", kh.LIB], capture_output=True, text=True, check=True).stdout
    exported = set(re.findall(r"\bT (kv8_hip_\w+)", out))
    assert names and not [n for n in names if n not in exported]
    assert sorted(kv8.SIGNATURES) == names


def desc(**k):
    f = {**dict(data=A, exps=A, pages=4, kv_heads=4, blocks=2, dim=128, page_stride=4 * 2 * 2 * 8192, exp_stride=16), **k}
    return ctypes.byref(kv8._Cache(*f.values()))


BAD = [dict(data=None), dict(data=A + 8), dict(exps=None), dict(pages=0), dict(kv_heads=0), dict(blocks=0), dict(dim=96), dict(page_stride=4 * 2 * 2 * 8192 - 16),
       dict(page_stride=4 * 2 * 2 * 8192 + 8), dict(exp_stride=15), dict(exp_stride=17), dict(exps=A + 1)]


def refused(lib, rc, word):
    assert rc == -1 and word in lib.kv800_hip_last_error(), (rc, lib.kv800_hip_last_error())


def test_append_host_checks(lib):
    base = dict(k=A, kt=512, kh=128, v=A, vt=512, vh=128, bt=A, bs=4, bc=4, lens=A, qsl=A, R=2, T=5, cos=None, sin=None, rr=0, F=0, s=None)
    f = lambda c=None, **k: lib.kv8_hip_append(c or desc(), *{**base, **k}.values())
    for k in BAD:
        refused(lib, f(desc(**k)), b"descriptor")
    for k in (dict(k=None), dict(v=None), dict(bt=None), dict(lens=None), dict(qsl=None), dict(k=A + 2), dict(kt=516), dict(vh=4), dict(R=-1), dict(T=-1),
              dict(bc=-1), dict(cos=A), dict(cos=A, sin=A, rr=0, F=32), dict(cos=A, sin=A, rr=9, F=12), dict(cos=A, sin=A, rr=9, F=72), dict(R=1 << 30), dict(T=1 << 30), dict(R=1 << 23, T=1 << 27), dict(R=(1 << 63) - 1), dict(T=(1 << 63) - 1)):
        refused(lib, f(**k), b"kv8_append")
    for k in (dict(R=0), dict(T=0), dict(bc=0)):
        assert f(**k) == 0


def test_dequantize_host_checks(lib):
    for k in BAD:
        refused(lib, lib.kv8_hip_dequantize(desc(**k), A, A, None), b"descriptor")
    refused(lib, lib.kv8_hip_dequantize(desc(), None, A, None), b"kv8_dequantize")
    refused(lib, lib.kv8_hip_dequantize(desc(), A, A + 8, None), b"kv8_dequantize")


def test_attend_host_checks(lib):
    need = lib.kv8_hip_attend_workspace(desc(), 16, 2, 5, 64, 0)
    assert need > 0
    base = dict(q=A, heads=16, bt=A, bs=64, bc=64, lens=A, qsl=A, R=2, T=5, win=0, scale=0.1, out=A, ws=A, wsb=need, s=None)
    f = lambda c=None, **k: lib.kv8_hip_attend(c or desc(), *{**base, **k}.values())
    for k in BAD:
        refused(lib, f(desc(**k)), b"descriptor")
    for k in (dict(q=None), dict(out=None), dict(bt=None), dict(lens=None), dict(qsl=None), dict(q=A + 8), dict(out=A + 8), dict(heads=0), dict(heads=6), dict(heads=68),
              dict(R=0), dict(R=-1), dict(T=-1), dict(win=-1), dict(scale=0.0), dict(scale=float('inf')), dict(scale=float('nan')), dict(bc=1 << 24), dict(ws=None), dict(ws=A + 8), dict(wsb=need - 1),
              dict(R=1 << 22, T=1 << 22, bc=8), dict(R=1 << 40), dict(T=1 << 40)):
        refused(lib, f(**k), b"kv8_attend")
    for win in (1 << 40, 1 << 62, (1 << 63) - 1):          # past every position: as without a window
        assert lib.kv8_hip_attend_workspace(desc(), 16, 2, 5, 64, win) == need
    assert f(T=0) == 0
    for k in (dict(heads=0), dict(heads=6), dict(heads=68), dict(R=0), dict(T=0), dict(R=1 << 62), dict(T=1 << 62), dict(bc=1 << 62), dict(bc=-1), dict(win=-1),
              dict(heads=64, T=1 << 27)):
        a = {**dict(heads=16, R=2, T=5, bc=64, win=0), **k}
        assert lib.kv8_hip_attend_workspace(desc(), *a.values()) == 0


def test_cache8_refuses():
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for data, exps in ((z(2, 4, 2, 2, 64 * 96), z(2, 4, 2, 2)), (z(2, 4, 2, 64 * 128), z(2, 4, 2)), (z(2, 4, 2, 2, 64 * 64), z(2, 4, 2)),
                       (z(2, 4, 2, 2, 64 * 64), z(2, 4, 1, 2)), (z(2, 4, 2, 2, 64 * 64)[:, :, :1], z(2, 4, 1, 2)), (z(0, 4, 2, 2, 64 * 64), z(0, 4, 2, 2))):
        with pytest.raises(ValueError):
            kv8.Cache8(data, exps)
    with pytest.raises(TypeError):
        kv8.Cache8(z(2, 4, 2, 2, 64 * 64), z(2, 4, 2, 2).int())
    for bs, dim in ((0, 128), (96, 128), (64, 96)):
        with pytest.raises(ValueError):
            kv8.Cache8.empty(2, 4, bs, dim, "cpu")
    c = kv8.Cache8(z(4, 4, 2, 2, 64 * 64)[::2], z(2, 4, 2, 2))           # pages apart
    assert (c.pages, c.heads, c.bs, c.dim) == (2, 4, 128, 64) and c._c.page_stride == 2 * 4 * 2 * 2 * 64 * 64
