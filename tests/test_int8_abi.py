"""The C entries and argument checks of the products in 8-bit integers (CPU, no GPU calls): exported, bound, bad arguments rejected
on the host before any launch."""
import os
import re
import subprocess

import pytest

import lfm3_kv800_amd.int8_ops as i8
import lfm3_kv800_amd.kv800_hip as kh

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20          # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not os.path.isfile(kh.LIB):
        pytest.fail(f"{kh.LIB} not built: run __graft_entry__.build()")
    L = kh.load_library()
    for name, (res, args) in i8.SIGNATURES.items():
        getattr(L, name).restype, getattr(L, name).argtypes = res, args
    return L


def refused(lib, rc, word):
    assert rc == -1 and word in lib.kv800_hip_last_error(), (rc, lib.kv800_hip_last_error())


def test_header_exported_and_bound(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "lfm3_int8.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(lfm3_hip_\w+)\s*\(", src)))
    out = subprocess.run(["nm", "-D", "--defined-only", kh.LIB], capture_output=True, text=True, check=True).stdout
    exported = set(re.findall(r"\bT (lfm3_hip_\w+)", out))
    assert names and not [n for n in names if n not in exported]
    assert sorted(i8.SIGNATURES) == names


def test_layout_and_quantize_host_checks(lib):
    f = lambda **k: lib.lfm3_hip_int8_layout(*{**dict(w=A, ld=64, s=A, N=10, K=64, gated=0, wsh=A, ssh=A, st=None), **k}.values())
    for k in (dict(w=None), dict(s=None), dict(wsh=None), dict(wsh=A + 8), dict(ssh=None), dict(N=0), dict(N=(1 << 24) + 2), dict(N=1 << 24), dict(N=(1 << 23) + 2, K=8192), dict(K=0), dict(K=60), dict(K=65544),
              dict(gated=2), dict(gated=1, N=9), dict(ld=-1)):
        refused(lib, f(**k), b"int8_layout")
    g = lambda **k: lib.lfm3_hip_int8_quantize(*{**dict(w=A, ld=64, N=10, K=64, w8=A, s=A, st=None), **k}.values())
    for k in (dict(w=None), dict(w=A + 8), dict(w8=None), dict(w8=A + 4), dict(s=None), dict(N=0), dict(K=12), dict(ld=60)):
        refused(lib, g(**k), b"int8_quantize")


@pytest.mark.parametrize("R", [1, 40, 500])
def test_linear8_host_checks(lib, R):
    need = lib.lfm3_hip_linear8_workspace(R, 96, 128, 0)
    assert need == 0 if R == 1 else need >= R * 128 + 4 * R
    f = lambda **k: lib.lfm3_hip_linear8(*{**dict(x=A, ldx=128, w=A, s=A, R=R, N=96, K=128, gated=0, y=A, ldy=96, ws=A, wsb=need, st=None), **k}.values())
    for k in (dict(x=None), dict(x=A + 8), dict(ldx=132), dict(w=None), dict(w=A + 8), dict(s=None), dict(s=A + 4), dict(R=-1), dict(R=(1 << 24) + 1), dict(R=1 << 24), dict(N=0), dict(K=0),
              dict(K=100), dict(K=65544), dict(gated=2), dict(gated=1, N=95), dict(y=None), dict(ldy=-1)) + ((dict(ws=None), dict(ws=A + 8), dict(wsb=need - 1)) if need else ()):
        refused(lib, f(**k), b"linear8")
    assert f(R=0) == 0
    for a in ((0, 96, 128, 0), (4, 0, 128, 0), (4, 96, 100, 0), (4, 95, 128, 1)):
        assert lib.lfm3_hip_linear8_workspace(*a) == 0
