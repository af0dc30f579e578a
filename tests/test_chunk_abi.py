"""The C entries of the operators of a step with several new tokens per row (CPU, no GPU calls): exported, bound, and bad
arguments rejected on the host before any launch."""
import ctypes
import os
import re
import subprocess

import pytest

import lfm3_kv800_amd.kv800_hip as kh
import lfm3_kv800_amd.spec_ops as so

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20          # a pointer that is never followed


@pytest.fixture(scope="module")
def lib():
    if not os.path.isfile(kh.LIB):
        pytest.fail(f"{kh.LIB} not built: run __graft_entry__.build()")
    L = kh.load_library()
    for name, (res, args) in so.SIGNATURES.items():
        getattr(L, name).restype, getattr(L, name).argtypes = res, args
    return L


def test_spec_header_exported_and_bound(lib):
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "lfm3_spec.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(lfm3_hip_\w+)\s*\(", src)))
    out = subprocess.run(["nm", "-D", "--defined-only", kh.LIB], capture_output=True, text=True, check=True).stdout
    exported = set(re.findall(r"\bT (lfm3_hip_\w+)", out))
    assert names and not [n for n in names if n not in exported]
    assert sorted(so.SIGNATURES) == names


def refused(lib, rc, word):
    assert rc == -1 and word in lib.kv800_hip_last_error(), lib.kv800_hip_last_error()


def test_chunk_meta_host_checks(lib):
    f = lambda **k: lib.kv800_hip_chunk_meta(*{**dict(bt=A, bs=4, np=4, lens=A, ql=A, R=2, ebs=64, tok=4, held=None, free=None, nf=0,
                                                      taken=None, ho=None, to=None, qsl=A, slot=A, pos=A, row=A, l32=A, s=None), **k}.values())
    for k in (dict(R=0), dict(ebs=0), dict(np=5), dict(tok=-1), dict(bt=None), dict(lens=None), dict(ql=None), dict(qsl=None),
              dict(slot=None), dict(l32=None), dict(held=A), dict(held=A, free=A, nf=-1, taken=A, ho=2 * A, to=2 * A),
              dict(held=A, free=A, nf=3, taken=A, ho=A, to=2 * A), dict(held=A, free=A, nf=3, taken=A, ho=2 * A, to=A)):
        refused(lib, f(**k), b"chunk_meta")


def paged(**k):
    p = kh.Paged(qpool=A, boff=A, boff_stride=4, epool=A, eoff=A, eoff_stride=4, ebs=64, e_hs=256, e_ts=1024, e_v=128, N=A, NQ=A,
                 nqmax=4, win=0)
    for n, v in k.items():
        setattr(p, n, v)
    return p


def test_decode_chunk_host_checks(lib):
    ws = lib.kv800_hip_decode_chunk_workspace(2, 8, 4)
    assert ws > 0 and lib.kv800_hip_decode_chunk_workspace(2, 8, 0) == 0 and lib.kv800_hip_decode_chunk_workspace(0, 0, 4) == 0
    assert lib.kv800_hip_decode_chunk_workspace(200, 800, 4) > ws

    def f(P=None, **k):
        a = {**dict(q=A, qsl=A, R=2, T=8, cos=A, sin=A, rr=512, cs2=A, qb=1 << 20, ee=1 << 20, se=0, out=A, ws=A, wsb=ws, s=None), **k}
        return lib.kv800_hip_decode_chunk(ctypes.byref(paged(**(P or {}))), *a.values())
    assert f(T=0) == 0
    for P, k in ((None, dict(R=0)), (None, dict(R=-1)), (None, dict(T=-1)), (None, dict(q=None)), (None, dict(qsl=None)),
                 (None, dict(out=None)), (None, dict(q=A + 2)), (None, dict(out=A + 8)), (None, dict(cos=None)),
                 (None, dict(cos=None, sin=None)), (None, dict(cos=A + 2)), (None, dict(rr=0)), (None, dict(cs2=None)),
                 (None, dict(qb=51199)), (None, dict(ws=None)), (None, dict(ws=A + 8)), (None, dict(wsb=ws - 1)),
                 (dict(epool=None), {}), (dict(eoff=None), {}), (dict(N=None), {}), (dict(NQ=None), {}), (dict(ebs=0), {}),
                 (dict(eoff_stride=0), {}), (dict(win=-1), {}), (dict(win=1 << 31), {}), (dict(nqmax=-1), {}), (dict(e_ts=1020), {}),
                 (dict(e_hs=4), {}), (dict(e_v=1), {}), (dict(qpool=None), {}), (dict(boff=None), {}), (dict(qpool=A + 4), {}),
                 (dict(win=256, sk=A), {}), (dict(win=256, sk=A, sv=A + 2, skoff=A, svoff=A), {}), (None, dict(rr=1 << 24))):
        refused(lib, f(P, **k), b"decode_chunk")


def test_conv_host_checks(lib):
    f = lambda **k: lib.lfm3_hip_conv_chunk(*{**dict(x=A, st=48, w=A, state=A, qsl=A, R=1, T=4, H=16, out=A, taps=A, s=None), **k}.values())
    assert f(T=0) == 0
    for k in (dict(R=0), dict(T=-1), dict(H=0), dict(H=12), dict(st=47), dict(st=40), dict(st=52), dict(x=None), dict(w=None),
              dict(state=None), dict(qsl=None), dict(out=None), dict(taps=None), dict(x=A + 2), dict(state=A + 8)):
        refused(lib, f(**k), b"conv_chunk")
    f = lambda **k: lib.lfm3_hip_conv_commit(*{**dict(state=A, taps=A, qsl=A, kept=A, R=1, T=4, H=16, s=None), **k}.values())
    assert f(T=0) == 0
    for k in (dict(R=0), dict(T=-1), dict(H=4), dict(state=None), dict(taps=None), dict(qsl=None), dict(kept=None), dict(taps=A + 4)):
        refused(lib, f(**k), b"conv_commit")


def test_verify_host_checks(lib):
    ws = lib.lfm3_hip_verify_workspace(2, 4, 100)
    assert ws > 0 and lib.lfm3_hip_verify_workspace(2, 0, 100) == 0
    f = lambda **k: lib.lfm3_hip_verify_drafts(*{**dict(x=A, ld=100, tok=A, qsl=A, temp=A, u=A, un=A, q=None, ldq=0, R=2, T=4, V=100, out=A,
                                                        cnt=A, ws=A, wsb=ws, s=None), **k}.values())
    for k in (dict(R=0), dict(T=-1), dict(V=0), dict(V=1 << 31), dict(ld=99), dict(q=A, ldq=99), dict(x=None), dict(tok=None),
              dict(qsl=None), dict(temp=None), dict(u=None), dict(un=None), dict(out=None), dict(cnt=None), dict(ws=None),
              dict(ws=A + 8), dict(wsb=ws - 1)):
        refused(lib, f(**k), b"verify_drafts")
