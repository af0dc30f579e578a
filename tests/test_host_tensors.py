"""Tensors left on the host are refused before any launch (CPU; every entry of the library is a stand-in that fails the test)."""
import pytest
import torch

import lfm3_kv800_amd.int8_ops as i8
import lfm3_kv800_amd.kv800_hip as kh
import lfm3_kv800_amd.kv8 as kv8


class NoLaunch:
    def __getattr__(self, name):
        def entry(*a):
            pytest.fail(f"{name} reached with host tensors")
        if name.endswith("_workspace"):
            return lambda *a: 64
        entry.restype = entry.argtypes = None
        return entry


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    lib = NoLaunch()
    monkeypatch.setattr(kh, "ops", lambda: lib)
    for m in (kv8, i8):
        monkeypatch.setattr(m, "_lib", lambda: lib)


def bf(*s):
    return torch.ones(*s, dtype=torch.bfloat16)


def test_products():
    for w in (bf(64, 64), bf(64, 64)[:, 8:16], torch.ones(64, 64, dtype=torch.bfloat16, device="cpu:0")):
        with pytest.raises(ValueError, match="GPU"):
            i8.quantize_rows(w)
        with pytest.raises(ValueError, match="GPU"):
            i8.Weight8(w)
    with pytest.raises(ValueError, match="GPU"):
        i8.Weight8(torch.ones(64, 64, dtype=torch.int8), torch.ones(64))


def test_cache():
    c = kv8.Cache8.empty(2, 2, 64, 64, "cpu")
    bt, lens, qsl = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int64), torch.tensor([0, 1])
    cos = bf(9, 8)
    for call in (lambda: kv8.append(c, bf(1, 2, 64), bf(1, 2, 64), bt, lens, qsl), lambda: kv8.append(c, bf(1, 2, 64), bf(1, 2, 64), bt, lens, qsl, cos, cos),
                 lambda: kv8.append(c, bf(0, 2, 64), bf(0, 2, 64), bt[:0], lens[:0], qsl[:1]), lambda: kv8.attend(c, bf(1, 4, 64), bt, lens, qsl),
                 lambda: kv8.attend(c, bf(0, 4, 64), bt[:0], lens[:0], qsl[:1]), lambda: kv8.dequantize(c)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_800h_entries():
    """The launches of kv800_hip go by the same question."""
    kv = bf(1, 256, 4, 128)
    for call in (lambda: kh.quantize_blocks(kv, kv), lambda: kh.dequantize_blocks(torch.zeros(1, 51200, dtype=torch.uint8)),
                 lambda: kh.step_meta(torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int64), 64)):
        with pytest.raises(ValueError, match="GPU"):
            call()
