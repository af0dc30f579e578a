"""The tests' mirror of kv8.attend's rules against the library's workspace sizes (CPU)."""
import random

import torch

import kv8_reference as ref
from kv8_plan import plan
from test_gpu_kv8 import rows
from test_gpu_kv8_paths import want_of
from test_kv8_abi import desc, lib


def test_mirror(lib):
    rng, seen = random.Random(1), set()
    for _ in range(20000):
        kv, blocks, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4]), rng.choice([64, 128])
        heads = kv * rng.choice([1, 2, 3, 4, 8, 16])
        R = int(2 ** rng.uniform(0, 9.5))
        T = max(1, int(R * 2 ** rng.uniform(-2, 7)))
        cols = int(2 ** rng.uniform(0, 12)) // blocks + 1
        window = rng.choice([0, 0, 1, 256, int(2 ** rng.uniform(0, 13))])
        want = plan(kv, blocks, dim, heads, R, T, cols, window)
        d = desc(kv_heads=kv, blocks=blocks, dim=dim, page_stride=kv * blocks * 2 * 64 * dim, exp_stride=2 * kv * blocks)
        assert lib.kv8_hip_attend_workspace(d, heads, R, T, cols, window) == want[3], (kv, blocks, dim, heads, R, T, cols, window)
        seen.add((want[0], want[1], want[0] == "PROMPT" and want[2] > 1))
    assert seen == {("LISTED", 16, False), ("LISTED", 32, False), ("DIRECT", 16, False), ("PROMPT", 128, False), ("PROMPT", 128, True)}


def test_reference_of_a_row_at_once():
    """The paths' reference is kv8_reference.attend."""
    data, exps, bt, lens, qsl, T, g = rows(None, 3, [100, 0, 64], [3, 2, 0], 2, 64, 64, pad=1)
    q = torch.randn(T, 4, 64, generator=g).to(torch.bfloat16)
    for window in (0, 50):
        for a, b in zip(want_of(data, exps, q, bt, lens, qsl, window), ref.attend(data, exps, q, bt, lens, qsl, window)):
            assert torch.allclose(a, b, rtol=1e-12, atol=1e-18)
