"""kv800_hip.rope_pairs around graph capture: how long its tables live and how often they are made."""
import gc
import weakref

import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import check

pytestmark = pytest.mark.gpu


def capture(f):
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


def evict(hip, sin):
    for _ in range(9):
        hip.rope_pairs(torch.rand_like(sin), sin)


def test_a_captured_table_lives_as_long_as_what_it_is_made_of(hip):
    c = ref.Cache(hip, [700, 1400], [4, 3], seed=71)
    want, other = c.want(hip), ref.Cache(hip, [700], [2], seed=72)
    table = weakref.ref(hip.rope_pairs(c.cos, c.sin))
    g, out = capture(lambda: hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin))
    evict(hip, c.sin.clone())
    hip.rope_pairs(other.cos, other.sin)
    capture(lambda: hip.decode_chunk(other.P, other.q, other.qsl, other.cos, other.sin))
    gc.collect()
    assert table() is not None                       # the graph may be replayed
    out.zero_()
    g.replay()
    check(out, want, "a table that only the graph reads")
    before = len(hip._CAPTURED)
    del g, out
    cos = c.cos[:]                                   # another name for the storage keeps it
    c.cos = None
    capture(lambda: hip.decode_chunk(other.P, other.q, other.qsl, other.cos, other.sin))
    gc.collect()
    assert table() is not None and len(hip._CAPTURED) == before
    del cos
    capture(lambda: hip.decode_chunk(other.P, other.q, other.qsl, other.cos, other.sin))
    gc.collect()
    assert table() is None and len(hip._CAPTURED) == before - 1
