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


def test_a_table_missing_at_capture_is_made_once(hip):
    """Calls of one capture share the table that the first of them makes; it belongs to that capture, and every replay fills it."""
    c = ref.Cache(hip, [700, 1400], [4, 3], seed=73)
    want = c.want(hip)
    hip.rope_pairs(torch.ones_like(c.cos), c.sin)     # the library's first launch
    tables, graphs = [], []
    for _ in range(2):
        def step():
            a = hip.rope_pairs(c.cos, c.sin)
            outs = [hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin) for _ in range(2)]
            b = hip.rope_pairs(c.cos, c.sin)
            assert b is a
            tables.append(a)
            return outs
        graphs.append(capture(step))
    assert tables[0] is not tables[1]
    eager = hip.rope_pairs(c.cos, c.sin)
    assert eager is not tables[0] and eager is not tables[1] and not hip._BUILDING
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, "eager after the captures")
    for k in range(3):
        for (g, outs), t in zip(graphs, tables):
            for x in (*outs, t):
                x.zero_()
            g.replay()
            hip.rope_pairs(torch.rand_like(c.cos), c.sin)
            torch.cuda.synchronize()
            for out in outs:
                check(out, want, f"replay {k}")


def test_tables_changed_inside_a_capture(hip):
    """A table written between two calls of a capture is paired anew by the second."""
    c = ref.Cache(hip, [700, 1400], [4, 3], seed=74)
    cos, want = c.cos.clone(), c.want(hip)
    hip.rope_pairs(torch.ones_like(c.cos), c.sin)

    def step():
        c.cos.zero_()
        hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
        c.cos.copy_(cos)
        return hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
    g, out = capture(step)
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        check(out, want, f"replay {k}")
