"""decode_chunk's tables of blocks and pages: rows of any stride, widths apart from it, positions past the widths. Tolerance as in
test_gpu_chunk.py."""
import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import check

pytestmark = pytest.mark.gpu


def column(t):
    """A one-row table as a transposed column: shape (1, n), strides (1, 1)."""
    x = t.reshape(-1, 1).contiguous().T
    assert x.shape[0] == 1 and x.stride() == (1, 1)
    return x


@pytest.mark.parametrize("win", [0, 256])
def test_one_row_of_any_stride(hip, win):
    c = ref.Cache(hip, [1500], [5], ebs=64, win=win, seed=51)
    want = c.want(hip)
    c.P.eoff, c.P.boff = column(c.P.eoff), column(c.P.boff)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, f"a column as the table, window {win}")


def test_one_row_of_any_stride_in_the_decode(hip):
    c = ref.Cache(hip, [1500], [1], ebs=64, seed=52)
    want = hip.decode(c.P, c.q, c.cos, c.sin)
    c.P.eoff, c.P.boff = column(c.P.eoff), column(c.P.boff)
    assert torch.equal(hip.decode(c.P, c.q, c.cos, c.sin), want)


def last_columns(t, n, fill):
    """The first n columns of t as the last ones of a wider table, whose other entries `fill` leads elsewhere: behind the last
    row's there is no further entry."""
    wide = torch.full((t.shape[0], n + 3), fill, dtype=t.dtype, device=t.device)
    wide[:, 3:] = t[:, :n]
    return wide[:, 3:]


@pytest.mark.parametrize("launches", [1, 2])
@pytest.mark.parametrize("prev,new", [([1500, 800, 2100], [4, 2, 3]), ([1500, 800, 2100], [7, 2, 13])])
def test_positions_past_columns_of_a_wider_table(hip, prev, new, launches):
    """Blocks and pages that a row's table does not hold are left out, whatever stands behind it in the wider one."""
    c = ref.Cache(hip, prev, new, ebs=64, seed=53)
    if launches == 2:
        c.P.nqmax = 8 * torch.cuda.get_device_properties(0).multi_processor_count // len(prev) + 1
    nb, ne = max(c.nq) - 2, 1472 // 64
    c.P.boff, c.P.eoff = last_columns(c.P.boff, nb, 0), last_columns(c.P.eoff, ne, 0)
    lost = lambda r, p: ((p >= 256 * nb) & (p < 256 * c.nq[r])) | (p >= 64 * ne)
    assert any(bool(lost(r, torch.arange(c.N[r])).any()) for r in range(3))
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip, lost), f"past a wider table's columns, {launches} launches")


def test_window_past_columns_of_a_wider_table(hip):
    c = ref.Cache(hip, [700, 390, 90], [4, 9, 2], ebs=40, win=256, seed=54)
    ne = 640 // 40
    c.P.eoff = last_columns(c.P.eoff, ne, 0)
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), c.want(hip, lambda r, p: p >= 40 * ne), "a window past its table")


def test_rows_that_share_a_table(hip):
    """An expanded table (row stride 0): every row reads the same pages."""
    c = ref.Cache(hip, [700], [4], ebs=64, seed=55)
    want = c.want(hip)
    c.P.N, c.P.NQ = c.P.N.repeat(3), c.P.NQ.repeat(3)
    c.P.eoff, c.P.boff = c.P.eoff.expand(3, -1), c.P.boff.expand(3, -1)
    qsl = torch.tensor([0, 4, 8, 12], device=c.dev)
    check(hip.decode_chunk(c.P, c.q.repeat(3, 1, 1), qsl, c.cos, c.sin), want.repeat(3, 1, 1), "a shared table")


def test_tables_without_columns_are_refused(hip):
    c = ref.Cache(hip, [700], [4], ebs=64, seed=56)
    for name in ("eoff", "boff"):
        keep = getattr(c.P, name)
        setattr(c.P, name, keep[:, :0])
        with pytest.raises((RuntimeError, ValueError)):
            hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin)
        setattr(c.P, name, keep)


def test_lengths_far_past_the_tables(hip):
    """A length of 2^31 - 1 over a short table: its positions alone, without a walk over the others."""
    far = (1 << 31) - 1
    c = ref.Cache(hip, [1500, 300], [4, 9], ebs=32, seed=57)
    want = c.want(hip)
    K, V, pos = c.row(hip, 0)
    want[:4] = ref.attend(c.q[:4], K, V, pos, torch.arange(far - 4, far, device=c.dev))
    c.P.N[0] = far
    check(hip.decode_chunk(c.P, c.q, c.qsl, c.cos, c.sin), want, "a far length")
    w = ref.Cache(hip, [700, 300], [4, 9], ebs=32, win=256, sinks=True, seed=58)
    want = w.want(hip)
    K, V = w.P.sk[0].double(), w.P.sv[0].double()
    pos = torch.arange(4, device=w.dev)
    want[:4] = ref.attend(w.q[:4], ref.rotate(K, pos, w.cos, w.sin), V, pos, pos + 1000)
    w.P.N[0] = far
    check(hip.decode_chunk(w.P, w.q, w.qsl, w.cos, w.sin), want, "a far length of a window")
