"""Inputs of conv_chunk, conv_commit and verify_drafts as views that torch counts as contiguous and the kernels cannot read as they
are: one row of any stride, data off a 16-byte boundary. The same bits as from a fresh copy."""
import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import conv_case, verify_case

pytestmark = pytest.mark.gpu


def shifted(t):
    """A contiguous copy of t two bytes or four behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    view = flat[1:].view(t.shape)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("width", [48, 53, 56])
def test_conv_of_rows_of_a_wider_product(hip, T, width):
    from lfm3_kv800_amd import spec_ops as so
    bcx, w, state, qsl = conv_case([T], 16, 0, seed=T)
    q = torch.tensor(qsl, device="cuda")
    want, taps = so.conv_chunk(bcx, w, state, q)
    wide = torch.full((T + 2, width), float("nan"), dtype=torch.bfloat16, device="cuda")
    for at in (0, 1):
        wide[at:at + T, :48] = bcx
        for x in (wide[at:at + T], wide[at:at + T, :48], bcx.T.contiguous().T, shifted(bcx)):
            out, tp = so.conv_chunk(x, w, state, q)
            assert torch.equal(out, want) and torch.equal(tp, taps), (at, x.stride(), x.storage_offset())
    assert torch.equal(so.conv_chunk(bcx, shifted(w), state, q)[0], want)
    kept = torch.tensor([T], dtype=torch.int32, device="cuda")
    a, b = state.clone(), state.clone()
    so.conv_commit(a, taps, q, kept)
    so.conv_commit(b, shifted(taps), q, kept)
    assert torch.equal(a, b) and not torch.equal(a, state)


@pytest.mark.parametrize("T", [1, 4])
@pytest.mark.parametrize("V", [1, 9, 1001, 20001])
def test_verify_of_columns(hip, T, V):
    """Logits as a transposed product, (V, T).T: for one token torch calls it contiguous with strides (1, 1)."""
    from lfm3_kv800_amd import spec_ops as so
    x, tokens, qsl, temp, u, un, q = verify_case([T], V, 3, True, (0.9,))
    want = ref.verify(x, tokens, qsl, temp, u, un, q), ref.verify(x, tokens, qsl, temp, u, un)
    d = [t.cuda() for t in (tokens, torch.tensor(qsl), temp, u, un)]
    x, q = x.cuda(), q.cuda()
    columns = lambda t: torch.empty(V, T, dtype=t.dtype, device="cuda").copy_(t.T).T
    for f in (columns, shifted):
        for p, w in zip((f(q), None), want):
            out, count = so.verify_drafts(f(x), *d, p)
            assert (out.tolist(), count.tolist()) == w, (f, p is None)


def test_a_state_off_its_boundary_is_refused(hip):
    """The state is moved on in place, so it cannot be copied."""
    from lfm3_kv800_amd import spec_ops as so
    bcx, w, state, qsl = conv_case([3], 16, 0)
    q, kept = torch.tensor(qsl, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    _, taps = so.conv_chunk(bcx, w, state, q)
    with pytest.raises(RuntimeError):
        so.conv_commit(shifted(state), taps, q, kept)
