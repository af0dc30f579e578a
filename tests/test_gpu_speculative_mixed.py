"""speculative_loop between other ways to decode the same caches."""
import pytest
import torch

from test_gpu_speculative import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("after", ["eager", "graph"])
def test_between_recorded_and_eager_steps(hip, after):
    """Steps of a recorded graph, speculative steps, further steps: the same tokens as with eager steps throughout."""
    from lfm3_kv800_amd import model as M
    first, most = torch.tensor([1, 2, 3], device="cuda"), 2
    runs = []
    for graph in (False, True):
        model, attn = build([500, 129, 1020], 40)
        a = M.decode_loop(model, attn, first, 4, graph=graph)

        def draft(last, lens):
            d = (last[:, None] + torch.arange(1, most + 1, device="cuda")) % 8192
            return d, torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda"), None
        rows, counts = M.speculative_loop(model, attn, a[-1], 3, draft, most)
        b = M.decode_loop(model, attn, torch.stack([r[-1] for r in rows]), 5, graph=graph and after == "graph")
        runs.append((a.tolist(), [r.tolist() for r in rows], counts.tolist(), b.tolist(), attn.lens.tolist()))
    assert runs[0] == runs[1]


def test_a_recorded_step_behind_a_speculative_one_is_refused(hip):
    from lfm3_kv800_amd import model as M
    model, attn = build([300, 20], 20)
    first = torch.tensor([1, 2], device="cuda")
    dg = M.DecodeGraph(model, attn, first, 6)
    dg.step()
    empty = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    M.speculative_loop(model, attn, dg.tokens.clone(), 2, lambda last, lens: (empty, torch.zeros(2, device="cuda"), None), 0)
    assert attn.lens.tolist() == [304, 24]
    with pytest.raises(RuntimeError):
        dg.step()
    M.decode_loop(model, attn, first, 2)
    assert attn.lens.tolist() == [306, 26]
