"""speculative_loop refuses steps that the caches have no room for before the first of them (CPU)."""
import pytest
import torch


class Attention:
    lens, nmax = torch.tensor([10, 90]), 100


class Model:
    def chunk(self, *a):
        raise AssertionError("a step was taken")


def test_room_is_checked_before_the_first_step():
    from lfm3_kv800_amd import model as M

    def draft(last, lens):
        raise AssertionError("drafts were asked for")
    with pytest.raises(ValueError, match="102"):
        M.speculative_loop(Model(), Attention(), torch.tensor([1, 2]), 3, draft, 3)
    with pytest.raises(AssertionError, match="asked for"):
        M.speculative_loop(Model(), Attention(), torch.tensor([1, 2]), 2, draft, 3)
