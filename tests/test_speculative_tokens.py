"""speculative_loop's tokens with drafts outside the vocabulary (CPU): the embedding sees none of them, the verification all."""
from types import SimpleNamespace

import torch


def test_drafts_outside_the_vocabulary_do_not_reach_the_embedding(monkeypatch):
    from lfm3_kv800_amd import model as M
    V, R, most = 50, 2, 3
    T = R * (most + 1)
    seen = []

    class Attention:
        lens, nmax = torch.tensor([10, 20]), 100

        def thaw(self):
            pass

        def begin_chunk(self, lens, ql, tokens, most, bound):
            qsl = torch.cat([torch.zeros(1, dtype=torch.int64), ql.long().cumsum(0)])
            row = torch.searchsorted(qsl[1:], torch.arange(tokens), right=True)
            return SimpleNamespace(qsl=qsl, row=torch.where(row < R, row, 0))

    class Model:
        cfg = SimpleNamespace(vocab=V)
        embed = torch.randn(V, 4)

        def chunk(self, tok, meta):
            assert int(tok.min()) >= 0 and int(tok.max()) < V
            return self.embed[tok] @ self.embed.T

        def commit(self, kept):
            pass

    def verify(logits, tok, qsl, temperature, u, u_next, q):
        seen.append(tok.tolist())
        out = torch.full((T,), -1)
        out[qsl[:-1]] = 7
        return out, torch.ones(R, dtype=torch.int32)
    monkeypatch.setattr(M.so, "verify_drafts", verify)
    drafts = torch.tensor([[V, 1 << 40, -5], [3, -(1 << 40), V + 9]])
    rows, counts = M.speculative_loop(Model(), Attention(), torch.tensor([1, 2]), 2,
                                      lambda last, lens: (drafts, torch.tensor([1, 2], dtype=torch.int32), None), most)
    assert [r.tolist() for r in rows] == [[7, 7], [7, 7]] and counts.tolist() == [[1, 1], [1, 1]]
    assert seen[0][:5] == [1, V, 2, 3, -(1 << 40)]
