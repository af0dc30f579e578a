"""Chunk steps whose tokens make a block eligible and are then taken back, through the cache layers: the sub-blocks' bytes and every
step's attention against a 64-bit reference that is built from the rows as they were written. Tolerance as in test_gpu_chunk.py."""
import random

import pytest
import torch

import chunk_reference as ref
from test_gpu_chunk import check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("lens0,most,steps", [([380, 379, 383, 636, 250, 3], 5, 8), ([256, 300, 500, 1, 383, 512, 257], 128, 5)])
@pytest.mark.parametrize("layer", [6, 2])                # quantized; window + sinks
def test_drafts_taken_back_across_a_flush(hip, lens0, most, steps, layer):
    from lfm3_kv800_amd import model as M
    R, rng = len(lens0), random.Random(most + layer)
    g = torch.Generator(device=DEV).manual_seed(91)
    new = lambda n: (torch.randn(n, 4, 128, generator=g, device=DEV)).to(torch.bfloat16)
    attn = M.PagedAttention800(lens0, steps * most, DEV, seed=92)
    K, V = [new(n) for n in lens0], [new(n) for n in lens0]
    attn.fill(lambda l, r, p0, p1: (K[r][p0:p1], V[r][p0:p1]))
    host = attn.layers[layer]
    crossed = taken_back = 0
    for s in range(steps):
        prev = [k.shape[0] for k in K]
        ql = [rng.choice([1, most, rng.randint(1, most)]) for _ in range(R)]
        T = sum(ql) + 2
        lens = torch.tensor([p + c for p, c in zip(prev, ql)], device=DEV)
        m = attn.begin_chunk(lens, torch.tensor(ql, dtype=torch.int32, device=DEV), T, most, lens.cpu())
        k, v = new(T), new(T)
        q = (2 * torch.randn(T, 16, 128, generator=g, device=DEV)).to(torch.bfloat16)
        out = attn.attend(layer, q, k, k, v)
        qsl, want = m.qsl.tolist(), torch.zeros(T, 16, 128, dtype=torch.float64, device=DEV)
        for r in range(R):
            a, b = qsl[r], qsl[r + 1]
            KR, VR = torch.cat([K[r], k[a:b]]), torch.cat([V[r], v[a:b]])
            n, pos = prev[r] + ql[r], torch.arange(prev[r] + ql[r], device=DEV)
            KD, VD = KR.double(), VR.double()
            if layer == 6:
                nb = ref.nq(n)                           # what the step has flushed
                if nb:
                    sb = hip.quantize_blocks(KR[:256 * nb].view(nb, 256, 4, 128), VR[:256 * nb].view(nb, 256, 4, 128))
                    for j in range(nb):
                        page = host.qv[int(attn.qbt[r, 256 * j // 1280])]
                        at = 256 * j % 1280 // 256 * 51200
                        assert torch.equal(page[at:at + 51200], sb[j]), (s, r, j)
                crossed += nb > ref.nq(prev[r] + 1)
                nb = ref.nq(prev[r] + 1)                 # what its queries read quantized
                if nb:
                    x, y = hip.dequantize_blocks(sb[:nb])
                    KD = torch.cat([x.double().view(-1, 4, 128), KD[256 * nb:]])
                    VD = torch.cat([y.double().view(-1, 4, 128), VD[256 * nb:]])
            KD = ref.rotate(KD, pos, attn.cos, attn.sin)
            want[a:b] = ref.attend(q[a:b], KD, VD, pos, pos[prev[r]:], *((256, 4) if layer == 2 else (0, 0)))
        check(out, want, f"step {s}, layer {layer}")
        for r in range(R):                               # some of the tokens stay
            a, kept = qsl[r], rng.choice([1, rng.randint(1, ql[r]), ql[r]])
            taken_back += ref.nq(prev[r] + kept) < ref.nq(prev[r] + ql[r])
            K[r], V[r] = torch.cat([K[r], k[a:a + kept]]), torch.cat([V[r], v[a:a + kept]])
    assert layer == 2 or (crossed and taken_back), (crossed, taken_back)
