"""Decode loop of an LFM3-1.7B-shaped model whose attention layers run on the 800h path (C5), without
vLLM.

The layer stack follows the reference's vLLM model (vllm_model.py:542-653) and its attention routing with
LFM3_KV800=1 (vllm_model.py:268-304): 24 layers of width 2048, each `h += post_norm(op(norm(h)))` then
`h += post_ffn_norm(ffn(ffn_norm(h)))` (sandwich norms, vllm_model.py:446-471), then a final norm and the tied LM head.
  * 13 gated short-conv layers (width 7, vllm_model.py:327-431): in_proj -> B, C, x; y = C * conv(B * x); out_proj.
  * 6 full-attention layers, 16 query / 4 KV heads of 128, QK RMSNorm per head, RoPE theta 1e6 on 32 of the 64
    frequencies (zero tail), per-head sigmoid output gate (vllm_model.py:195-304): quantized 6, 10, 14, 22 and window +
    sinks 2, 18 on the 800h caches (vllm_cache.KV800DecodeLayer), keys handed over before RoPE.
  * 5 native sliding layers 4, 8, 12, 16, 20 (RoPE theta 1e4 on all frequencies, window 256) on exact window caches
    (vllm_cache.KV800SlideLayer), keys handed over after RoPE.
The vocabulary and feed-forward sizes are not in the reference (its weights are not available offline): 65,536 and
8,192 here, about 1.67 B parameters. Weights are random N(0, 0.02) in bf16, norm weights 1.

With int8=True the layers' products run in 8-bit integers (int8_ops), and PagedAttention8 keeps every attention layer's keys and values
in 8 bits (kv8): all 6 full-attention layers over their whole history, the sliding layers over their window.

Attention goes through an object with begin_step() -> the new tokens' positions and attend(layer, q, k_pre, k_post, v)
-> (R, 16, 128): PagedAttention800 (below) keeps vLLM's page geometry and runs every layer on libkv800_hip.so; tests
substitute an oracle implementation to check the logits. Between the GEMMs, the model's elementwise work runs on the
fused kernels of model_ops (include/lfm3_model.h). DecodeGraph captures one whole decode step (metadata, 24 layers,
greedy token) as a HIP graph and replays it per step."""
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import int8_ops as i8
from . import kv8, kv800, kv800_hip
from . import model_ops as mo
from . import spec_ops as so
from . import vllm_cache as vc

CONV, FULL, SLIDE = "conv", "full", "slide"
EXACT_GROUPS = {"A": (2, 10, 18), "B": (6, 14, 22)}       # exact KV groups of the full layers (sliding window 640)
SLIDE_GROUPS = {"C": (4, 12, 20), "D": (8, 16)}           # KV groups of the native sliding layers (window 256)


@dataclass
class Lfm3Config:
    hidden: int = 2048
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 128
    ffn: int = 8192
    vocab: int = 65536
    layers: int = 24
    conv_len: int = 7
    window: int = 256
    eps: float = 1e-5

    def layer_type(self, l):
        if l in vc.QUANT_LAYERS or l in vc.WINDOW_LAYERS:
            return FULL
        if l in vc.SLIDE_LAYERS:
            return SLIDE
        return CONV


def model_rope_tables(theta, angles, n, device):
    """(cos, sin) (n, 64) bf16 of the model's neox RoPE (vllm_model.py:106-151): frequency f < angles is
    theta^(-2f/128), the rest 0 (cos 1, sin 0); angles in fp32, then bf16, as the reference's cos / sin caches."""
    inv = 1.0 / (theta ** (torch.arange(0, 2 * angles, 2, dtype=torch.float32) / 128))
    inv = torch.cat((inv, torch.zeros(64 - angles)))
    fr = torch.arange(n, dtype=torch.float32)[:, None] * inv[None]
    return fr.cos().to(torch.bfloat16).to(device), fr.sin().to(torch.bfloat16).to(device)


def kernel_tables(n, device):
    """(cos, sin) (n, 32) bf16 of the full layers' 32 rotating frequencies, the tables the decode kernels read
    (vllm_attn.py:147-159)."""
    inv = 1.0 / (1e6 ** (torch.arange(0, 64, 2, dtype=torch.float32) / 128))
    fr = torch.arange(n, dtype=torch.float32)[:, None] * inv[None]
    return fr.cos().to(torch.bfloat16).to(device), fr.sin().to(torch.bfloat16).to(device)


def glu_rows(rows):
    """Whether the fused up-projection + gated activation (128-row tiles) is used for a batch of `rows`: measured
    on MI355X against hipBLASLt + silu_mul at hidden 2048, ffn 8192 (device time per layer): 192 rows 28.7 vs 29.8 us,
    256 rows 25.7 vs 33.2, 320 rows 38.6 vs 35.2 (a third row tile a quarter full), 398 rows 41.1 vs 41.7, 128 rows
    23.1 vs 22.1."""
    return 128 < rows <= 256 or rows > 384


def product(x, w):
    """x W^T, (R, N) bf16, of a bf16 matrix or an int8_ops.Weight8."""
    return i8.linear8(x, w) if isinstance(w, i8.Weight8) else F.linear(x, w)


class Lfm3Decoder:
    """Random-init LFM3-shaped model for batched decode: step(tokens) appends one token to every row and returns the
    logits. The dense products are torch GEMMs; everything between them is one fused HIP kernel (model_ops): the
    sandwich norms with the residual add, the q / k norms with RoPE, the short-conv step, the gated activation and
    the attention output gate. The FFN's up-projection and gated activation run as one HIP GEMM (model_ops.linear on
    a [g | u] weight) at the batch sizes where it beats the library product plus the activation kernel (glu_rows).
    conv_state: per conv layer (R, hidden, conv_len - 1) bf16. max_pos bounds the positions of the model's RoPE
    tables. int8: the layers' weights are quantized by rows and their products take tokens rounded to 8 bits (int8_ops.linear8, the
    gated activation in the product's epilogue); embedding and LM head stay bf16."""

    def __init__(self, cfg: Lfm3Config, attention, rows, device, seed=0, max_pos=65536, int8=False):
        self.cfg, self.attn, self.R, self.dev = cfg, attention, rows, device
        g = torch.Generator(device=device).manual_seed(seed)
        H, D, G = cfg.hidden, cfg.head_dim, cfg.heads

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) * 0.02).to(torch.bfloat16)

        ones = lambda n: torch.ones(n, dtype=torch.bfloat16, device=device)
        self.embed = w(cfg.vocab, H)
        self.final_norm = ones(H)
        self.tables = {FULL: model_rope_tables(1e6, 32, max_pos, device),
                       SLIDE: model_rope_tables(1e4, 64, max_pos, device)}
        self.int8 = bool(int8)
        self.fused_ffn = not self.int8 and glu_rows(rows)
        self.layers = []
        for l in range(cfg.layers):
            t = cfg.layer_type(l)
            L = {"type": t, "norm": ones(H), "post_norm": ones(H), "ffn_norm": ones(H), "post_ffn_norm": ones(H),
                 "w13": w(2 * cfg.ffn, H), "w2": w(H, cfg.ffn)}
            if self.fused_ffn:
                L["w13p"] = mo.PackedWeight(L["w13"], glu=True)
            if t == CONV:
                L.update(in_proj=w(3 * H, H), conv=w(H, cfg.conv_len), out_proj=w(H, H),
                         state=torch.zeros(rows, H, cfg.conv_len - 1, dtype=torch.bfloat16, device=device))
            else:
                # q, k, v and the 16 output-gate logits from one product: rows [q | k | v | gate]
                L.update(qkvg=torch.cat((w((G + 2 * cfg.kv_heads) * D, H), w(G, H))), q_norm=ones(D), k_norm=ones(D),
                         o_proj=w(H, G * D))
            if self.int8:
                for name in ("w13", "w2", "in_proj", "out_proj", "qkvg", "o_proj"):
                    if name in L:
                        L[name] = i8.Weight8(L[name], gated=name == "w13")
            self.layers.append(L)

    def randomize_conv_states(self, seed):
        g = torch.Generator(device=self.dev).manual_seed(seed)
        for L in self.layers:
            if L["type"] == CONV:
                L["state"].copy_(torch.randn(L["state"].shape, generator=g, device=self.dev) * 0.1)

    def _conv(self, L, n, qsl=None):
        bcx = product(n, L["in_proj"])
        if qsl is None:
            y = mo.conv_step(bcx, L["conv"], L["state"])
        else:
            y, L["taps"] = so.conv_chunk(bcx, L["conv"], L["state"], qsl)
        return product(y, L["out_proj"])

    def _attention(self, l, L, n, pos):
        cfg = self.cfg
        qkvg = product(n, L["qkvg"])                                                   # (R, 3088)
        cos, sin = self.tables[L["type"]]
        q, k_pre, k_rot, v = mo.qkv_post(qkvg, L["q_norm"], L["k_norm"], cos, sin, pos, cfg.eps)
        o = self.attn.attend(l, q, k_pre, k_rot, v)
        o = mo.gate_mul(o, qkvg[:, (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim:])
        return product(o.reshape(o.shape[0], -1), L["o_proj"])

    def step(self, tokens, pos, fp32=True):
        """tokens (R,) int64, pos (R,) int64 the new tokens' positions (device); the attention object's begin_step
        has been called with the rows' lengths including this token. Returns (R, vocab) logits, fp32 (the bf16 LM-head
        output widened) or, with fp32=False, bf16."""
        logits = self._layers(tokens, pos, None, self.fused_ffn)
        return logits.float() if fp32 else logits

    def chunk(self, tokens, meta):
        """Logits (T, vocab) bf16 behind every token of a step whose rows bring any number of tokens: tokens (T,) int64, row
        after row, meta the kv800_hip.ChunkMeta that the attention object's begin_chunk returned. The conv states stay where
        they are until commit()."""
        self.qsl = meta.qsl
        return self._layers(tokens, meta.pos, meta.qsl, self.fused_ffn and glu_rows(tokens.shape[0]))

    def commit(self, kept):
        """Move the conv states on over the first kept[r] ((R,) int32) of each row's tokens of the last chunk()."""
        for L in self.layers:
            if L["type"] == CONV:
                so.conv_commit(L["state"], L["taps"], self.qsl, kept)

    def _layers(self, tokens, pos, qsl, fused_ffn):
        cfg = self.cfg
        x = self.embed[tokens]
        _, n = mo.add_rmsnorm(None, x, None, self.layers[0]["norm"], cfg.eps)
        for l, L in enumerate(self.layers):
            h = self._conv(L, n, qsl) if L["type"] == CONV else self._attention(l, L, n, pos)
            x, n = mo.add_rmsnorm(h, x, L["post_norm"], L["ffn_norm"], cfg.eps)
            if self.int8:
                a = i8.linear8(n, L["w13"])
            else:
                a = mo.linear(n, L["w13p"]) if fused_ffn else mo.silu_mul(F.linear(n, L["w13"]))
            h = product(a, L["w2"])
            nxt = self.layers[l + 1]["norm"] if l + 1 < len(self.layers) else self.final_norm
            x, n = mo.add_rmsnorm(h, x, L["post_ffn_norm"], nxt, cfg.eps)
        return F.linear(n, self.embed)

    def greedy(self, tokens, pos):
        """One step's greedy tokens (R,) int64: the first index of each row's largest logit (one HIP launch on the
        bf16 logits, the same choice as argmax over their fp32 widening)."""
        return mo.argmax(self.step(tokens, pos, fp32=False))


class PagedAttention800:
    """The model's 11 attention layers on libkv800_hip.so with vLLM's page geometry: one quant KV group (1280-token
    pages of 262,144 B) for layers 6, 10, 14, 22; exact KV groups A (2, 10, 18) and B (6, 14, 22) of ebs-token pages
    holding each row's last positions; sliding KV groups C (4, 12, 20) and D (8, 16) (window 256). Each row of an exact
    or sliding group owns a ring of `ring` shuffled physical pages and logical page p maps to its (p % ring)-th one
    (the pages a sliding-window KV group recycles): the ring holds a prompt chunk of FILL tokens plus the 384 exact
    positions before it, and the decode steps' windows.

    lens0: the rows' history lengths; steps: decode steps to provide for."""

    FILL = 2048   # prompt tokens per row per fill step (the reference's prefill chunk, vllm_attn.py:196)

    def __init__(self, lens0, steps, device, ebs=128, seed=0):
        self.dev, self.ebs = device, ebs
        self.lens = torch.tensor([int(x) for x in lens0], dtype=torch.int64)
        R = self.R = len(lens0)
        nmax = self.nmax = int(self.lens.max()) + steps + 1
        self.cos, self.sin = kernel_tables(nmax + 64, device)
        rng = torch.Generator().manual_seed(seed)
        lp = nmax // ebs + 1                                                   # logical exact pages per row

        # a fill step writes FILL positions and flushes sub-blocks starting up to 383 positions before them; a decode
        # step reads the 384 positions before its token: the ring spans both with a page to spare
        self.ring = ring = max(self.FILL, 384 + steps + 1) // ebs + 5

        def table():
            """block table (R, lp) int32: row r's logical page p -> the (p % ring)-th of its ring of shuffled pages."""
            perm = torch.randperm(R * ring, generator=rng).view(R, ring).to(torch.int32)
            return perm[:, torch.arange(lp) % ring].contiguous(), R * ring

        self.bt, npages = {}, {}
        for grp in (*EXACT_GROUPS, *SLIDE_GROUPS):
            bt, npages[grp] = table()
            self.bt[grp] = bt.to(device)
        self.bt_cpu = {g: t.cpu() for g, t in self.bt.items()}
        qlp = nmax // vc.QBLOCK + 1
        self.qbt_cpu = torch.randperm(R * qlp, generator=rng).view(R, qlp).to(torch.int32)
        self.qbt = self.qbt_cpu.to(device)
        self.group_of = {l: g for g, ls in {**EXACT_GROUPS, **SLIDE_GROUPS}.items() for l in ls}
        self.layers = {}
        for l in (2, 6, 10, 14, 18, 22):
            ev = torch.zeros(npages[self.group_of[l]], 4, ebs, 256, dtype=torch.bfloat16, device=device)
            qv = None if l in vc.WINDOW_LAYERS else torch.zeros(R * qlp, vc.QPAGE, dtype=torch.uint8, device=device)
            self.layers[l] = vc.KV800DecodeLayer(l, ev, qv)
        for l in vc.SLIDE_LAYERS:
            ev = torch.zeros(npages[self.group_of[l]], 4, ebs, 256, dtype=torch.bfloat16, device=device)
            self.layers[l] = vc.KV800SlideLayer(l, ev)
        self.metas = None
        self.lens_dev = self.lens_bound = None   # set by freeze()

    # ---- prompt history
    def fill(self, history):
        """Write every row's history into the caches through the layers' step path (vllm_cache write_step: exact rows,
        sinks of window layers in the hosts' aux areas, flush of every sub-block that becomes eligible, from the
        layer's own exact group), in prefill steps of up to FILL positions per row, as vLLM schedules prompt chunks:
        step c carries positions [c FILL, min(n, (c + 1) FILL)) of every row still short of its length n. Prompt
        attention is not computed (no queries exist for a synthetic history). history(l, r, p0, p1) -> (K, V)
        (p1 - p0, 4, 128) bf16 on the device: pre-RoPE K for full layers, post-RoPE K for sliding layers."""
        lens = self.lens
        for c0 in range(0, int(lens.max()) if self.R else 0, self.FILL):
            rows = torch.nonzero(lens > c0).flatten()
            sl = torch.clamp(lens[rows], max=c0 + self.FILL)
            ql = sl - c0
            me = {g: vc.mixed_step_meta(self.bt_cpu[g][rows], sl, ql, self.ebs, self.dev, num_decodes=0)
                  for g in self.bt}
            mq = vc.mixed_step_meta(self.qbt_cpu[rows], sl, ql, vc.QBLOCK, self.dev, num_decodes=0)
            for l, layer in self.layers.items():
                parts = [history(l, int(r), c0, int(n)) for r, n in zip(rows.tolist(), sl.tolist())]
                K = torch.cat([p[0] for p in parts])
                V = torch.cat([p[1] for p in parts])
                if isinstance(layer, vc.KV800SlideLayer):
                    layer.write_step(K, V, me[self.group_of[l]])
                else:
                    layer.write_step(K, V, me[self.group_of[l]], mq, hosts=self.layers)
                del K, V, parts

    # ---- decode steps
    def freeze(self, steps):
        """Make the next `steps` decode steps replayable from one recorded step: the rows' lengths then advance on the
        device (an add inside the step instead of a copy from the host), and the host values of the step metadata are
        taken at the lengths after the last of those steps. Those values are bounds that hold for every step in
        between: the largest flushed sub-block count (the width of the decode tables and the clamp of each row's own
        count, which the kernels read on the device) and the rows of the sliding layers' identity tables."""
        self.lens_dev = self.lens.to(self.dev)
        self.lens_bound = self.lens + steps

    def thaw(self):
        """Undo freeze(): the next step goes by `lens` again. A step recorded before keeps its own lengths and cannot follow."""
        self.lens_dev = self.lens_bound = None

    def begin_step(self):
        """Metadata of the next decode step (every row appends one token) and the start of its flushes."""
        self.lens += 1
        if self.lens_dev is None:
            host, dl = self.lens, vc.step_lens(self.lens, self.dev)
        else:
            self.lens_dev += 1
            host, dl = self.lens_bound, self.lens_dev
        me = {g: vc.step_meta(self.bt[g], host, self.ebs, self.dev, dl) for g in self.bt}
        mq = vc.step_meta(self.qbt, host, vc.QBLOCK, self.dev, dl)
        self.metas = (me, mq)
        full = [self.layers[l] for l in (2, 6, 10, 14, 18, 22)]
        vc.launch_flushes(full, {l.l: me[self.group_of[l.l]] for l in full}, mq)
        return mq.positions

    def begin_chunk(self, lens, qlens, tokens, most, bound):
        """Metadata of a step whose rows bring qlens (R,) int32 <= most new tokens each, to lengths lens (R,) int64, both on
        the device; tokens: room for them; bound (R,): the host's bound of lens. Returns the step's kv800_hip.ChunkMeta."""
        if int(bound.max()) > self.nmax:
            raise ValueError(f"the caches hold {self.nmax} positions per row, the step may reach {int(bound.max())}")
        me = {g: vc.chunk_step_meta(self.bt[g], lens, qlens, self.ebs, tokens, most, bound) for g in self.bt}
        mq = vc.chunk_step_meta(self.qbt, lens, qlens, vc.QBLOCK, tokens, most, bound)
        self.metas = (me, mq)
        return mq.chunk

    def attend(self, l, q, k_pre, k_post, v):
        me, mq = self.metas
        layer = self.layers[l]
        if isinstance(layer, vc.KV800SlideLayer):
            return layer.forward(q, k_post, v, me[self.group_of[l]])
        return layer.forward(q, k_pre, v, me[self.group_of[l]], mq, hosts=self.layers, cos_t=self.cos, sin_t=self.sin)


class PagedAttention8:
    """The model's 11 attention layers over paged 8-bit caches (kv8): the 6 full layers over their whole history (no sinks, no
    800h blocks), the 5 sliding layers over a window of 256. Keys are rotated on their way into the cache. One block table for the
    full layers, one for the sliding ones, whose rows own a ring of `ring` shuffled pages that holds a chunk of FILL tokens and the
    window before it. The same steps as PagedAttention800: begin_step / attend, begin_chunk / attend (rows with any number of
    new tokens up to FILL: prompts, drafts), freeze / thaw for recorded steps, fill for synthetic histories.

    A draft larger than its block's tokens raises the block's exponent, for its keys or its values, and stays in it when it is taken
    back: the block's tokens, earlier and later ones, are then held at that exponent, of which values below 2^-6 lose a bit for each
    power of two (those above are held as before). The chunk's own earlier queries see them so, too. So a loop with drafts can differ
    from one without by that rounding.

    lens0: the rows' history lengths; steps: decode steps to provide for; bs: tokens per page."""

    FILL = 2048

    def __init__(self, lens0, steps, device, bs=128, seed=0):
        self.dev = device
        self.lens = torch.tensor([int(x) for x in lens0], dtype=torch.int64)
        R = len(lens0)
        nmax = self.nmax = int(self.lens.max()) + steps + 1
        rng = torch.Generator().manual_seed(seed)
        lp = (nmax - 1) // bs + 1
        self.ring = min(lp, (self.FILL + kv800.WIN) // bs + 2)
        perm = lambda n: torch.randperm(R * n, generator=rng).view(R, n).to(torch.int32)
        self.bt = {FULL: perm(lp).to(device), SLIDE: perm(self.ring)[:, torch.arange(lp) % self.ring].contiguous().to(device)}
        self.tables = {FULL: kernel_tables(nmax, device), SLIDE: model_rope_tables(1e4, 64, nmax, device)}
        kind = {**{l: FULL for l in (*vc.QUANT_LAYERS, *vc.WINDOW_LAYERS)}, **{l: SLIDE for l in vc.SLIDE_LAYERS}}
        self.kind = dict(sorted(kind.items()))
        self.layers = {l: kv8.Cache8.empty(R * (lp if t == FULL else self.ring), 4, bs, 128, device) for l, t in self.kind.items()}
        self.one = torch.arange(R + 1, dtype=torch.int64, device=device)      # starts of rows with one token each
        self.step = None                                                      # (lens, qsl) of the present step
        self.lens_dev = None                                                  # set by freeze()

    def fill(self, history):
        """Write every row's history into the caches, up to FILL positions per row at a time. history(l, r, p0, p1) -> (K, V)
        (p1 - p0, 4, 128) bf16 on the device: pre-RoPE K for full layers, post-RoPE K for sliding layers."""
        for c0 in range(0, int(self.lens.max()) if len(self.lens) else 0, self.FILL):
            n = torch.clamp(self.lens, max=c0 + self.FILL)
            new = torch.clamp(n - c0, min=0)
            qsl = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).to(self.dev)
            n = n.to(self.dev)
            for l, t in self.kind.items():
                parts = [history(l, r, c0, c0 + c) for r, c in enumerate(new.tolist()) if c]
                K, V = (torch.cat([p[i] for p in parts]) for i in (0, 1))
                cos, sin = self.tables[FULL] if t == FULL else (None, None)
                kv8.append(self.layers[l], K, V, self.bt[t], n, qsl, cos, sin)

    def provide(self, steps):
        """Whether the caches hold `steps` more positions of every row; a ValueError if not."""
        if int(self.lens.max()) + int(steps) > self.nmax:
            raise ValueError(f"the caches hold {self.nmax} positions per row, the steps reach {int(self.lens.max()) + int(steps)}")

    def freeze(self, steps):
        """Make the next `steps` decode steps replayable from one recorded step: the lengths then advance on the device, where nothing
        looks at the caches' room, so that it is looked at here."""
        self.provide(steps)
        self.lens_dev = self.lens.to(self.dev)

    def thaw(self):
        """Undo freeze(): the next step goes by `lens` again."""
        self.lens_dev = None

    def begin_step(self):
        """Metadata of the next decode step (every row appends one token): the new tokens' positions (R,) int64."""
        if not (self.one.is_cuda and torch.cuda.is_current_stream_capturing()):   # recording a step takes no position
            self.provide(1)
        self.lens += 1
        if self.lens_dev is None:
            lens = vc.step_lens(self.lens, self.dev)
        else:
            self.lens_dev += 1
            lens = self.lens_dev
        self.step = (lens, self.one)
        return lens - 1

    def begin_chunk(self, lens, qlens, tokens, most, bound):
        """Metadata of a step whose rows bring qlens (R,) int32 <= most new tokens each, to lengths lens (R,) int64, both on
        the device; tokens: room for them; bound (R,): the host's bound of lens. Returns the step's kv800_hip.ChunkMeta."""
        if int(bound.max()) > self.nmax:
            raise ValueError(f"the caches hold {self.nmax} positions per row, the step may reach {int(bound.max())}")
        if most > self.FILL:
            raise ValueError(f"a row may bring {self.FILL} tokens a step, not {most}")
        m = kv800_hip.chunk_meta(self.bt[FULL], lens, qlens, self.layers[next(iter(self.layers))].bs, tokens)
        self.step = (lens, m.qsl)
        return m

    def attend(self, l, q, k_pre, k_post, v):
        lens, qsl = self.step
        t, cache = self.kind[l], self.layers[l]
        kv8.append(cache, k_pre, v, self.bt[t], lens, qsl, *self.tables[t])
        return kv8.attend(cache, q, self.bt[t], lens, qsl, window=kv800.WIN if t == SLIDE else 0)


class DecodeGraph:
    """Greedy decode with one HIP graph per step. Construction runs the first step eagerly on the graph's own stream
    (it builds the cached tables, library handles and the flush stream that the recorded step reuses; its tokens are
    `tokens` afterwards, its bf16 logits `first_logits`), then freezes the attention for `steps` further steps and records
    one step, whose input is the token buffer and whose greedy tokens are copied back into it. Each step() replays it:
    one graph launch instead of ~250 kernel launches from the host. `tokens` and `logits` (the last replay's bf16
    logits) are buffers that the next step overwrites. The attention must be a PagedAttention800 or a PagedAttention8."""

    def __init__(self, model, attention, tokens, steps):
        self.attn, self.left = attention, int(steps)
        if isinstance(attention, PagedAttention8):
            attention.provide(1 + self.left)
        self.stream = torch.cuda.Stream(device=tokens.device)
        self.stream.wait_stream(torch.cuda.current_stream(tokens.device))
        with torch.cuda.stream(self.stream):
            self.first_logits = model.step(tokens, attention.begin_step(), fp32=False)
            self.tokens = mo.argmax(self.first_logits)
        self.stream.synchronize()
        attention.freeze(self.left)
        lens = attention.lens.clone()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            logits = model.step(self.tokens, attention.begin_step(), fp32=False)
            self.tokens.copy_(mo.argmax(logits))
        attention.lens = lens          # recording ran no step
        self.lens_dev = attention.lens_dev   # which the recorded step moves on
        self.logits = logits
        torch.cuda.current_stream(tokens.device).wait_stream(self.stream)

    def step(self):
        """One decode step: returns the (R,) greedy tokens."""
        if self.left <= 0:
            raise RuntimeError("DecodeGraph: the steps it was recorded for are used up")
        if self.attn.lens_dev is not self.lens_dev:
            raise RuntimeError("DecodeGraph: the attention's lengths have moved on without it")
        self.left -= 1
        self.attn.lens += 1
        self.graph.replay()
        return self.tokens


def decode_loop(model, attention, tokens, steps, graph=False):
    """Greedy decode: `steps` steps from `tokens` (R,) int64; returns the (steps, R) generated tokens. graph=True runs
    the steps after the first as replays of one recorded step (DecodeGraph; the paged attentions only)."""
    if graph and steps > 0:
        dg = DecodeGraph(model, attention, tokens, steps - 1)
        out = [dg.tokens.clone()]
        for _ in range(steps - 1):
            out.append(dg.step().clone())
        return torch.stack(out)
    out = []
    for _ in range(steps):
        tokens = model.greedy(tokens, attention.begin_step())
        out.append(tokens)
    return torch.stack(out)


def speculative_loop(model, attention, tokens, steps, draft, most, temperature=None, generator=None):
    """Decode with drafted tokens: `steps` steps from `tokens` (R,) int64, each of which appends to every row its last token
    and up to `most` drafts, keeps the drafts that the model confirms (spec_ops.verify_drafts) and takes one more token
    behind them. draft(last (R,), lens (R,)) -> (drafts (R, most) int64, counts (R,) int32 of them in use, their
    distributions (R, most, vocab) fp32 or None), all on the device; lens counts the positions in the caches. Drafts behind a
    row's count may hold anything, one outside the vocabulary is never kept. temperature
    (R,) fp32, None: greedy. Lengths stay on the device, so a step does not wait for the one before; the attention must be a
    PagedAttention800 or PagedAttention8 with room for steps (most + 1) more positions, most < 128. Greedy tokens are those of the one-token loop
    up to near-ties: the short conv rounds once a sum and not every product, and a block that becomes eligible inside a chunk
    is read exact by that chunk; with PagedAttention8, drafts may also have left a block a larger exponent, and of 8-bit products a
    rounding before them may move a token's code by a whole step, so that there more is near. Returns the rows' new tokens, a list of R
    tensors, and the (steps, R) counts; attention.lens follows."""
    dev, R = tokens.device, tokens.shape[0]
    if not 0 <= most < 128:
        raise ValueError("most must be in [0, 128)")
    if steps > 0 and int(attention.lens.max()) + steps * (most + 1) > attention.nmax:
        raise ValueError(f"the caches hold {attention.nmax} positions per row, the steps may reach "
                         f"{int(attention.lens.max()) + steps * (most + 1)}")
    if temperature is None:
        temperature = torch.zeros(R, dtype=torch.float32, device=dev)
    lens = attention.lens.to(dev)
    T, last, got = R * (most + 1), tokens, []
    at = torch.arange(T, device=dev)
    for s in range(steps):
        drafts, counts, probs = draft(last, lens)
        ql = (counts.clamp(0, most) + 1).to(torch.int32)
        meta = attention.begin_chunk(lens + ql, ql, T, most + 1, attention.lens + (s + 1) * (most + 1))
        i = (at - meta.qsl[meta.row]).clamp(max=most)
        tok = torch.cat((last[:, None], drafts), 1)[meta.row, i]
        logits = model.chunk(tok.clamp(0, model.cfg.vocab - 1), meta)     # unused and foreign drafts: any token, never kept
        q = None if probs is None or not most else probs[meta.row, i.clamp(max=most - 1)]
        out, kept = so.verify_drafts(logits, tok, meta.qsl, temperature, torch.rand(T, device=dev, generator=generator),
                                     torch.rand(R, device=dev, generator=generator), q)
        model.commit(kept)
        lens = lens + kept
        last = out[meta.qsl[:-1] + kept - 1]
        got.append((out, kept, meta.row))
    if steps > 0:
        attention.lens = lens.cpu()
        attention.thaw()
    rows = [torch.cat([out[(row == r) & (out >= 0)] for out, _, row in got]) if got else tokens[:0] for r in range(R)]
    return rows, torch.stack([kept for _, kept, _ in got]) if got else torch.zeros(0, R, dtype=torch.int32, device=dev)
