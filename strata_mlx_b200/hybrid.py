"""A small synthetic decoder on the context operators (context.py): a batch of sequences through a trunk of linear and
of full attention layers around the MoE blocks. What a sequence keeps is bounded at any length: a state a linear layer,
and a cache of `capacity` slots a full attention layer, cut to the `keep` tokens that gathered the most attention weight
whenever it is full.

    python -m strata_mlx_b200.hybrid [--batch 8] [--prompt 512] [--steps 64]

    prompt   linear layers by linear_attention (ragged prompts by their lengths); full layers write their keys and
             values into the cache and take the prompt's tokens, ROWS at a time, as rows of decode_attention over one
             row of the table
    step     one token a sequence: linear_attention_step, KVPages.attend with weights, the MoE block's decode kernels
    evict    every full layer's KVPages.evict, then one new length for all of them

Weights are seeded random ones (no model file exists here): projections bfloat16 through cuBLAS, experts as GGUF
blocks. Layer l is full attention where l % every == every - 1.
"""

from __future__ import annotations

import torch

from . import blocks as B
from . import fused as F
from ._lib import check_device_errors
from .context import KVPages, linear_attention, linear_attention_step
from .decoder import HEAD_DIM, PAGE, Dense, Rope, rmsnorm
from .synthetic import blocks_cuda

ROWS = 4096  # a prompt's tokens that one attention call takes: its scores are as many rows of the cache's slots


class LinearMixer:
    """Linear attention with a decay a head and token: g = -rate softplus(x W), keys of unit length."""

    def __init__(self, hidden: int, heads: int, dim: int, gen, device):
        self.heads, self.dim = heads, dim
        self.wqkv = Dense(3 * heads * dim, hidden, "bf16", gen, device)
        self.wg = Dense(heads, hidden, "bf16", gen, device)
        self.wo = Dense(hidden, heads * dim, "bf16", gen, device)
        self.rate = torch.logspace(-3, -0.5, heads, device=device)
        self.state = None

    def _inputs(self, h: torch.Tensor) -> tuple:
        q, k, v = self.wqkv(h).unflatten(-1, (3, self.heads, self.dim)).unbind(-3)
        k = torch.nn.functional.normalize(k.float(), dim=-1).to(h.dtype)
        return q, k, v, -self.rate * torch.nn.functional.softplus(self.wg(h).float())

    def prompt(self, h: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        out, self.state = linear_attention(*self._inputs(h), lengths=lengths)
        return self.wo(out.flatten(-2))

    def step(self, h: torch.Tensor) -> torch.Tensor:
        return self.wo(linear_attention_step(*self._inputs(h), self.state).flatten(-2))


class CacheMixer:
    """Grouped-query attention over a batch's paged cache (KVPages), whose slots gather their attention weight. The
    decoder's table, lengths and positions are shared by all of its layers; keys, values and weights are the layer's."""

    def __init__(self, hidden: int, q_heads: int, kv_heads: int, own, gen, device):
        self.hq, self.hkv, self.own = q_heads, kv_heads, own
        self.wqkv = Dense((q_heads + 2 * kv_heads) * HEAD_DIM, hidden, "bf16", gen, device)
        self.wo = Dense(hidden, q_heads * HEAD_DIM, "bf16", gen, device)
        pages = own.table.numel() + 1  # the last takes what lies past a prompt's length
        self.k, self.v = (torch.zeros((pages, PAGE, kv_heads, HEAD_DIM), dtype=torch.bfloat16, device=device)
                          for _ in range(2))
        self.weight = torch.zeros((own.batch, own.capacity), device=device)
        self.position = torch.zeros((own.batch, own.capacity), dtype=torch.int32, device=device)
        self.cache = KVPages(self.k, self.v, own.table, own.lengths, weight=self.weight, position=self.position)

    def _qkv(self, h: torch.Tensor, at: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """The queries of tokens (n, hidden) at positions `at`, their keys and values written at the pools' `rows`."""
        q, k, v = self.wqkv(h).unflatten(-1, (-1, HEAD_DIM)).split([self.hq, self.hkv, self.hkv], dim=-2)
        self.k.view(-1, self.hkv, HEAD_DIM)[rows] = self.own.rope(k, at)
        self.v.view(-1, self.hkv, HEAD_DIM)[rows] = v
        return self.own.rope(q, at)

    def prompt(self, h: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        n, t = h.shape[:2]
        at = torch.arange(t, device=h.device)
        live = at < lengths[:, None]
        rows = torch.where(live, self.own.rows(at.expand(n, t)), (self.k.shape[0] - 1) * PAGE)
        q = self._qkv(h.flatten(0, 1), at.repeat(n), rows.flatten())
        self.position[:, :t] = at
        # token i sees slots 0 .. i of its sequence's row; tokens past a length see none
        seen = torch.where(live, at + 1, 0).to(torch.int32)
        q = q.unflatten(0, (n, t))
        out = torch.empty_like(q)
        self.weight.zero_()
        each = max(1, ROWS // n)
        for i in range(0, t, each):
            m = min(each, t - i)
            weight = torch.zeros((n * m, self.own.capacity), device=h.device)
            table = self.own.table.repeat_interleave(m, 0)
            part = KVPages(self.k, self.v, table, seen[:, i : i + m].flatten(), weight=weight).attend(
                q[:, i : i + m].flatten(0, 1))
            out[:, i : i + m] = part.unflatten(0, (n, m))
            self.weight += weight.unflatten(0, (n, m)).sum(1)
        return self.wo(out.flatten(0, 1).flatten(-2)).unflatten(0, (n, t))

    def step(self, h: torch.Tensor) -> torch.Tensor:
        own = self.own
        slot = own.lengths.long() - 1  # this token's, counted already
        q = self._qkv(h, own.seen.long(), own.rows(slot[:, None])[:, 0])
        each = torch.arange(own.batch, device=h.device)
        self.weight[each, slot] = 0.0
        self.position[each, slot] = own.seen
        return self.wo(self.cache.attend(q).flatten(-2))

    def evict(self, lengths: torch.Tensor) -> None:
        own = self.own
        self.cache.evict(own.seen, own.keep, sinks=own.sinks, recent=own.recent,
                         out=(self.weight, self.position, lengths))


class HybridDecoder:
    """The decoder: prompt(tokens, lengths) once, then step(tokens) for each further token; both return float32 logits
    (batch, vocab). The batch is at most 8 sequences where the MoE blocks' decode kernels run (experts > 0)."""

    def __init__(self, layers: int = 4, batch: int = 4, capacity: int = 512, keep: int = 384, sinks: int = 4,
                 recent: int = 128, hidden: int = 2048, every: int = 2, linear_heads: int = 16, linear_dim: int = 128,
                 q_heads: int = 16, kv_heads: int = 2, experts: int = 64, top_k: int = 8, inter: int = 512,
                 kind: str = "Q2_0", vocab: int = 1024, max_pos: int = 8192, device=None, seed: int = 0):
        if capacity % PAGE or not sinks + recent <= keep < capacity:
            raise ValueError("capacity in whole pages, keep below it, sinks and recent within keep")
        self.device = device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.batch, self.capacity, self.keep, self.sinks, self.recent = batch, capacity, keep, sinks, recent
        g = torch.Generator(device=device).manual_seed(seed)
        per = capacity // PAGE
        self.table = torch.randperm(batch * per, generator=g, device=device).to(torch.int32).reshape(batch, per)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)  # slots in use
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)     # positions so far
        self.most = 0  # no sequence holds more slots
        self.reached, self.max_pos = 0, max_pos  # no sequence has had more positions; those that rope has angles for
        self.rope = Rope(max_pos, device)
        self.embed = torch.randn((vocab, hidden), generator=g, device=device).to(torch.bfloat16)
        self.head = torch.randn((vocab, hidden), generator=g, device=device) * hidden ** -0.5
        self.norm = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        self.layers = []
        for l in range(layers):
            mixer = (CacheMixer(hidden, q_heads, kv_heads, self, g, device) if l % every == every - 1
                     else LinearMixer(hidden, linear_heads, linear_dim, g, device))
            self.layers.append((mixer, self._moe(l, experts, top_k, inter, hidden, kind, seed) if experts else None))

    def _moe(self, l: int, experts: int, top_k: int, inter: int, hidden: int, kind: str, seed: int) -> tuple:
        """The MoE block as its prompt form and its decode form, on the same weights."""
        def stack(mats, rows, cols, sd):
            raw = blocks_cuda(kind, mats, rows, cols, 1000 * seed + 10 * l + sd, self.device, sigma=0.025)
            return B.BlockSwitchLinear(raw, kind, (mats, rows, cols))

        gate, up, down = stack(experts, inter, hidden, 1), stack(experts, inter, hidden, 2), stack(experts, hidden, inter, 3)
        shared = stack(1, inter, hidden, 4), stack(1, inter, hidden, 5), stack(1, hidden, inter, 6)
        g = torch.Generator(device=self.device).manual_seed(1000 * seed + 10 * l + 7)
        router = (torch.randn((experts, hidden), generator=g, device=self.device) * 0.02).half()
        shared_gate = (torch.randn((hidden,), generator=g, device=self.device) * 0.02).half()
        return (F.RoutedMoE(router, B.BlockSwitchGLU(gate, up, down), F.SharedExpert(*shared), shared_gate, top_k),
                F.MoEDecodeLayer(router, gate, up, down, top_k, shared=shared, shared_gate=shared_gate))

    def rows(self, slots: torch.Tensor) -> torch.Tensor:
        """The pools' rows of each sequence's `slots` (batch, n)."""
        page = (slots // PAGE).clamp(max=self.table.shape[1] - 1)
        return self.table.long().gather(1, page) * PAGE + slots % PAGE

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return rmsnorm(x, self.norm).float() @ self.head.T

    def prompt(self, tokens: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        """Prompts (batch, t), sequence b's the first lengths[b] >= 1 tokens: the logits behind each one's last token. Lengths
        stay on the device; one past t counts as t, one below 0 as 0."""
        n, t = tokens.shape
        if n != self.batch or t > self.capacity:
            raise ValueError(f"prompts ({self.batch}, at most {self.capacity}) expected, got {tuple(tokens.shape)}")
        if t > self.max_pos:
            raise ValueError(f"prompts of {t} tokens, but max_pos is {self.max_pos}")
        lengths = lengths.clamp(0, t)
        x = self.embed[tokens]
        for mixer, moe in self.layers:
            x = x + mixer.prompt(rmsnorm(x, self.norm), lengths)
            if moe is not None:
                x = x + moe[0](rmsnorm(x, self.norm).flatten(0, 1)).unflatten(0, (n, t))
        self.lengths.copy_(lengths)
        self.seen.copy_(lengths)
        self.most = self.reached = t
        return self._logits(x[torch.arange(n, device=x.device), (lengths.long() - 1).clamp(min=0)])

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One more token a sequence (batch,), up to max_pos positions, the prompt's width among them. A full cache is cut
        to its budget first."""
        if self.reached == self.max_pos:
            raise ValueError(f"all {self.max_pos} positions (max_pos) are taken")
        self.reached += 1
        if self.most == self.capacity:
            self.evict()
        self.most += 1
        self.lengths += 1
        x = self.embed[tokens]
        for mixer, moe in self.layers:
            x = x + mixer.step(rmsnorm(x, self.norm))
            if moe is not None:
                x = x + moe[1](rmsnorm(x, self.norm))
        self.seen += 1
        return self._logits(x)

    def evict(self) -> None:
        """Every full attention layer keeps its own `keep` tokens; the lengths, one for all layers, change last."""
        left = torch.empty_like(self.lengths)
        for mixer, _ in self.layers:
            if isinstance(mixer, CacheMixer):
                mixer.evict(left)
        torch.minimum(self.lengths, torch.full_like(self.lengths, self.keep), out=self.lengths)
        self.most = min(self.most, self.keep)


def main() -> None:
    import argparse
    import time

    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args()
    capacity = -(-(a.prompt + a.steps // 2) // PAGE) * PAGE
    dec = HybridDecoder(a.layers, a.batch, capacity=capacity, keep=capacity * 3 // 4, recent=capacity // 4,
                        max_pos=a.prompt + a.steps)
    g = torch.Generator(device=dec.device).manual_seed(1)
    tokens = torch.randint(0, dec.embed.shape[0], (a.batch, a.prompt), generator=g, device=dec.device)
    lengths = torch.randint(1, a.prompt + 1, (a.batch,), generator=g, device=dec.device, dtype=torch.int32)
    nxt = dec.prompt(tokens, lengths).argmax(-1)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        nxt = dec.step(nxt).argmax(-1)
    torch.cuda.synchronize()
    s = time.perf_counter() - t
    check_device_errors(dec.device)
    print(f"{a.batch} sequences, {a.layers} layers: {a.batch * a.steps / s:.0f} tokens/s, caches of {capacity} slots hold "
          f"{dec.lengths.tolist()} of {dec.seen.tolist()} tokens")


if __name__ == "__main__":
    main()
