"""Speculative decoding with draft trees: several drafted tokens a sequence are
verified by one forward pass of the target model.

A step takes a tree of T nodes a sequence (node 0 is the token chosen last, the
others are drafted), runs the model over the B * T nodes, verifies the trees
against the target's logits and commits the accepted paths' K/V: one launch
each of tpp_qk_norm_rope_tree and tpp_attention_tree a layer, then one of
tpp_verify_tree and one of tpp_kv_commit for all layers, the whole of it one CUDA
graph.  What is emitted follows the target model alone, greedily or sampled,
whatever was drafted.

The drafts here come from the sequence's own history (the continuations of
earlier occurrences of its last tokens), so no second model is needed; `draft`
may be any function of the same form.  The reference accepts and rejects a draft
model's chain in Python, without a KV cache (torchpp/llmops/spec_decoding.py:62)."""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence

import torch

from .. import ops
from ..attention._core import norm_eps
from .kvcache import KVCache

# history -> (tokens, parents) of at most `nodes` - 1 drafted nodes; parents count
# from 0, the root; a drafted node i (from 1 on) has parents[i - 1] < i
Draft = Callable[[Sequence[int], int], "tuple[List[int], List[int]]"]


def tree_mask(parents: torch.Tensor, window_left: int = -1) -> tuple[torch.Tensor, torch.Tensor]:
    """parents int [T] or [B,T] (any value < 0 at a root, parents[i] < i) ->
    (mask int64 [.., T, ceil(T/64)] for ops.attention_tree: each node sees its
    ancestors and itself, depth int32 [.., T]).  With a sliding window
    (window_left >= 0, the one given to ops.attention_tree) a node sees of them
    those at most window_left above it.  Computed on the host."""
    par = parents.cpu().long()
    flat = par.reshape(-1, par.shape[-1])
    B, T = flat.shape
    see = torch.zeros(B, T, (T + 63) // 64 * 64, dtype=torch.bool)
    rows = torch.arange(B)
    for i in range(T):
        p = flat[:, i]
        if bool((p >= i).any()):
            raise ValueError("a parent must come before its children")
        see[:, i] = see[rows, p.clamp_min(0)] & (p >= 0)[:, None]
        see[:, i, i] = True
    depth = see.sum(-1) - 1
    if window_left >= 0:
        see[..., :T] &= depth[:, None, :] >= depth[..., None] - window_left
    words = see.view(B, T, -1, 64).long() << torch.arange(64)
    shape = par.shape
    return (words.sum(-1).view(*shape, -1).to(parents.device),
            depth.to(torch.int32).view(shape).to(parents.device))


def lookup_draft(history: Sequence[int], nodes: int, ngram: int = 3, branches: int = 3
                 ) -> tuple[List[int], List[int]]:
    """Drafts from the history itself: up to `branches` latest continuations of
    the longest suffix (at most `ngram` tokens) that occurred before, merged into
    one tree of at most nodes - 1 drafted tokens."""
    h = list(history)
    tokens: List[int] = []
    parents: List[int] = []
    child: dict = {}
    for n in range(min(ngram, len(h) - 1), 0, -1):
        tail, found = h[-n:], 0
        for at in range(len(h) - n - 1, -1, -1):
            if h[at:at + n] != tail:
                continue
            cur = 0
            for t in h[at + n:at + n + (nodes - 1)]:
                key = (cur, t)
                if key not in child:
                    if len(tokens) >= nodes - 1:
                        break
                    tokens.append(t)
                    parents.append(cur)
                    child[key] = len(tokens)
                cur = child[key]
            found += 1
            if found >= branches or len(tokens) >= nodes - 1:
                break
        if tokens:
            break
    return tokens, parents


class SpeculativeDecoder:
    """Decodes `batch_size` sequences of a Qwen3-shaped model with trees of
    `nodes` nodes (1..256).  `draft` proposes the trees (default: lookup_draft)."""

    def __init__(self, model, batch_size: int, max_seq_len: int, nodes: int = 8,
                 draft: Optional[Draft] = None):
        cfg = model.cfg
        if not 1 <= nodes <= 256:
            raise ValueError("nodes must be in [1, 256]")
        if model.cos.shape[0] < max_seq_len + nodes:
            raise ValueError("max_seq_len + nodes exceeds the model's rotary table")
        self.model, self.cfg = model, cfg
        self.batch_size, self.max_seq_len, self.nodes = batch_size, max_seq_len, nodes
        self.draft = draft or lookup_draft
        self.device = dev = model.out_head.weight.device
        B, T, L, dt = batch_size, nodes, cfg.n_layers, cfg.dtype
        Hq, Hkv, D = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        self.k = torch.zeros(L, B, Hkv, max_seq_len, D, dtype=dt, device=dev)
        self.v = torch.zeros_like(self.k)
        self.caches = []
        for l in range(L):  # the prompt's K/V go through the model's own cache path
            c = KVCache(max_seq_len, Hkv, D, dt, dev)
            c.k_cache, c.v_cache, c.batch_size = self.k[l], self.v[l], B
            self.caches.append(c)
        # the nodes' K (normed, rotated) and projections (V is a part of them)
        self.k_tree = torch.zeros(L, B, T, Hkv, D, dtype=dt, device=dev)
        self.qkv = torch.zeros(L, B, T, (Hq + 2 * Hkv) * D, dtype=dt, device=dev)
        self.v_tree = self.qkv[..., (Hq + Hkv) * D:].view(L, B, T, Hkv, D)
        i32 = dict(dtype=torch.int32, device=dev)
        self.ctx = torch.zeros(B, **i32)         # rows in the cache
        self.active = torch.ones(B, **i32)
        self.positions = torch.zeros(B, T, **i32)
        self.depth = torch.zeros(B, T, **i32)
        self.parents = torch.full((B, T), -1, **i32)
        self.tokens = torch.zeros(B, T, dtype=torch.int64, device=dev)
        self.mask = torch.zeros(B, T, (T + 63) // 64, dtype=torch.int64, device=dev)
        self.uniforms = torch.zeros(B, T, device=dev)
        self.temperature = 0.0
        self._graph: Optional[torch.cuda.CUDAGraph] = None
        self._graph_temperature: Optional[float] = None
        self._graph_weights: List[torch.Tensor] = []
        self.path = self.count = self.next = None
        self.steps = 0

    # ------------------------------------------------------------ one step
    def _step(self) -> None:
        """The device's part: tokens, parents, depth, mask (and uniforms) ->
        path, count, next; the caches and ctx advance."""
        m, cfg = self.model, self.cfg
        Hq, Hkv = cfg.n_heads, cfg.n_kv_heads
        B, T = self.batch_size, self.nodes
        torch.add(self.ctx[:, None], self.depth, out=self.positions)
        x = ops.embedding(self.tokens, m.tok_embed.weight)
        for l, blk in enumerate(m.transformer_blocs):
            a = blk.attn
            h = ops.rmsnorm(x, blk.rms_norm1.weight, blk.rms_norm1.eps)
            ops.linear(h, a._qkv.get(a.Wq.weight, a.Wk.weight, a.Wv.weight), out=self.qkv[l])
            q, _ = ops.qk_norm_rope_tree(
                self.qkv[l], None if a.q_norm is None else a.q_norm.weight,
                None if a.k_norm is None else a.k_norm.weight,
                1e-6 if a.q_norm is None else norm_eps(a.q_norm), m.cos, m.sin,
                self.positions, Hq, Hkv, k_out=self.k_tree[l])
            o = ops.attention_tree(q, self.k[l], self.v[l], self.k_tree[l], self.v_tree[l],
                                   self.ctx, self.max_seq_len, self.mask)
            x = ops.linear(o.view(B, T, -1), a.out_projection.weight, residual=x)
            h = ops.rmsnorm(x, blk.rms_norm2.weight, blk.rms_norm2.eps)
            x = blk.ffn(h, residual=x)
        logits = ops.linear(ops.rmsnorm(x, m.final_rmsnorm.weight, m.final_rmsnorm.eps),
                            m.out_head.weight)
        self.path, self.count, self.next = ops.verify_tree(
            logits, self.tokens, self.parents, self.uniforms, self.temperature)
        ops.kv_commit(self.k_tree, self.v_tree, self.path, self.count, self.ctx, self.k, self.v)
        self.ctx.add_(self.count * self.active)

    def _weights(self) -> List[torch.Tensor]:
        """Every tensor of the model that a step reads (concatenations that a
        changed weight has made stale are rebuilt)."""
        m = self.model
        ws = [m.tok_embed.weight, m.final_rmsnorm.weight, m.out_head.weight, m.cos, m.sin]
        for blk in m.transformer_blocs:
            a = blk.attn
            ws += [blk.rms_norm1.weight, a._qkv.get(a.Wq.weight, a.Wk.weight, a.Wv.weight),
                   a.out_projection.weight, blk.rms_norm2.weight, blk.ffn.gate_up_weight(),
                   blk.ffn.linear_layer2.weight]
            ws += [n.weight for n in (a.q_norm, a.k_norm) if n is not None]
        return ws

    def _record(self) -> None:
        """Records the step as a CUDA graph where there is none yet, the
        temperature differs or the model's weights have moved."""
        # A graph reads the addresses it was recorded with: it holds the storages
        # behind them, so none is freed or handed out again while it lives.
        ws = [w.detach() for w in self._weights()]
        if self._graph is not None and self._graph_temperature == self.temperature and \
                [w.data_ptr() for w in ws] == [w.data_ptr() for w in self._graph_weights]:
            return
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):
            ctx = self.ctx.clone()  # in the order of side, ahead of what changes it
            self._step()  # warm-up: library set-up does not belong into a graph
            self.ctx.copy_(ctx)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                self._step()
        torch.cuda.current_stream(self.device).wait_stream(side)
        self._graph, self._graph_temperature, self._graph_weights = g, self.temperature, ws

    def _replay(self) -> None:
        self._graph.replay()
        self.steps += 1

    def step(self) -> None:
        """One verified step of the trees in the static buffers, as a CUDA graph
        (recorded again when the temperature or the model's weights change)."""
        self._record()
        self._replay()

    def set_trees(self, trees: "list[tuple[List[int], List[int]]]", roots: Sequence[int]) -> None:
        """Puts each sequence's root token and drafted (tokens, parents) into the
        static buffers; unused nodes hold token -1, which is never accepted."""
        B, T = self.batch_size, self.nodes
        tok = torch.full((B, T), -1, dtype=torch.int64)
        par = torch.zeros((B, T), dtype=torch.int32)
        par[:, 0] = -1
        for b, (t, p) in enumerate(trees):
            n = min(len(t), T - 1)
            tok[b, 0] = roots[b]
            if n:
                tok[b, 1:1 + n] = torch.tensor(t[:n])
                par[b, 1:1 + n] = torch.tensor(p[:n], dtype=torch.int32)
        mask, depth = tree_mask(par)
        for dst, src in ((self.tokens, tok), (self.parents, par), (self.mask, mask),
                         (self.depth, depth)):
            dst.copy_(src.pin_memory(), non_blocking=True)

    # ------------------------------------------------------------ generate
    @torch.inference_mode()
    def generate(self, input_ids: torch.Tensor, max_new_token: int, temperature: float = 0.0,
                 seed: int = 0, eos_token_id: Optional[int] = None) -> List[List[int]]:
        """input_ids [B, S] -> each sequence's new tokens (max_new_token of them,
        fewer where eos_token_id ends one).  temperature 0 decodes greedily."""
        B, S = input_ids.shape
        if B != self.batch_size or S + max_new_token > self.max_seq_len:
            raise ValueError("prompt + max_new_token does not fit the decoder")
        if max_new_token < 0:
            raise ValueError("max_new_token must not be negative")
        if max_new_token == 0:
            return [[] for _ in range(B)]
        m = self.model
        self.temperature = float(temperature)
        gen = torch.Generator(device=self.device).manual_seed(seed)
        for c in self.caches:
            c.cache_len = 0
        x = ops.embedding(input_ids.to(self.device), m.tok_embed.weight)
        for blk, c in zip(m.transformer_blocs, self.caches):
            x = blk(x, m.cos, m.sin, c, 0)
        logits = ops.linear(ops.rmsnorm(x[:, -1], m.final_rmsnorm.weight, m.final_rmsnorm.eps),
                            m.out_head.weight)
        self.ctx.fill_(S)
        self.active.fill_(1)
        root = torch.zeros(B, 1, dtype=torch.int64, device=self.device)
        u = torch.rand(B, 1, generator=gen, device=self.device)
        first = ops.verify_tree(logits[:, None], root, torch.full_like(root, -1, dtype=torch.int32),
                                u, self.temperature)[2].tolist()
        history = [ids + [t] for ids, t in zip(input_ids.tolist(), first)]
        done = [max_new_token == 1 or h[-1] == eos_token_id for h in history]
        self.steps = 0
        while not all(done):
            self.set_trees([([], []) if d else self.draft(h, self.nodes)
                            for h, d in zip(history, done)], [h[-1] for h in history])
            self.active.copy_(torch.tensor([0 if d else 1 for d in done], dtype=torch.int32))
            if self.temperature > 0:
                self.uniforms.uniform_(generator=gen)
            if self.steps == 0:   # weights are looked over once a request
                self._record()
            self._replay()
            path, count, nxt, tok = (t.tolist() for t in (self.path, self.count, self.next,
                                                          self.tokens))
            for b, h in enumerate(history):
                if done[b]:
                    continue
                for t in [tok[b][i] for i in path[b][1:count[b]]] + [nxt[b]]:
                    h.append(t)
                    if t == eos_token_id or len(h) - S >= max_new_token:
                        done[b] = True
                        break
        return [h[S:] for h in history]
