"""Shared attention-block path: fused QKV projection -> fused per-head q/k
RMSNorm + RoPE + K/V write -> flash attention (prefill) or split-KV decode
attention -> output projection.  All on the sm_100a kernels.

Replaces, per forward, the reference's 3 nn.Linear + 2 nn.RMSNorm + 2
rope_apply launches + KVCache slice copies + 2 repeat_interleave copies +
transposes + flash_attn_func (torchpp/attention/gqa.py:80-131)."""
from __future__ import annotations

import torch

from .. import ops


def _version(t: torch.Tensor) -> int:
    try:
        return t._version
    except RuntimeError:  # inference tensors carry no version counter
        return -1


class FusedQKV:
    """Caches cat(Wq, Wk, Wv) so one GEMM produces q, k and v; rebuilt when any
    weight changes (tracked through the tensors' version counters)."""

    def __init__(self):
        self._key = None
        self._w = None

    def get(self, *ws: torch.Tensor) -> torch.Tensor:
        key = tuple((w.data_ptr(), _version(w), w.shape) for w in ws)
        if key != self._key:
            self._w = torch.cat([w.detach() for w in ws], dim=0).contiguous()
            self._key = key
        return self._w


def rotary_tables(cos: torch.Tensor | None, sin: torch.Tensor | None, D: int, like: torch.Tensor
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, or identity tables where there is no rotary embedding."""
    if cos is None:
        cos = torch.ones((1, D), dtype=like.dtype, device=like.device).expand(1 << 20, D)
        sin = torch.zeros((1, D), dtype=like.dtype, device=like.device).expand(1 << 20, D)
    return cos, sin


def attention_block(x: torch.Tensor, wqkv: torch.Tensor, wo: torch.Tensor,
                    bo: torch.Tensor | None, Hq: int, Hkv: int, D: int,
                    qn_w: torch.Tensor | None, kn_w: torch.Tensor | None, eps: float,
                    cos: torch.Tensor | None, sin: torch.Tensor | None, kv_cache=None,
                    cache_pos: int | None = None, causal: bool = True,
                    window_left: int = -1, residual: torch.Tensor | None = None) -> torch.Tensor:
    B, S, _ = x.shape
    qkv = ops.linear(x, wqkv)                                  # [B, S, (Hq+2Hkv) D]
    cos, sin = rotary_tables(cos, sin, D, x)
    if kv_cache is not None:
        start = int(cache_pos) if cache_pos is not None else kv_cache.cache_len
        kv_cache._ensure_allocated(B)
        if start + S > kv_cache.max_seq_len:
            raise ValueError("KV cache overflow")
        kc, vc = kv_cache.k_cache[:B], kv_cache.v_cache[:B]
        positions = torch.full((B,), start, dtype=torch.int32, device=x.device)
        q = ops.qk_norm_rope_cache(qkv, qn_w, kn_w, eps, cos, sin, positions, kc, vc, Hq, Hkv)
        kv_cache.cache_len = max(kv_cache.cache_len, start + S)
        L = start + S
        if S == 1:
            o = ops.attention_decode(q[:, 0], kc, vc, None, L, window_left=window_left)
        else:
            o = ops.attention(q, kc[:, :, :L].transpose(1, 2), vc[:, :, :L].transpose(1, 2),
                              causal=causal, window_left=window_left)
    else:
        kbuf = torch.empty((B, Hkv, S, D), dtype=x.dtype, device=x.device)
        vbuf = torch.empty_like(kbuf)
        positions = torch.zeros((B,), dtype=torch.int32, device=x.device)
        q = ops.qk_norm_rope_cache(qkv, qn_w, kn_w, eps, cos, sin, positions, kbuf, vbuf, Hq, Hkv)
        o = ops.attention(q, kbuf.transpose(1, 2), vbuf.transpose(1, 2), causal=causal,
                          window_left=window_left)
    return ops.linear(o.reshape(B, S, Hq * D), wo, bo, residual=residual)


def longest_prompt(cu_seqlens: torch.Tensor, rows: int, room: int) -> int:
    """A length that no prompt of a packed batch of `rows` rows exceeds: all its rows where so
    many fit `room` anyway, else the longest prompt's, read from the device."""
    if rows <= room or cu_seqlens.shape[0] < 2:
        return min(rows, room)
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("a recorded call has to be given max_seqlen")
    return int((cu_seqlens[1:] - cu_seqlens[:-1]).max())


def packed_attention_block(x: torch.Tensor, wqkv: torch.Tensor, wo: torch.Tensor,
                           bo: torch.Tensor | None, Hq: int, Hkv: int, D: int,
                           qn_w: torch.Tensor | None, kn_w: torch.Tensor | None, eps: float,
                           cos: torch.Tensor | None, sin: torch.Tensor | None,
                           cu_seqlens: torch.Tensor,
                           kv_cache=None, window_left: int = -1,
                           residual: torch.Tensor | None = None,
                           max_seqlen: int | None = None) -> torch.Tensor:
    """attention_block over prompts of different lengths packed row after row: x [N, E],
    sequence b in rows cu_seqlens[b] .. cu_seqlens[b+1]-1 (int32 on the device), causal,
    whole prompts.  A KVCache of batch B receives each sequence's K and V from row 0 on;
    its cache_len is left to the caller (the lengths differ).  max_seqlen: the longest prompt's
    length, if the caller has it; it is otherwise read from the device where N rows are more
    than the rotary tables or the cache hold."""
    cos, sin = rotary_tables(cos, sin, D, x)
    room = cos.shape[0] if kv_cache is None else min(cos.shape[0], kv_cache.max_seq_len)
    if max_seqlen is None:
        max_seqlen = longest_prompt(cu_seqlens, x.shape[0], room)
    if max_seqlen > cos.shape[0]:
        raise ValueError("a prompt exceeds the rotary tables")
    if max_seqlen > room:
        raise ValueError("KV cache overflow")
    qkv = ops.linear(x, wqkv)                                  # [N, (Hq+2Hkv) D]
    kc = vc = None
    if kv_cache is not None:
        B = cu_seqlens.shape[0] - 1
        kv_cache._ensure_allocated(B)
        kc, vc = kv_cache.k_cache[:B], kv_cache.v_cache[:B]
    q, k = ops.qk_norm_rope_packed(qkv, qn_w, kn_w, eps, cos, sin, cu_seqlens, Hq, Hkv,
                                   k_cache=kc, v_cache=vc)
    v = qkv[:, (Hq + Hkv) * D:].view(-1, Hkv, D)               # as the projection leaves it
    o = ops.attention_packed(q, k, v, cu_seqlens, window_left=window_left)
    return ops.linear(o.view(-1, Hq * D), wo, bo, residual=residual)


def norm_eps(m) -> float:
    e = getattr(m, "eps", None)
    return 1e-6 if e is None else float(e)
