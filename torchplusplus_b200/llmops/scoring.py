"""Prompts of different lengths in one pass, and their scores.

`pack` lays prompts row after row; Qwen3.forward_packed runs them without padding
(ops.qk_norm_rope_packed, ops.attention_packed), and `score` gives the log probability of every
token of every prompt under the model, for perplexities, evaluations by likelihood or a
reference policy's log probabilities.  The reference has neither (its generate takes one prompt
length, torchpp/llmops/llm.py:226-286)."""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch

from .. import ops

ROWS = 4096  # rows whose logits are written at a time where alternatives are asked for


class PromptScores(NamedTuple):
    """Of one prompt's tokens 1 .. n-1, each given those before it (empty for n <= 1)."""
    logprobs: torch.Tensor                  # float32 [n-1]
    entropy: torch.Tensor                   # float32 [n-1], nats, of the distribution there
    ranks: Optional[torch.Tensor] = None    # int64 [n-1], 1: the most likely token
    top_logprobs: Optional[torch.Tensor] = None  # float32 [n-1, top]
    top_tokens: Optional[torch.Tensor] = None    # int64 [n-1, top]


def pack(prompts: Sequence[torch.Tensor], device) -> tuple[torch.Tensor, torch.Tensor, List[int]]:
    """1-D prompts of token ids -> ids int64 [N] and cu_seqlens int32 [B+1] on the device,
    and the lengths."""
    if len(prompts) == 0:
        raise ValueError("no prompts")
    prompts = [torch.as_tensor(p) for p in prompts]
    if any(p.dim() != 1 or p.is_floating_point() for p in prompts):
        raise ValueError("prompts must be 1-D tensors of token ids")
    lens = [len(p) for p in prompts]
    if all(p.device.type == "cpu" for p in prompts):
        ids = torch.cat([p.long() for p in prompts]).to(device, non_blocking=True)
    else:
        ids = torch.cat([p.to(device, torch.int64) for p in prompts])
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(device)
    return ids, cu, lens


@torch.inference_mode()
def score(model, prompts: Sequence[torch.Tensor], temperature: float = 1.0,
          top: Optional[int] = None) -> List[PromptScores]:
    """Scores of a Qwen3-shaped model.  top None: log probabilities and entropies, straight
    from the LM head's operands (ops.linear_logprobs: the logits in 32 bits, never written).
    top >= 0: also ranks and `top` alternatives, from logits in the model's type
    (ops.token_logprobs), some rows at a time."""
    ids, cu, lens = pack(prompts, model.out_head.weight.device)
    if max(lens) > model.cos.shape[0]:
        raise ValueError("a prompt exceeds the model's rotary table")
    if len(ids) == 0:
        parts = None
    else:
        h = model.final_rmsnorm(model.forward_packed(ids, cu, max_seqlen=max(lens)))
        # the token that each row predicts; -1 behind the last (its score is dropped)
        nxt = torch.cat([ids[1:], ids.new_full((1,), -1)])
        w = model.out_head.weight
        if top is None:
            parts = ops.linear_logprobs(h, w, nxt, temperature=temperature)
        else:
            rows = [ops.token_logprobs(ops.linear(h[i:i + ROWS], w), nxt[i:i + ROWS],
                                       temperature=temperature, top=top)
                    for i in range(0, len(ids), ROWS)]
            parts = [torch.cat(p) for p in zip(*rows)]
    out, a = [], 0
    for n in lens:
        e = a + max(n - 1, 0)
        if parts is None:
            new = lambda *s, t=torch.float32: torch.empty(s, dtype=t, device=cu.device)
            out.append(PromptScores(new(0), new(0)) if top is None else PromptScores(
                new(0), new(0), new(0, t=torch.int64), new(0, top), new(0, top, t=torch.int64)))
        else:
            out.append(PromptScores(*(t[a:e] for t in parts)))
        a += n
    return out
