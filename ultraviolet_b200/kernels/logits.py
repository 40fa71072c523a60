"""What stands between the head and the sampler: softcap, penalties for repeated tokens, biases and a mask of allowed tokens."""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor

from .. import _lib


@torch.library.custom_op("uvb200::adjust_logits", mutates_args=())
def _adjust_op(x: Tensor, softcap: Optional[Sequence[float]], history: Optional[Tensor], lengths: Optional[Tensor],
               prompt_lengths: Optional[Tensor], parents: Optional[Tensor], tokens: Optional[Tensor], repetition: Optional[Tensor],
               frequency: Optional[Tensor], presence: Optional[Tensor], bias_ids: Optional[Tensor], bias: Optional[Tensor],
               allowed: Optional[Tensor]) -> Tensor:
    return _lib.host().adjust_logits(x, None if softcap is None else tuple(softcap), history, lengths, prompt_lengths, parents, tokens,
                                     repetition, frequency, presence, bias_ids, bias, allowed, None, True)


@_adjust_op.register_fake
def _(x, softcap, history, lengths, prompt_lengths, parents, tokens, repetition, frequency, presence, bias_ids, bias, allowed):
    return x.new_empty(x.shape, dtype=torch.float32)


def adjust_logits(x: Tensor, *, softcap=None, history: Tensor | None = None, lengths: Tensor | None = None,
                  prompt_lengths: Tensor | None = None, parents: Tensor | None = None, tokens: Tensor | None = None,
                  repetition=None, frequency=None, presence=None, bias_ids: Tensor | None = None, bias: Tensor | None = None,
                  allowed: Tensor | None = None, out: Tensor | None = None) -> Tensor:
    """Logits for the sampler from the head's output x (B, V) or, one row per node of a tree, (B, T, V); fp32 unless ``out`` says
    otherwise (any of fp32 / fp16 / bf16; ``out=x`` works in place).  In this order, each step where it is asked for:

    * softcap (a, b, c): z = a * sigmoid((x + b) / c)
    * repetition (a number or (B,) fp32): of every token in the row's text, z / repetition where z > 0, else z * repetition
    * frequency, presence: z -= frequency * n + presence * (n > 0), n = how often the token was drawn
    * bias_ids, bias (B, n) or (n,): added to those tokens; of several entries for one token the last counts
    * allowed (B, words) or (B, T, words) int32: tokens v whose bit v % 32 of word v // 32 is 0 become -inf, whatever they were

    The text of row b is history[b, :lengths[b]] (int32 or int64; default: all of it), its first prompt_lengths[b] tokens the prompt
    and the others drawn.  With a tree (parents, tokens (B, T)) the tokens of a node's ancestors and its own count as drawn in
    its row.  Tokens and ids outside the vocabulary are ignored.  A row whose mask allows nothing is -inf throughout."""
    per_row = [v if v is None or isinstance(v, Tensor) else torch.full((x.size(0),), float(v), dtype=torch.float32, device=x.device)
               for v in (repetition, frequency, presence)]
    cap = None if softcap is None else tuple(float(v) for v in softcap)
    if not torch.compiler.is_compiling():
        got = _lib.host().adjust_logits(x, cap, history, lengths, prompt_lengths, parents, tokens, *per_row, bias_ids, bias, allowed, out,
                                        False)
        if got is not None:
            return got
    if out is not None and (out.shape != x.shape or out.dtype not in (torch.float32, torch.float16, torch.bfloat16)):
        raise ValueError(f"out has to be float32, float16 or bfloat16 and like x; got {tuple(out.shape)} {out.dtype}")
    got = _adjust_op(x, cap, history, lengths, prompt_lengths, parents, tokens, *per_row, bias_ids, bias, allowed)
    return got if out is None else out.copy_(got)
