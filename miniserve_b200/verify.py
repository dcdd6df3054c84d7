"""Verification of drafted tokens: ``verify_drafts``.

A cheap draft (a small model, or a lookup in the text so far) proposes a few
tokens; the target model scores all of them in one step; ``verify_drafts``
keeps the longest prefix that the target agrees with and draws one token more,
so that what comes out is distributed as the target's own samples
(miniserve/sampler.py:23-68 without its filters; ``Sampler`` draws single
tokens with them).  Random numbers are inputs, as they are for ``Sampler``.
"""
from __future__ import annotations

from typing import Sequence, Tuple, Union

from . import _lib
from .sampler import Number, _param, _torch


def verify_drafts(logits, drafts, uniforms, *, draft_probs=None,
                  temperature: Union[Number, Sequence, "object"] = 1.0) -> Tuple["object", "object", "object", "object"]:
    """Check ``drafts`` [B, n] int64 against the target's ``logits`` [B, n + 1, V]
    (fp32, bf16 or fp16), position i holding the logits after i drafts.

    A row's drafts end at its first negative entry.  With p = softmax(logits[b,
    i] / temperature[b]) and q = ``draft_probs[b, i]`` ([B, n, V] fp32, the
    distribution that the draft was drawn from; None for drafts that come from
    none), draft i is accepted when ``uniforms[b, i] * q[draft] < p[draft]``; at
    the first one that is not, a token is drawn from max(p - q, 0) (without q:
    from p without the draft), and where all are accepted, one from p at the
    next position.  ``uniforms`` [B, n + 1] float64: the last one is the draw's,
    in index order.  Temperature 0 accepts the first largest logit only.  Tokens
    that a filter or a grammar forbids have logits -inf.

    Returns ``(tokens, probs, counts, status)``: [B, n + 1] int64 (the accepted
    drafts, the drawn token, then -1), [B, n + 1] fp32 (p of each, 0 behind the
    last), [B] int32 (how many tokens) and [B] int32 MS_ROW_* bits.  Rows flagged
    MS_ROW_BAD_TEMPERATURE, MS_ROW_BAD_DRAFT (a draft past the vocabulary) or
    MS_ROW_ALL_MASKED (nothing but -inf at the position drawn from) have tokens
    -1 and count 0; MS_ROW_NONFINITE marks rows that met a NaN (read as -inf) or
    +inf logit (such tokens share the probability), or an entry of draft_probs
    that is negative, NaN or infinite.
    """
    torch = _torch()
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise TypeError("verify_drafts needs a CUDA tensor of logits")
    if logits.dim() != 3:
        raise ValueError("logits must be [B, drafts + 1, V]")
    heat = _param(temperature, logits.shape[0], torch.float64, logits.device)
    entry = _lib.binding()
    try:
        return entry.verify_drafts(logits, drafts, uniforms, draft_probs, heat)
    except entry.CallError as e:
        _lib.check(e.args[0], "ms_verify_drafts")
        raise
