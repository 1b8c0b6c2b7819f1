"""Losses over a vocabulary (CDNA4 kernels, csrc/token_loss.hip).

``token_logprobs`` gives the log probabilities of given tokens, the entropy of
each row and its most likely alternatives; minus its ``logprob`` is the
masked-token loss of BERT pretraining (reference dear/bert_benchmark.py:
101-112), and its alternatives are what a distillation teacher writes down.
``topk_distill_loss`` is the loss of a student that learns from such
alternatives. Both are differentiable once in the logits.

Logits are float32, bfloat16 or float16, of any strides, with the vocabulary
last; results are float32. A row whose logits hold NaN or +inf, or nothing but
-inf, gives NaN; single logits of -inf are tokens of probability zero. A token
id outside of the vocabulary gives NaN as well, and nothing is read there.

On the CPU the same numbers come from a torch composition; on a GPU the native
extension is required, and forward-mode derivatives and tracing
(torch.jit.trace, make_fx) raise.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from .fused import _native

__all__ = ["MAX_TOP", "TokenLogProbs", "token_logprobs", "topk_distill_loss"]

MAX_TOP = 128

_TYPES = (torch.float32, torch.bfloat16, torch.float16, torch.float64)


class TokenLogProbs(NamedTuple):
    logprob: Optional[torch.Tensor]       # [...], None without tokens
    entropy: torch.Tensor                 # [...]
    top_logprobs: Optional[torch.Tensor]  # [..., top], None for top = 0
    top_ids: Optional[torch.Tensor]       # [..., top] int64, best first


def _check_temperature(name, temperature):
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"{name}: temperature must be 1e-4 to 1e4, "
                         f"got {temperature}")


def _check_logits(name, logits):
    if logits.dtype not in _TYPES:
        raise TypeError(f"{name}: logits must be a float tensor, got "
                        f"{logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.size(-1) < 1 << 30:
        raise ValueError(f"{name}: logits need a last axis of 1 to 2^30 - 1 "
                         "tokens")


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor],
                   *, top: int = 0, temperature: float = 1.0,
                   ignore_index: int = -1) -> TokenLogProbs:
    """Log probabilities under softmax(logits / temperature).

    logits [..., V]; tokens int64 [...] or None, where only entropy and
    alternatives are wanted. Rows whose token is ``ignore_index`` are not
    looked at: log probability and entropy 0, ids -1 with log probability
    -inf, gradient 0. ``top`` (0 to MAX_TOP) alternatives are given best
    first; of equal logits the lower id comes first.
    """
    _check_temperature("token_logprobs", temperature)
    if logits.is_cuda:
        out = _native().token_logprobs(logits, tokens, top, temperature,
                                       ignore_index)
    else:
        out = _logprobs_torch(logits, tokens, top, temperature, ignore_index)
    i = 0 if tokens is None else 1
    return TokenLogProbs(out[0] if i else None, out[i],
                         out[i + 1] if top else None,
                         out[i + 2] if top else None)


def _log_softmax(x):
    """log_softmax in float64, with the digits of a probability near one: the
    largest elements' exp is 1, and log1p takes the sum of the others."""
    lp = torch.log_softmax(x, dim=-1)
    with torch.no_grad():
        d = x - x.amax(-1, keepdim=True)
        best = d == 0
        others = torch.where(best, 0.0, d.exp()).sum(-1, keepdim=True) \
            + (best.sum(-1, keepdim=True) - 1)
        more = torch.where(best, -others.log1p() - lp, 0.0)
    return lp + more


def _logprobs_torch(logits, tokens, top, temperature, ignore_index):
    _check_logits("token_logprobs", logits)
    V = logits.size(-1)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"token_logprobs: top must be 0 to {MAX_TOP} and at "
                         "most the vocabulary")
    x = logits.double()
    keep = None
    if tokens is not None:
        if tokens.dtype != torch.int64 or tokens.device != logits.device \
                or tokens.shape != logits.shape[:-1]:
            raise ValueError("token_logprobs: tokens are int64, on the "
                             "logits' device, one for each row")
        keep = tokens != ignore_index
        x = torch.where(keep[..., None], x, 0.0)
    lp = _log_softmax(x / temperature)
    p = lp.exp()
    h = -(p * lp.masked_fill(lp == -math.inf, 0.0)).sum(-1)
    out = []
    if tokens is not None:
        known = (tokens >= 0) & (tokens < V)
        at = tokens.clamp(0, V - 1)
        picked = lp.gather(-1, at[..., None])[..., 0]
        picked = picked * torch.where(known, 1.0, math.nan).to(picked.dtype)
        out.append(torch.where(keep, picked, 0.0))
        h = torch.where(keep, h, 0.0)
    out.append(h)
    if top:
        ids = x.sort(dim=-1, descending=True, stable=True)[1][..., :top]
        best = lp.gather(-1, ids)
        if keep is not None:
            best = torch.where(keep[..., None], best, -math.inf)
            ids = torch.where(keep[..., None], ids, -1)
        out += [best, ids]
    wide = logits.dtype == torch.float64
    return [t if wide or t.dtype == torch.int64 else t.float() for t in out]


def topk_distill_loss(logits: torch.Tensor, top_ids: torch.Tensor,
                      top_logprobs: torch.Tensor, *, temperature: float = 1.0,
                      tail: bool = False) -> torch.Tensor:
    """Distillation loss of every row, from a teacher's top logits:

        temperature^2 * KL(teacher || softmax(logits / temperature))

    logits [..., V]; top_ids int64 [..., K] and top_logprobs [..., K] (float32
    or 16-bit), K of 1 to MAX_TOP. Entries with a negative id are absent; a row
    with no entry has loss 0 and gradient 0 and is not looked at. An id that is
    named twice counts with the sum of its shares.

    top_logprobs are the teacher's log probabilities at this temperature.
    tail=False: the teacher is their softmax over the named tokens, so that
    its logits divided by the temperature do as well. tail=True: what their
    exponentials leave up to one is the share of all other tokens together,
    and is compared with what the student gives to these together, however
    little that is; where it gives them nothing at all (all of their logits are
    -inf) that term is left out.

    The teacher is constant: its tensors must not ask for a gradient.
    """
    _check_temperature("topk_distill_loss", temperature)
    if top_logprobs.requires_grad:
        raise ValueError("topk_distill_loss: top_logprobs asks for a gradient "
                         "and would get none: detach the teacher's answers")
    if logits.is_cuda:
        return _native().topk_distill_loss(logits, top_ids, top_logprobs,
                                           temperature, tail)
    return _distill_torch(logits, top_ids, top_logprobs, temperature, tail)


def _distill_torch(logits, ids, teacher, temperature, tail):
    _check_logits("topk_distill_loss", logits)
    if teacher.dtype not in _TYPES:
        raise TypeError("topk_distill_loss: top_logprobs must be a float "
                        f"tensor, got {teacher.dtype}")
    if ids.dtype != torch.int64 or ids.shape != teacher.shape \
            or ids.shape[:-1] != logits.shape[:-1] \
            or ids.dim() != logits.dim() \
            or ids.device != logits.device or teacher.device != logits.device:
        raise ValueError("topk_distill_loss: top_ids (int64) and top_logprobs "
                         "have the logits' leading shape and device, and one "
                         "length")
    if not 1 <= ids.size(-1) <= MAX_TOP:
        raise ValueError(f"topk_distill_loss: 1 to {MAX_TOP} entries a row")
    V = logits.size(-1)
    x = logits.double()
    present = ids >= 0
    live = present.any(-1)
    x = torch.where(live[..., None], x, 0.0)
    t = teacher.double().masked_fill(~present, -math.inf)
    if tail:
        q = t.exp()
        rest = (1.0 - q.sum(-1)).clamp(min=0.0)
    else:
        m = t.amax(-1, keepdim=True)
        q = (t - m.masked_fill(m == -math.inf, 0.0)).exp()
        total = q.sum(-1, keepdim=True)
        q = q / total.masked_fill(total == 0.0, 1.0)
        rest = torch.zeros_like(q[..., 0])
    lp = _log_softmax(x / temperature)
    at = ids.clamp(0, V - 1)
    l_at = lp.gather(-1, at) * torch.where(ids < V, 1.0, math.nan).double()
    loss = torch.where(q == 0.0, torch.where(ids < V, 0.0, math.nan).double(),
                       q * (q.log() - l_at)).sum(-1)
    if tail:
        named = torch.zeros(lp.shape, dtype=torch.int32, device=lp.device)
        named = named.scatter_add_(-1, at, present.int()) > 0
        # log p_t from the distances to the outside's own largest logit: next
        # to that of a far mask, the sum's logarithm would have no digits
        with torch.no_grad():
            far = x.masked_fill(named, -math.inf).amax(-1, keepdim=True)
            some = far[..., 0] != -math.inf
        left = torch.where(some[..., None], x - far, 0.0) / temperature
        out = left.masked_fill(named & some[..., None], -math.inf) \
            .logsumexp(-1)
        best = x.argmax(-1, keepdim=True)
        out = out + ((far - x.gather(-1, best)) / temperature
                     + lp.gather(-1, best))[..., 0]
        out = torch.where(some, out, 0.0)
        loss = loss + torch.where(some & (rest != 0.0), rest * (
            rest.masked_fill(rest == 0.0, 1.0).log() - out), 0.0)
    # a student's row that is no distribution: NaN, whatever the teacher says
    peak = x.detach().amax(-1)
    loss = loss * torch.where(peak.abs() < math.inf, 1.0, math.nan).double()
    loss = torch.where(live, loss * temperature ** 2, 0.0)
    return loss if logits.dtype == torch.float64 else loss.float()
