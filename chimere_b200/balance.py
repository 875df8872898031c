"""The router's balance loss, its pairs per expert and its gradient, over the C ABI.

What a router is trained and watched with: it takes the logits and the expert ids the package's router leaves (MoeScratch.router_logits,
.topk_indices) or any others.  The reference only logs the experts' load (chimere-server/src/qwen35_model/moe_ffn.rs:120-131).

    p = softmax(logits), or sigmoid(logits) / their sum          n = tokens that the mask leaves
    loss = coef * E / (top_k * n) * sum_e counts[e] * prob[e]    prob[e] = mean of p over them; an even load gives coef, n = 0 gives 0
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import abi
from .w8a8 import _TYPES, _call, _need


class BalanceLoss(NamedTuple):
    """Of each sequence (without the leading dimension for logits [T, E])."""
    loss: torch.Tensor     # f32 [S]
    counts: torch.Tensor   # int32 [S, E]: pairs per expert
    prob: torch.Tensor     # f32 [S, E]: mean probability
    tokens: torch.Tensor   # int32 [S]: tokens that the mask leaves


class _Args(NamedTuple):
    S: int
    L: int
    E: int
    k: int
    mode: int
    coef: float


def _check(logits, topk_idx, mask, route_mode, coef) -> _Args:
    _need(logits.is_cuda and logits.dim() in (2, 3) and logits.dtype in _TYPES, "logits: [T, E] or [S, L, E] of float32, float16 or bfloat16 on a CUDA device")
    _need(logits.stride(-1) == 1 or logits.shape[-1] == 1, "logits: the values of a row lie side by side")
    lead, E = logits.shape[:-1], logits.shape[-1]
    S, L = (1, lead[0]) if len(lead) == 1 else lead
    _need(topk_idx.dtype == torch.int32 and topk_idx.device == logits.device and topk_idx.shape[:-1] == lead and topk_idx.dim() == logits.dim() and topk_idx.is_contiguous(),
          "topk_idx: contiguous int32, one row of ids per row of logits")
    if mask is not None:
        _need(mask.dtype in (torch.bool, torch.uint8) and mask.device == logits.device and mask.shape == lead and mask.is_contiguous(),
              "mask: contiguous bool or uint8, one value per row of logits")
    return _Args(S, L, E, topk_idx.shape[-1], route_mode, float(coef))


def _place(t: torch.Tensor, a: _Args) -> Tuple[int, int, int]:
    """(address, row stride, sequence stride); rows do not overlap."""
    ld = t.stride(-2) if a.L > 1 else a.E
    return t.data_ptr(), ld, t.stride(0) if t.dim() == 3 and a.S > 1 else 0


def _forward(logits, topk_idx, mask, a: _Args, grad_loss, d_logits) -> BalanceLoss:
    dev = logits.device
    nbytes = (abi._lib or abi.load()).chimere_b200_balance_loss_bytes(a.S, a.L, a.E, a.k)
    _need(nbytes > 0, "logits up to 256 wide, up to 256 ids per row, fewer than 2^31 rows and ids")
    S = () if logits.dim() == 2 else (a.S,)
    loss = torch.empty(S, dtype=torch.float32, device=dev)
    tokens = torch.empty(S, dtype=torch.int32, device=dev)
    counts = torch.empty(*S, a.E, dtype=torch.int32, device=dev)
    prob = torch.empty(*S, a.E, dtype=torch.float32, device=dev)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    p, ld, stride = _place(logits, a)
    dp, ldd, stride_d = (None, a.E, 0) if d_logits is None else _place(d_logits, a)
    _call("chimere_b200_balance_loss", logits.get_device(), p, _TYPES[logits.dtype], ld, stride, topk_idx.data_ptr(), None if mask is None else mask.data_ptr(), a.S, a.L, a.E, a.k, a.mode,
          a.coef, loss.data_ptr(), counts.data_ptr(), prob.data_ptr(), tokens.data_ptr(), None if grad_loss is None else grad_loss.data_ptr(), dp, ldd, stride_d,
          ws.data_ptr(), nbytes)
    return BalanceLoss(loss, counts, prob, tokens)


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, topk_idx, mask, a):
        r = _forward(logits, topk_idx, mask, a, None, None)
        ctx.a = a
        ctx.save_for_backward(logits, r.counts, r.tokens, *(() if mask is None else (mask,)))
        ctx.mark_non_differentiable(r.counts, r.prob, r.tokens)
        return r.loss, r.counts, r.prob, r.tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss, *_):
        logits, counts, tokens, *mask = ctx.saved_tensors
        return balance_loss_backward(logits, counts, tokens, ctx.a.k, mask[0] if mask else None, ctx.a.mode, ctx.a.coef, grad_loss.contiguous()), None, None, None


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, mask: Optional[torch.Tensor] = None, route_mode: int = abi.ROUTE_SOFTMAX_RENORM,
                 coef: float = 1.0) -> BalanceLoss:
    """Loss, counts, mean probabilities and tokens of each sequence.  logits [T, E] or [S, L, E] (E <= 256) of float32, float16 or bfloat16; topk_idx int32 [..., top_k]: an
    id outside [0, E) counts nowhere; mask bool or uint8 [T] or [S, L]: tokens that are false are left out, whatever they hold.  The loss is differentiable
    with respect to the logits (the counts are constants in it); where gradients are wanted at once, balance_loss_grad saves a pass."""
    a = _check(logits, topk_idx, mask, route_mode, coef)
    if torch.is_grad_enabled() and logits.requires_grad:
        return BalanceLoss(*_Loss.apply(logits, topk_idx, mask, a))
    return _forward(logits, topk_idx, mask, a, None, None)


def _grad_loss(grad_loss, logits, a: _Args):
    if grad_loss is None:
        return None
    shape = () if logits.dim() == 2 else (a.S,)
    _need(grad_loss.dtype == torch.float32 and grad_loss.device == logits.device and grad_loss.shape == shape and grad_loss.is_contiguous(),
          f"grad_loss: contiguous float32 {shape} on the logits' device")
    return grad_loss


def balance_loss_grad(logits: torch.Tensor, topk_idx: torch.Tensor, mask: Optional[torch.Tensor] = None, route_mode: int = abi.ROUTE_SOFTMAX_RENORM,
                      coef: float = 1.0, grad_loss: Optional[torch.Tensor] = None) -> Tuple[BalanceLoss, torch.Tensor]:
    """balance_loss and, in the same pass over the logits, their gradient: (result, grad_logits).  grad_loss: f32, one per sequence, 1 unless
    given.  grad_logits has the logits' type and shape; tokens that the mask leaves out have zeros.  No autograd graph is made."""
    a = _check(logits, topk_idx, mask, route_mode, coef)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    return _forward(logits, topk_idx, mask, a, _grad_loss(grad_loss, logits, a), d), d


def balance_loss_backward(logits: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor, top_k: int, mask: Optional[torch.Tensor] = None,
                          route_mode: int = abi.ROUTE_SOFTMAX_RENORM, coef: float = 1.0, grad_loss: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of the logits from a balance_loss result's counts and tokens -- or from those of several ranks, added up, for a loss over the
    whole batch."""
    a = _check(logits, torch.empty(*logits.shape[:-1], 0, dtype=torch.int32, device=logits.device), mask, route_mode, coef)._replace(k=top_k)
    shape = () if logits.dim() == 2 else (a.S,)
    for t, s, name in ((counts, shape + (a.E,), "counts"), (tokens, shape, "tokens")):
        _need(t.dtype == torch.int32 and t.device == logits.device and t.shape == s and t.is_contiguous(), f"{name}: contiguous int32 {s} on the logits' device")
    g = _grad_loss(grad_loss, logits, a)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    p, ld, stride = _place(logits, a)
    dp, ldd, stride_d = _place(d, a)
    _call("chimere_b200_balance_loss_backward", logits.get_device(), p, _TYPES[logits.dtype], ld, stride, None if mask is None else mask.data_ptr(), counts.data_ptr(),
          tokens.data_ptr(), a.S, a.L, a.E, top_k, a.mode, a.coef, None if g is None else g.data_ptr(), dp, ldd, stride_d)
    return d
