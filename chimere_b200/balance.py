"""The router's balance loss, its pairs per expert and its gradient, over the C ABI.

What a router is trained and watched with: it takes the logits and the expert ids the package's router leaves (MoeScratch.router_logits,
.topk_indices) or any others.  The reference only logs the experts' load (chimere-server/src/qwen35_model/moe_ffn.rs:120-131).

    p = softmax(logits), or sigmoid(logits) / their sum          n = tokens that the mask leaves
    loss = coef * E / (top_k * n) * sum_e counts[e] * prob[e]    prob[e] = mean of p over them; an even load gives coef, n = 0 gives 0
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import abi
from .w8a8 import _TYPES, _call, _ints


class BalanceLoss(NamedTuple):
    """Of each sequence (without the leading dimension for logits [T, E])."""
    loss: torch.Tensor     # f32 [S]
    counts: torch.Tensor   # int32 [S, E]: pairs per expert
    prob: torch.Tensor     # f32 [S, E]: mean probability
    tokens: torch.Tensor   # int32 [S]: tokens that the mask leaves


_Args = Tuple[int, int, int, int, int, float]     # S, L, E, top_k, route mode, coef


def _check(logits, topk_idx, mask, route_mode, coef) -> _Args:
    shape, index = logits.shape, logits.get_device()
    if index < 0 or len(shape) not in (2, 3) or logits.dtype not in _TYPES:
        raise ValueError("logits: [T, E] or [S, L, E] of float32, float16 or bfloat16 on a CUDA device")
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(logits).tangent is not None:     # (below 0: no dual tensors at all)
        raise NotImplementedError("logits: a dual tensor (there is no forward mode, its tangent would be lost)")
    if logits.stride(-1) != 1 and shape[-1] != 1:
        raise ValueError("logits: the values of a row lie side by side")
    if topk_idx.dtype is not torch.int32 or topk_idx.get_device() != index or topk_idx.shape[:-1] != shape[:-1] or not topk_idx.is_contiguous():
        raise ValueError("topk_idx: contiguous int32, one row of ids per row of logits")
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.get_device() != index or mask.shape != shape[:-1] or not mask.is_contiguous()):
        raise ValueError("mask: contiguous bool or uint8, one value per row of logits")
    S, L, E = shape if len(shape) == 3 else (1, *shape)
    _ints(E | topk_idx.shape[-1] | route_mode)
    return S, L, E, topk_idx.shape[-1], route_mode, float(coef)


def _place(t: torch.Tensor, S: int, L: int, E: int) -> Tuple[int, int, int]:
    """(address, row stride, sequence stride)"""
    strides = t.stride()
    return t.data_ptr(), strides[-2] if L > 1 else E, strides[0] if S > 1 else 0


@lru_cache(maxsize=4096)
def _bytes(S: int, L: int, E: int, k: int) -> int:
    return abi.load().chimere_b200_balance_loss_bytes(S, L, E, k)


def _forward(logits, topk_idx, mask, a: _Args, grad_loss, d_logits) -> BalanceLoss:
    dev = logits.device
    S, L, E, k, mode, coef = a
    nbytes = _bytes(S, L, E, k)
    if nbytes < 0:
        raise ValueError("logits 1 to 256 wide, 1 to 256 ids per row, fewer than 2^31 rows and ids")
    if logits.dim() == 2:
        loss, tokens = torch.empty((), dtype=torch.float32, device=dev), torch.empty((), dtype=torch.int32, device=dev)
        counts, prob = torch.empty(E, dtype=torch.int32, device=dev), torch.empty(E, dtype=torch.float32, device=dev)
    else:
        loss, tokens = torch.empty(S, dtype=torch.float32, device=dev), torch.empty(S, dtype=torch.int32, device=dev)
        counts, prob = torch.empty(S, E, dtype=torch.int32, device=dev), torch.empty(S, E, dtype=torch.float32, device=dev)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p, ld, stride = _place(logits, S, L, E)
    dp, ldd, stride_d = (None, E, 0) if d_logits is None else _place(d_logits, S, L, E)
    _call("chimere_b200_balance_loss", logits.get_device(), p, _TYPES[logits.dtype], ld, stride, topk_idx.data_ptr(), None if mask is None else mask.data_ptr(), S, L, E, k, mode,
          coef, loss.data_ptr(), counts.data_ptr(), prob.data_ptr(), tokens.data_ptr(), None if grad_loss is None else grad_loss.data_ptr(), dp, ldd, stride_d,
          None if ws is None else ws.data_ptr(), nbytes)
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
        k, mode, coef = ctx.a[3:]
        return balance_loss_backward(logits, counts, tokens, k, mask[0] if mask else None, mode, coef, grad_loss.contiguous()), None, None, None


def balance_loss(logits: torch.Tensor, topk_idx: torch.Tensor, mask: Optional[torch.Tensor] = None, route_mode: int = abi.ROUTE_SOFTMAX_RENORM,
                 coef: float = 1.0) -> BalanceLoss:
    """Loss, counts, mean probabilities and tokens of each sequence.  logits [T, E] or [S, L, E] (E <= 256) of float32, float16 or bfloat16; topk_idx int32 [..., top_k]: an
    id outside [0, E) counts nowhere; mask bool or uint8 [T] or [S, L]: tokens that are false are left out, whatever they hold.  The loss is differentiable
    with respect to the logits (the counts are constants in it); where gradients are wanted at once, balance_loss_grad saves a pass.  There is no forward mode: a dual tensor is refused.  (A backward() captured in a CUDA graph follows torch's rule: no earlier autograd graph of the same
    leaves may be alive on another stream.  balance_loss_grad has no such rule.)"""
    a = _check(logits, topk_idx, mask, route_mode, coef)
    if torch.is_grad_enabled() and logits.requires_grad:
        return BalanceLoss(*_Loss.apply(logits, topk_idx, mask, a))
    return _forward(logits, topk_idx, mask, a, None, None)


def _grad_loss(grad_loss, logits):
    if grad_loss is None:
        return None
    if grad_loss.dtype is not torch.float32 or grad_loss.get_device() != logits.get_device() or grad_loss.shape != logits.shape[:-2] or not grad_loss.is_contiguous():
        raise ValueError(f"grad_loss: contiguous float32 {tuple(logits.shape[:-2])} on the logits' device")
    return grad_loss


def balance_loss_grad(logits: torch.Tensor, topk_idx: torch.Tensor, mask: Optional[torch.Tensor] = None, route_mode: int = abi.ROUTE_SOFTMAX_RENORM,
                      coef: float = 1.0, grad_loss: Optional[torch.Tensor] = None) -> Tuple[BalanceLoss, torch.Tensor]:
    """balance_loss and, in the same pass over the logits, their gradient: (result, grad_logits).  grad_loss: f32, one per sequence, 1 unless
    given.  grad_logits has the logits' type and shape; tokens that the mask leaves out have zeros.  No autograd graph is made."""
    a = _check(logits, topk_idx, mask, route_mode, coef)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    return _forward(logits, topk_idx, mask, a, _grad_loss(grad_loss, logits), d), d


def balance_loss_backward(logits: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor, top_k: int, mask: Optional[torch.Tensor] = None,
                          route_mode: int = abi.ROUTE_SOFTMAX_RENORM, coef: float = 1.0, grad_loss: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of the logits from a balance_loss result's counts and tokens -- or from those of several ranks, added up, for a loss over the
    whole batch."""
    S, L, E, _, mode, coef = _check(logits, torch.empty(*logits.shape[:-1], 0, dtype=torch.int32, device=logits.device), mask, route_mode, coef)
    _ints(top_k)
    lead = logits.shape[:-2]
    for t, s, name in ((counts, (*lead, E), "counts"), (tokens, lead, "tokens")):
        if t.dtype is not torch.int32 or t.get_device() != logits.get_device() or t.shape != s or not t.is_contiguous():
            raise ValueError(f"{name}: contiguous int32 {tuple(s)} on the logits' device")
    g = _grad_loss(grad_loss, logits)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    p, ld, stride = _place(logits, S, L, E)
    dp, ldd, stride_d = _place(d, S, L, E)
    _call("chimere_b200_balance_loss_backward", logits.get_device(), p, _TYPES[logits.dtype], ld, stride, None if mask is None else mask.data_ptr(), counts.data_ptr(),
          tokens.data_ptr(), S, L, E, top_k, mode, coef, None if g is None else g.data_ptr(), dp, ldd, stride_d)
    return d
