"""Balance-loss calls at the edges of what their documentation allows."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from chimere_b200 import balance

pytestmark = pytest.mark.gpu


def inputs(S, L, E, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(S, L, E, generator=g, device="cuda"), torch.randint(0, E, (S, L, k), generator=g, device="cuda", dtype=torch.int32)


def test_forward_mode_is_refused():
    """A tangent is not dropped without a word."""
    logits, ids = inputs(2, 9, 16, 2)
    tangent = torch.ones_like(logits)
    with forward_ad.dual_level():
        for primal in (logits, logits.clone().requires_grad_()):
            with pytest.raises((RuntimeError, NotImplementedError)):
                balance.balance_loss(forward_ad.make_dual(primal, tangent), ids)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
                balance.balance_loss(forward_ad.make_dual(primal, tangent), ids)
        with pytest.raises((RuntimeError, NotImplementedError)):
            balance.balance_loss_grad(forward_ad.make_dual(logits, tangent), ids)
        r = balance.balance_loss(logits, ids)          # (a plain tensor beside them)
        assert torch.equal(r.loss, balance.balance_loss(logits.clone(), ids).loss)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda l: balance.balance_loss(l, ids).loss, (logits,), (tangent,))
    assert torch.equal(balance.balance_loss(logits, ids).loss, r.loss)


def test_sizes_beyond_32_bits_are_refused():
    """What the C entry would see cut to 32 bits."""
    logits, ids = inputs(1, 4, 16, 2)
    wide = torch.zeros(1, 2 ** 32 + 16, dtype=torch.float16, device="cuda")
    r = balance.balance_loss(logits, ids)
    calls = [lambda: balance.balance_loss(wide, ids[0, :1]), lambda: balance.balance_loss_grad(wide, ids[0, :1]), lambda: balance.balance_loss(logits, ids, route_mode=2 ** 32),
             lambda: balance.balance_loss_backward(logits, r.counts, r.tokens, 2 ** 32 + 2), lambda: balance.balance_loss_backward(logits, r.counts, r.tokens, 2, route_mode=2 ** 32)]
    for i, f in enumerate(calls):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
