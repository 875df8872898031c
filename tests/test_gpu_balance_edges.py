"""Balance-loss calls at the edges of what their documentation allows."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from chimere_b200 import abi, balance
from test_gpu_balance import check, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


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


@pytest.mark.parametrize("mode", [abi.ROUTE_SOFTMAX_RENORM, abi.ROUTE_SIGMOID_NORM_SCALE])
@pytest.mark.parametrize("S,L,E", [(56, 400000, 3), (60, 40000, 130), (1, 1 << 23, 200), (1, 1 << 23, 64)])
def test_mean_probabilities_of_long_pieces(S, L, E, mode):
    """Equal rows, whose probabilities are no powers of two: sums in fp32 would drift, all in one direction.  Of a probability: the difference of the logits and the weighted
    one, 1 u each, and 32 u (as in the bounds of the other tests); in sigmoid mode 2 |z| + 4 <= 6.7 u more for log sigmoid, for the value and for the row's sum.  Up to 64 values, and the lanes of
    a warp that have the same expert, are added up in fp32: 63 + 2 u; the piece's sum and the mean are rounded once each."""
    row = torch.zeros(E, dtype=torch.float64, device="cuda")
    row[0] = 1.0
    logits = torch.zeros(S, L, E, dtype=torch.bfloat16, device="cuda")
    logits[..., 0] = 1.0
    ids = torch.zeros(S, L, 1, dtype=torch.int32, device="cuda")
    r = balance.balance_loss(logits, ids, route_mode=mode)
    p = torch.softmax(row if mode == abi.ROUTE_SOFTMAX_RENORM else torch.nn.functional.logsigmoid(row), 0)
    bound = (2 + 32 + (14 if mode == abi.ROUTE_SIGMOID_NORM_SCALE else 0) + 65 + 2) * U
    off = ((r.prob.double() - p) / p).abs().max().item()
    assert off <= bound, (off / U, bound / U)
    assert ((r.loss.double() - E * p[0]).abs() <= E * p[0] * (bound + 2 * U)).all() and (r.tokens == L).all() and (r.counts[:, 0] == L).all()


@pytest.mark.parametrize("mode", [abi.ROUTE_SOFTMAX_RENORM, abi.ROUTE_SIGMOID_NORM_SCALE])
@pytest.mark.parametrize("S,L,E", [(1, 40000, 256), (1, 100000, 8), (3, 1025, 130), (1, 1024, 33), (5, 5000, 60), (60, 700, 40), (1, 2049, 200), (2, 8191, 97), (55, 1500, 128), (1, 33, 5)])
def test_every_row_counts_once(S, L, E, mode):
    """Equal rows again, in pieces of up to 64 rows per lane: a row lost or taken twice at an edge of a piece moves the mean probability by 1 / L, at least 10^-5, which the bound above
    (115 u, 7 10^-6) does not hide.  The last row differs, so that it is seen whose place it takes."""
    logits = torch.zeros(S, L, E, device="cuda")
    logits[..., 0] = 1.0
    logits[:, -1, :] = logits[:, -1, :].flip(-1)
    ids = torch.zeros(S, L, 1, dtype=torch.int32, device="cuda")
    r = balance.balance_loss(logits, ids, route_mode=mode)
    z = logits.double() if mode == abi.ROUTE_SOFTMAX_RENORM else torch.nn.functional.logsigmoid(logits.double())
    p = torch.softmax(z, 2).mean(1)
    off = ((r.prob.double() - p) / p).abs().max().item()
    assert off <= 115 * U, off / U
    assert (r.tokens == L).all() and (r.counts[:, 0] == L).all()


@pytest.mark.parametrize("mode", [abi.ROUTE_SOFTMAX_RENORM, abi.ROUTE_SIGMOID_NORM_SCALE])
@pytest.mark.parametrize("S,L,E,k,dtype", [(60, 9001, 256, 2, torch.float32), (1, 700001, 130, 1, torch.bfloat16), (57, 70003, 31, 3, torch.float16), (60, 30001, 64, 2, torch.bfloat16)])
def test_long_pieces_against_64_bits(S, L, E, k, dtype, mode):
    logits, ids = inputs(S, L, E, k, seed=L)
    logits = logits.to(dtype)
    mask = torch.rand(S, L, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.6
    mask[0, L // 3:] = False
    r, d = balance.balance_loss_grad(logits, ids, mask=mask, route_mode=mode)
    alone = balance.balance_loss(logits, ids, mask=mask, route_mode=mode)
    assert all(torch.equal(a, b) for a, b in zip(alone, r))
    assert torch.equal(d, balance.balance_loss_backward(logits, r.counts, r.tokens, k, mask=mask, route_mode=mode))
    for s in range(0, S, 20):       # (64-bit copies of a few sequences at a time)
        part = slice(s, min(s + 20, S))
        check(balance.BalanceLoss(*(t[part] for t in r)), d[part], reference(logits[part], ids[part], mask[part], mode))


def test_the_longest_sequence():
    """Row numbers up to the last that 32 bits hold: one expert, whose probability is 1, and a mask that leaves the last rows and some in front."""
    L = 0x7FFFFF00
    logits, ids = torch.zeros(L, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(L, 1, dtype=torch.int32, device="cuda")
    r, d = balance.balance_loss_grad(logits, ids)
    assert r.tokens.item() == L and r.counts.item() == L and r.prob.item() == 1 and r.loss.item() == 1 and not d.any()
    mask = torch.zeros(L, dtype=torch.bool, device="cuda")
    mask[-1000:], mask[5], mask[L // 2] = True, True, True
    ids[-3:] = -1
    r = balance.balance_loss(logits, ids, mask=mask, route_mode=abi.ROUTE_SIGMOID_NORM_SCALE)
    assert r.tokens.item() == 1002 and r.counts.item() == 999 and r.prob.item() == 1 and abs(r.loss.item() - 999 / 1002) <= 2 * U


@pytest.mark.parametrize("E", [8, 200])
def test_counts_of_many_ranks(E):
    """Counts that add up to more than 31 bits, near an even load: the gradient hangs on their differences."""
    k, n = 2, 2 * 10 ** 9
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = torch.randn(50, E, generator=g, device="cuda")
    counts = (k * n // E + torch.randint(-1000, 1001, (E,), generator=g, device="cuda")).to(torch.int32)
    tokens = torch.tensor(n, dtype=torch.int32, device="cuda")
    d = balance.balance_loss_backward(logits, counts, tokens, k, grad_loss=torch.tensor(1e15, device="cuda"))
    l = logits.double()
    p = torch.softmax(l, 1)
    off = l.amax(1, keepdim=True) - l
    ep = p * (off + (p * off).sum(1, keepdim=True) + 32) * U             # (as in the bounds of the other tests)
    f = counts.double()
    slope = 1e15 * E / (k * float(n) ** 2) * (f - f.mean())
    dot = (p * slope).sum(1, keepdim=True)
    e_dot = (ep * slope.abs() + p * slope.abs() * 24 * U).sum(1, keepdim=True)
    want = p * (slope - dot)
    bound = ep * (slope - dot).abs() + (p + ep) * (2 * U * slope.abs() + e_dot + U * (slope - dot).abs()) + 5 * U * want.abs()
    assert ((d.double() - want).abs() <= bound * 1.01).all(), ((d.double() - want).abs() / bound).max()
