"""The balance loss, its counts and its gradient against their formulas in 64 bits, and against differences.

Bounds in u = 2^-24.  exp(l - max): the difference is rounded (its size times u), expf is off by two steps (4 u at most); the sum of a row's values adds up to 13
roundings, its reciprocal and the product two more: a probability is off by p * (d + sum_j p_j d_j + 32) u with d = max - l.  In sigmoid mode log sigmoid itself is
rounded: (2 |z| + 4) u more in d.  Sums over a piece: a lane adds up to rows / 8 values and eight warps meet in 64 bits."""
import math

import pytest
import torch

from chimere_b200 import abi, balance, configs
from chimere_b200.layer import MoeScratch, MoeWeightsTiled, route_only

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SOFTMAX, SIGMOID = abi.ROUTE_SOFTMAX_RENORM, abi.ROUTE_SIGMOID_NORM_SCALE
TYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(S, L, E, k, dtype=torch.float32, seed=0, spread=2.0):
    g = gen(seed + S * 1000 + L + E)
    logits = (torch.randn(S, L, E, generator=g, device="cuda") * spread).to(dtype)
    ids = torch.randint(0, E, (S, L, k), generator=g, device="cuda", dtype=torch.int32)
    return logits, ids


def reference(logits, ids, mask=None, mode=SOFTMAX, coef=1.0, grad_loss=None):
    """Everything in 64 bits, with bounds."""
    S, L, E = logits.shape
    k = ids.shape[2]
    on = torch.ones(S, L, dtype=torch.bool, device="cuda") if mask is None else mask.bool()
    l = torch.where(on[:, :, None], logits.double(), 0.0)
    z = l if mode == SOFTMAX else torch.nn.functional.logsigmoid(l)
    mx = z.amax(2, keepdim=True)
    none = torch.isneginf(mx)
    p = torch.where(none, 0.0, torch.softmax(z, 2)) * on[:, :, None]
    d = torch.where(p > 0, (mx - z).nan_to_num(0.0), 0.0)
    if mode == SIGMOID:
        d = d + torch.where(p > 0, 2 * z.abs().nan_to_num(0.0) + 4, 0.0)
    ep = p * (d + (p * d).sum(2, keepdim=True) + 32) * U + 2.0 ** -126
    inside = (ids >= 0) & (ids < E) & on[:, :, None]
    counts = torch.zeros(S, E + 1, dtype=torch.int64, device="cuda").scatter_add_(1, torch.where(inside, ids.long(), E).reshape(S, -1), torch.ones(S, L * k, dtype=torch.int64, device="cuda"))[:, :E]
    n = on.sum(1)
    nn = n.clamp_min(1).double()
    prob = p.sum(1) / nn[:, None]
    e_prob = (ep.sum(1) + p.sum(1) * (L / 8 + 8) * U) / nn[:, None] + prob * U + 2.0 ** -149
    c = coef * E / (k * nn)
    loss = c * (counts * prob).sum(1)
    e_loss = c * (counts * e_prob).sum(1) + 2 * U * loss.abs()
    gl = torch.ones(S, dtype=torch.float64, device="cuda") if grad_loss is None else grad_loss.double()
    g = ((c / nn * gl)[:, None] * (counts - counts.sum(1, keepdim=True) / E))[:, None, :]
    dot = (p * g).sum(2, keepdim=True)
    e_dot = (ep * g.abs() + p * g.abs() * 24 * U).sum(2, keepdim=True)
    grad = p * (g - dot)
    e = ep * (g - dot).abs() + (p + ep) * (U * g.abs() + e_dot + U * (g - dot).abs()) + 4 * U * grad.abs()
    if mode == SIGMOID:
        slope = torch.sigmoid(-l)
        e = e * slope + grad.abs() * 8 * U * slope
        grad = grad * slope
    e = e + torch.finfo(logits.dtype).eps / 2 * (grad.abs() + e) + TINY[logits.dtype]
    keep = on[:, :, None] & ~none
    return {"loss": (loss, e_loss), "counts": counts, "prob": (prob, e_prob), "tokens": n, "grad": (torch.where(keep, grad, 0.0), torch.where(keep, e, 0.0))}


def close(x, ref_bound, name):
    ref, bound = ref_bound
    assert x.shape == ref.shape, name
    off = (x.double() - ref).abs()
    bad = ~(off <= bound * 1.01)
    assert not bad.any(), (name, int(bad.sum()), off[bad][:4], bound[bad][:4], bad.nonzero()[:4])


def check(r, d, ref):
    close(r.loss, ref["loss"], "loss")
    close(r.prob, ref["prob"], "prob")
    assert r.counts.dtype == torch.int32 and torch.equal(r.counts.long(), ref["counts"]) and torch.equal(r.tokens.long(), ref["tokens"])
    if d is not None:
        close(d, ref["grad"], "grad")


def bits(r, d):
    return [t.clone() for t in r] + ([] if d is None else [d.clone()])


SHAPES = [(1, 1, 1, 1), (1, 1, 256, 8), (1, 24, 256, 8), (3, 17, 5, 2), (2, 64, 32, 4), (2, 65, 33, 3), (4, 1000, 128, 6), (5, 333, 64, 1), (1, 3000, 255, 8), (2, 2048, 60, 7), (300, 70, 16, 2), (60, 700, 40, 3), (100, 600, 64, 4), (500, 513, 8, 1), (7, 513, 256, 8), (2, 1025, 100, 4), (3, 1024, 48, 2),
          (1, 40000, 256, 8), (64, 129, 130, 256), (1, 100000, 8, 2)]


@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("S,L,E,k", SHAPES)
def test_against_64_bits(S, L, E, k, mode):
    for i, dtype in enumerate(TYPES):
        logits, ids = inputs(S, L, E, k, dtype, seed=i)
        mask = (torch.rand(S, L, generator=gen(i), device="cuda") < 0.7) if i else None
        gl = torch.randn(S, generator=gen(i), device="cuda") if i == 2 else None
        r, d = balance.balance_loss_grad(logits, ids, mask=mask, route_mode=mode, coef=0.5, grad_loss=gl)
        ref = reference(logits, ids, mask, mode, 0.5, gl)
        assert d.dtype == dtype
        check(r, d, ref)
        alone = balance.balance_loss(logits, ids, mask=mask, route_mode=mode, coef=0.5)
        assert all(torch.equal(a, b) for a, b in zip(alone, r))          # the same sums with and without the gradient
        d2 = balance.balance_loss_backward(logits, r.counts, r.tokens, k, mask=mask, route_mode=mode, coef=0.5, grad_loss=gl)
        assert torch.equal(d, d2)
        again, d3 = balance.balance_loss_grad(logits, ids, mask=mask, route_mode=mode, coef=0.5, grad_loss=gl)
        assert all(torch.equal(a, b) for a, b in zip(bits(r, d), bits(again, d3)))


@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("S,L,E,k", [(1, 6, 5, 2), (2, 200, 64, 4)])
def test_gradient_against_differences(S, L, E, k, mode):
    """(loss(l + h) - loss(l - h)) / 2h of the reference in 64 bits, in a few random directions: exact but for h^2."""
    logits, ids = inputs(S, L, E, k, seed=3)
    gl = torch.randn(S, generator=gen(5), device="cuda")
    _, d = balance.balance_loss_grad(logits, ids, route_mode=mode, coef=1.5, grad_loss=gl)

    def loss(l):
        p = torch.softmax(l, 2) if mode == SOFTMAX else torch.sigmoid(l) / torch.sigmoid(l).sum(2, keepdim=True)
        f = torch.zeros(S, E, dtype=torch.float64, device="cuda").scatter_add_(1, ids.reshape(S, -1).long(), torch.ones(S, L * k, dtype=torch.float64, device="cuda"))
        return (1.5 * E / (k * L) * (f * p.mean(1)).sum(1) * gl.double()).sum()

    h = 1e-4
    for seed in range(4):
        v = torch.randn(S, L, E, generator=gen(seed), device="cuda", dtype=torch.float64)
        want = (loss(logits.double() + h * v) - loss(logits.double() - h * v)) / (2 * h)
        got = (d.double() * v).sum()
        size = (d.double().abs() * v.abs()).sum()
        assert abs(got - want) <= size * (1e-6 + 100 * h * h) + 1e-9      # (differences: h^2 of the third derivative, rounding 1e-16 / h)


@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
def test_rows_left_out_may_hold_anything(mode):
    S, L, E, k = 3, 400, 96, 4
    logits, ids = inputs(S, L, E, k, seed=8)
    mask = torch.rand(S, L, generator=gen(1), device="cuda") < 0.5
    mask[1] = False                                  # a sequence with nothing left
    want = bits(*balance.balance_loss_grad(logits, ids, mask=mask, route_mode=mode))
    dirty, dirty_ids = logits.clone(), ids.clone()
    dirty[~mask] = float("nan")
    dirty[0][~mask[0]] = float("inf")
    dirty_ids[~mask] = 2 ** 31 - 1
    got = bits(*balance.balance_loss_grad(dirty, dirty_ids, mask=mask, route_mode=mode))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0][1] == 0 and got[3][1] == 0 and (got[1][1] == 0).all() and (got[2][1] == 0).all() and (got[4][~mask] == 0).all()
    assert torch.equal(bits(*balance.balance_loss_grad(dirty, dirty_ids, mask=mask.to(torch.uint8) * 7, route_mode=mode))[0], want[0])


@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("L", [20, 700])
def test_values_at_the_ends_of_the_range(mode, L):
    S, E, k = 2, 40, 3
    logits, ids = inputs(S, L, E, k, seed=9)
    logits[0, 0] = float("-inf")                     # no probabilities
    logits[0, 1, :39] = float("-inf")                # one expert left
    logits[0, 2] = torch.finfo(torch.float32).min    # a mask of the lowest value: even
    logits[0, 3] = 1e4 * logits[0, 3]
    logits[0, 4] = -200.0 + logits[0, 4]             # sigmoids below fp32's range
    logits[0, 5, 7] = torch.finfo(torch.float32).max
    r, d = balance.balance_loss_grad(logits, ids, route_mode=mode)
    check(r, d, reference(logits, ids, mode=mode))
    assert (d[0, 0] == 0).all()
    bad = logits.clone()
    bad[1, 5, 3] = float("nan")
    r2, d2 = balance.balance_loss_grad(bad, ids, route_mode=mode)
    assert torch.isnan(r2.loss[1]) and torch.isnan(d2[1, 5]).all() and torch.equal(r2.loss[0], r.loss[0]) and torch.equal(r2.counts, r.counts)
    rest = torch.ones(S, L, dtype=torch.bool, device="cuda")
    rest[1, 5] = False
    assert torch.equal(d2[rest], d[rest])
    top = logits.clone()
    top[1, 5, 3] = float("inf")
    r3, d3 = balance.balance_loss_grad(top, ids, route_mode=mode)
    if mode == SOFTMAX:
        assert torch.isnan(r3.loss[1]) and torch.isnan(d3[1, 5]).all()
    else:
        check(r3, d3, reference(top, ids, mode=mode))


@pytest.mark.parametrize("L", [30, 900, 1900])
def test_ids_outside_and_repeated(L):
    logits, ids = inputs(2, L, 48, 4, seed=10)
    ids[0, :, 0] = -1
    ids[0, 1] = 5                                    # the same expert four times
    ids[1, 2, 1], ids[1, 3, 1] = 48, -2 ** 31
    check(*balance.balance_loss_grad(logits, ids), reference(logits, ids))
    ids[:] = 47                                      # all on the last expert
    check(*balance.balance_loss_grad(logits, ids), reference(logits, ids))
    ids[:] = -7
    r, d = balance.balance_loss_grad(logits, ids)
    assert (r.loss == 0).all() and (r.counts == 0).all() and (d == 0).all()


@pytest.mark.parametrize("L", [40, 4000])
def test_a_grad_loss_that_is_not_finite_leaves_masked_rows_alone(L):
    logits, ids = inputs(3, L, 64, 4, seed=15)
    mask = torch.rand(3, L, generator=gen(3), device="cuda") < 0.5
    mask[2] = False
    _, d = balance.balance_loss_grad(logits, ids, mask=mask, grad_loss=torch.tensor([float("nan"), float("inf"), float("inf")], device="cuda"))
    assert (d[~mask] == 0).all() and torch.isnan(d[0][mask[0]]).all()


def test_more_than_2_31_logits():
    """Offsets beyond 32 bits: the last rows' gradients, and counts and mean probabilities of all."""
    T, E = (1 << 31) // 256 + 1000, 256
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    logits[-500:] = torch.randn(500, E, generator=gen(1), device="cuda").to(torch.bfloat16)
    ids[-500:] = torch.randint(0, E, (500, 1), generator=gen(2), device="cuda", dtype=torch.int32)
    r, d = balance.balance_loss_grad(logits, ids, grad_loss=torch.tensor(1e9, device="cuda"))
    counts = torch.bincount(ids.reshape(-1).long(), minlength=E)
    assert torch.equal(r.counts.long(), counts) and r.tokens.item() == T
    p = torch.softmax(logits[-500:].double(), 1)
    prob = (p.sum(0) + (T - 500) / E) / T
    assert ((r.prob.double() - prob).abs() <= prob * 20000 * U).all()       # (a lane adds 19000 / 8 values of 1 / 256 and fewer)
    g = 1e9 * E / float(T) ** 2 * (counts.double() - T / E)
    want = p * (g - (p * g).sum(1, keepdim=True))
    assert ((d[-500:].double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-3 * want.abs().max()).all()
    flat = 1 / E * (g - g.mean())
    assert ((d[12345].double() - flat).abs() <= flat.abs() * 2.0 ** -7 + 1e-6 * flat.abs().max()).all()


def test_even_load_gives_coef():
    E, k = 64, 4
    logits = torch.zeros(E, E, device="cuda")
    ids = ((torch.arange(E, device="cuda")[:, None] + torch.arange(k, device="cuda")) % E).to(torch.int32)
    r, d = balance.balance_loss_grad(logits, ids, coef=0.25)
    assert abs(r.loss.item() - 0.25) <= 0.25 * 64 * U and (r.counts == k).all() and (d == 0).all() and r.tokens.item() == E
    assert r.loss.shape == () and r.tokens.shape == () and r.counts.shape == (E,) and r.prob.shape == (E,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lo,hi", [(0, 128), (1, 129), (3, 98), (4, 100)])
def test_logits_inside_a_wider_tensor(dtype, lo, hi):
    wide, _ = inputs(4, 300, 200, 1, dtype, seed=11)
    for view in (wide[:, 10:130, lo:hi], wide[1:3, ::2, lo:hi], wide[::3, :1, lo:hi], wide[:1, 5:95, lo:hi]):
        ids = torch.randint(0, hi - lo, (*view.shape[:2], 3), generator=gen(lo), device="cuda", dtype=torch.int32)
        r, d = balance.balance_loss_grad(view, ids)
        check(r, d, reference(view, ids))
        want = balance.balance_loss_grad(view.contiguous(), ids)
        assert all(torch.equal(a, b) for a, b in zip(bits(r, d), bits(*want)))


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd(dtype):
    logits, ids = inputs(3, 500, 100, 4, dtype, seed=12)
    mask = torch.rand(3, 500, generator=gen(2), device="cuda") < 0.8
    weight = torch.tensor([0.5, -1.0, 2.0], device="cuda")
    leaf = logits.clone().requires_grad_()
    r = balance.balance_loss(leaf, ids, mask=mask, route_mode=SIGMOID, coef=0.01)
    assert r.loss.requires_grad and not r.prob.requires_grad and not r.counts.requires_grad
    (r.loss * weight).sum().backward()
    _, d = balance.balance_loss_grad(logits, ids, mask=mask, route_mode=SIGMOID, coef=0.01, grad_loss=weight)
    assert torch.equal(leaf.grad, d)
    leaf.grad = None
    balance.balance_loss(leaf, ids, mask=mask, route_mode=SIGMOID, coef=0.01).loss.sum().backward()      # (a gradient that is one number, broadcast)
    assert torch.equal(leaf.grad, balance.balance_loss_grad(logits, ids, mask=mask, route_mode=SIGMOID, coef=0.01)[1])
    with torch.no_grad():
        assert not balance.balance_loss(leaf, ids).loss.requires_grad
    flat = logits[0].clone().requires_grad_()
    balance.balance_loss(flat, ids[0]).loss.backward()
    assert torch.equal(flat.grad, balance.balance_loss_grad(logits[0], ids[0])[1])


def test_counts_of_several_ranks():
    """A batch split over two ranks: their counts and tokens added up give the gradient of the whole batch's loss."""
    logits, ids = inputs(1, 600, 64, 4, seed=13)
    whole, d = balance.balance_loss_grad(logits[0], ids[0])
    parts = [balance.balance_loss(logits[0, a:b], ids[0, a:b].contiguous()) for a, b in ((0, 250), (250, 600))]
    counts, tokens = parts[0].counts + parts[1].counts, parts[0].tokens + parts[1].tokens
    assert torch.equal(counts, whole.counts) and torch.equal(tokens, whole.tokens)
    mine = balance.balance_loss_backward(logits[0, 250:], counts, tokens, 4)
    assert torch.equal(mine, d[250:])


@pytest.mark.parametrize("cfg,T", [(configs.QWEN_Q4_0_ZIPF, 5), (configs.QWEN_Q4_0_ZIPF, 300), (configs.NEMOTRON_Q4_0, 64)])
def test_behind_the_router(cfg, T):
    """The package's router, its ids and logits, and the loads it traces."""
    cfg = configs.scaled(cfg, H=512, F=256, F_s=0)
    layer = MoeWeightsTiled(configs.make_layer(cfg, device="cuda"))
    sc = MoeScratch(layer, T)
    route_only(layer, sc, configs.make_input(cfg, T, device="cuda"))
    logits, ids = sc.router_logits(T), sc.topk_indices(T)
    r, d = balance.balance_loss_grad(logits, ids, route_mode=cfg.route_mode)
    ref = reference(logits[None], ids[None], mode=cfg.route_mode)
    check(balance.BalanceLoss(*(t[None] for t in r)), d[None], ref)
    assert torch.equal(torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), r.counts.cumsum(0)]), sc.offsets().long())


@pytest.mark.parametrize("L", [50, 5000])
def test_capture_and_replay_with_new_inputs(L):
    logits, ids = inputs(2, L, 64, 4, seed=14)
    leaf = logits.clone().requires_grad_()

    def run():
        r, d = balance.balance_loss_grad(logits, ids)
        t = balance.balance_loss(leaf, ids)
        return bits(r, d) + [torch.autograd.grad(t.loss.sum(), leaf)[0]]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        run()
        stream.synchronize()
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                outs.append(run())
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(3):
        new, new_ids = inputs(2, L, 64, 4, seed=20 + seed)
        logits.copy_(new)
        ids.copy_(new_ids)
        with torch.no_grad():
            leaf.copy_(new)
        for graph, out in zip(graphs, outs):
            graph.replay()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_two_streams_at_once():
    sets = [inputs(1, 20000, 128, 4, seed=s) for s in range(2)]
    want = [bits(*balance.balance_loss_grad(*s)) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(20):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(bits(*balance.balance_loss_grad(*s)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for r in got[i] for a, b in zip(r, want[i]))


def test_no_tokens():
    r, d = balance.balance_loss_grad(torch.empty(0, 16, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert r.loss.item() == 0 and r.tokens.item() == 0 and (r.counts == 0).all() and (r.prob == 0).all() and d.shape == (0, 16)
    r, d = balance.balance_loss_grad(torch.empty(0, 5, 16, device="cuda"), torch.empty(0, 5, 2, dtype=torch.int32, device="cuda"))
    assert r.loss.shape == (0,) and d.shape == (0, 5, 16)
    leaf = torch.empty(3, 0, 16, device="cuda", requires_grad=True)
    balance.balance_loss(leaf, torch.empty(3, 0, 2, dtype=torch.int32, device="cuda")).loss.sum().backward()
    assert leaf.grad.shape == (3, 0, 16)


def test_arguments_that_are_refused():
    logits, ids = inputs(2, 10, 16, 2)
    bad = [lambda: balance.balance_loss(logits.double(), ids), lambda: balance.balance_loss(logits.cpu(), ids), lambda: balance.balance_loss(logits, ids.long()),
           lambda: balance.balance_loss(logits, ids[:1]), lambda: balance.balance_loss(logits, ids[:, :, ::2]), lambda: balance.balance_loss(logits.transpose(1, 2), ids),
           lambda: balance.balance_loss(logits, ids, mask=torch.ones(2, 9, device="cuda").bool()), lambda: balance.balance_loss(logits, ids, mask=torch.ones(2, 10, device="cuda")),
           lambda: balance.balance_loss(logits, ids, mask=torch.ones(2, 10).bool()), lambda: balance.balance_loss(*inputs(1, 4, 257, 2)), lambda: balance.balance_loss(*inputs(1, 4, 16, 257)),
           lambda: balance.balance_loss_grad(logits, ids, grad_loss=torch.ones(3, device="cuda")), lambda: balance.balance_loss_grad(logits, ids, grad_loss=torch.ones(2, device="cuda").double()),
           lambda: balance.balance_loss_backward(logits, torch.zeros(2, 15, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda"), 2),
           lambda: balance.balance_loss_backward(logits, torch.zeros(2, 16, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda"), 2)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError, match="bad dimension"):
        balance.balance_loss(logits, ids, route_mode=2)
    with pytest.raises(RuntimeError, match="bad dimension"):
        balance.balance_loss(logits[:, :1].expand(2, 10, 16), ids)
    assert math.isfinite(balance.balance_loss(logits, ids).loss.sum().item())
