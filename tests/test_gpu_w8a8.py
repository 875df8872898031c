"""W8A8 products and their quantised rows against their definition in 64 bits.

Bounds, relative to 2^-24 (half a step of f32, u below): a sum converted to f32, its two scales and the bias are four roundings; an output of
fewer bits adds half a step of its own type.  silu(g) = g / (1 + exp(-g)): exp as 2^h (1 + r), ex2 off by 2^-22 (4 u), the sum 1 + r and the product one rounding
each; 1 + exp one, the reciprocal one step (2 u), the product with g one: 10 u, and silu's slope is at most 1.1; the product with u one more rounding.
Below -87, where the reciprocal is subnormal, it is 0: off by less than 88 * 2^-126."""
import numpy as np
import pytest
import torch

from chimere_b200 import abi, configs, w8a8
from chimere_b200.layer import MoeScratch, MoeWeightsTiled, route_only

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i8(g, *shape, lo=-127, hi=127):
    return w8a8.padded_i8(torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8))


def scales(g, *shape):
    return torch.rand(shape, generator=g, device="cuda") * 0.01 + 1e-4


def quantized(x):
    """The definition: both quotients rounded to f32 (from 64 bits the rounding is the same), ties to even."""
    x = x.double()
    a = x.abs().amax(dim=1)
    fine = torch.isfinite(a)
    s = torch.where(a > 0, (a / 127).float().double().clamp_min(2.0 ** -126), 0.0)
    q = torch.where((a > 0)[:, None], (x / s[:, None]).float().double().round().clamp(-127, 127), 0.0)
    q = torch.where(fine[:, None], q, 0.0).nan_to_num(0.0)
    return q.to(torch.int8), torch.where(fine, s, float("nan")).float()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


def product(q, sx, w, sw, bias, act, dtype):
    """(y, bound) in 64 bits."""
    acc = (q.double() @ w.double().T) * sx.double()[:, None] * sw.double()
    b = torch.zeros_like(sw).double() if bias is None else bias.double()
    v = acc + b
    e = 4 * U * (acc.abs() + b.abs() + v.abs())
    if act == abi.ACT_SWIGLU:
        n = v.shape[1] // 2
        g, u, eg, eu = v[:, :n], v[:, n:], e[:, :n], e[:, n:]
        s = g * torch.sigmoid(g)
        es = 1.1 * eg + 10 * U * s.abs() + 2.0 ** -119
        y, e = s * u, es * (u.abs() + eu) + s.abs() * eu + U * (s * u).abs()
    elif act == abi.ACT_RELU2:
        r = v.clamp_min(0)
        y, e = r * r, 2 * r * e + e * e + U * r * r
    else:
        y = v
    return y, 1.01 * (e + torch.finfo(dtype).eps / 2 * (y.abs() + e)) + TINY[dtype]


def check(y, ref, bound):
    assert y.shape == ref.shape
    off = (y.double() - ref).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (int(bad.sum()), off[bad][:4], bound[bad][:4], bad.nonzero()[:4])


# ---- rows ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (2, 8), (5, 2005), (4, 2048), (33, 96), (2, 40000), (1, 131071), (1200, 512), (1201, 1000), (1500, 2048), (1300, 4096), (1184, 2056),
                                 (1190, 5), (1190, 4100)])
def test_quantize_rows(M, K, dtype):
    x = (torch.randn(M, K, generator=gen(M * K), device="cuda") * 3).to(dtype)
    q, s = w8a8.quantize_i8(x)
    rq, rs = quantized(x)
    assert torch.equal(s, rs) and torch.equal(q, rq)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_ties_go_to_even(dtype):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 0.25, 0.75]], device="cuda").to(dtype)
    q, s = w8a8.quantize_i8(x)
    if dtype != torch.bfloat16:
        assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 126, 0, 1]
    assert torch.equal(q, quantized(x)[0]) and s.item() == 1.0


def test_quantize_values_at_the_ends_of_the_range():
    n = 70
    x = torch.randn(9, n, generator=gen(1), device="cuda")
    x[1] = 0
    x[2] *= 1e-42          # subnormal values, and a scale that would be one
    x[3] *= 1e-26
    x[4] *= 3e37
    x[5, 3] = float("inf")
    x[6, 69] = float("nan")
    x[7, 0], x[7, 1] = float("-inf"), float("nan")
    x[8] = 2.0 ** -149
    q, s = w8a8.quantize_i8(x)
    rq, rs = quantized(x)
    assert same(s, rs) and torch.equal(q, rq)
    assert s[1] == 0 and torch.isnan(s[[5, 6, 7]]).all() and (q[[1, 5, 6, 7]] == 0).all()
    w, sw = i8(gen(2), 3, n), scales(gen(3), 3)
    y = w8a8.matmul_w8a8(q, s, w, sw)
    fine = [0, 1, 2, 3, 4, 8]
    ref, bound = product(q[fine], s[fine], w, sw, None, abi.ACT_NONE, torch.float32)
    top = torch.finfo(torch.float32).max     # (row 4 has products near it: 127 * 127 * 70 * 1e36 * 0.01 = 1e40 at most)
    assert torch.isnan(y[[5, 6, 7]]).all() and (y[1] == 0).all()
    assert torch.equal(torch.isfinite(y[fine]), ref.abs() < top)
    check(torch.where(ref.abs() < top, y[fine], 0), torch.where(ref.abs() < top, ref, 0), bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_rows_of_a_wider_matrix_and_gathered(dtype):
    wide = torch.randn(6, 1000, generator=gen(5), device="cuda").to(dtype)
    for lo, hi in [(0, 500), (1, 500), (3, 77), (8, 8 + 512)]:      # (odd starts: rows off the 16-byte boundaries)
        x = wide[:, lo:hi]
        rq, rs = quantized(x)
        rows = torch.tensor([11, 0, 0, 5, 12, -1, 2 ** 31 - 1, -2 ** 31, 1, 10], dtype=torch.int32, device="cuda")
        q, s = w8a8.quantize_i8(x, rows, 2)
        for i, r in enumerate(rows.tolist()):
            if 0 <= r // 2 < 6 and r >= 0:
                assert torch.equal(q[i], rq[r // 2]) and s[i] == rs[r // 2]
            else:
                assert (q[i] == 0).all() and s[i] == 0
        q, s = w8a8.quantize_i8(x[::2])
        assert torch.equal(q, rq[::2]) and torch.equal(s, rs[::2])


# ---- dense ----
SHAPES = [(1, 1, 1), (1, 2048, 4096), (8, 2688, 96), (5, 8192, 70), (5, 8193, 70), (8, 65, 33), (4, 4100, 515), (9, 2048, 4096), (2, 128, 128), (3, 129, 5), (7, 2688, 3712), (16, 512, 100), (17, 100, 130), (33, 2005, 257), (61, 4096, 2048), (64, 64, 64),
          (65, 300, 700), (129, 1000, 513), (300, 640, 1000), (777, 2005, 1031), (1500, 384, 2500), (5000, 130, 260), (4000, 2048, 2048), (2300, 1000, 1024), (1111, 640, 4099), (20000, 64, 320), (3000, 512, 2048), (2500, 400, 1040), (40000, 128, 512)]


@pytest.mark.parametrize("act", [abi.ACT_NONE, abi.ACT_SWIGLU, abi.ACT_RELU2])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_matmul(M, K, N, act):
    g = gen(M + K + N)
    R = 2 * N if act == abi.ACT_SWIGLU else N
    q, w, sx, sw = i8(g, M, K), i8(g, R, K), scales(g, M) / max(1, K) ** 0.5, scales(g, R)
    for j, dtype in enumerate(TYPES):
        bias = torch.randn(R, generator=g, device="cuda") if j else None
        y = w8a8.matmul_w8a8(q, sx, w, sw, bias=bias, act=act, out_dtype=dtype)
        check(y, *product(q, sx, w, sw, bias, act, dtype))


def test_integer_sums_are_exact():
    """Unit scales: whole numbers, rounded once to f32; the largest sums that 32 bits hold among them."""
    for M, K, N, lo, hi in [(5, 131071, 40, -128, -128), (3, 131071, 130, 127, 127), (130, 131071, 129, -128, 127), (300, 1024, 300, -128, 127)]:
        g = gen(K + N)
        q, w = i8(g, M, K, lo=lo, hi=hi), i8(g, N, K, lo=lo, hi=hi)
        y = w8a8.matmul_w8a8(q, torch.ones(M, device="cuda"), w, torch.ones(N, device="cuda"))
        assert torch.equal(y, (q.double() @ w.double().T).float())


def test_matrices_inside_wider_ones():
    g = gen(9)
    W, X = i8(g, 600, 1024), i8(g, 200, 2048)
    w, q = W[3:503, 16:816], X[7:140, 32:832]
    sw, sx = scales(g, 500), scales(g, 133)
    big = torch.full((135, 520), 7.0, dtype=torch.bfloat16, device="cuda")
    out = big[1:134, 9:509]
    assert w8a8.matmul_w8a8(q, sx, w, sw, out=out) is out
    check(out, *product(q, sx, w, sw, None, abi.ACT_NONE, torch.bfloat16))
    keep = torch.ones_like(big, dtype=torch.bool)
    keep[1:134, 9:509] = False
    assert (big[keep] == 7).all()
    check(w8a8.matmul_w8a8(q[::3], sx[::3].contiguous(), w[::2], sw[::2].contiguous()), *product(q[::3], sx[::3], w[::2], sw[::2], None, abi.ACT_NONE, torch.float32))


def test_scales_of_zero_infinity_and_nan():
    g = gen(10)
    q, w = i8(g, 20, 64), i8(g, 30, 64)
    sx, sw = scales(g, 20), scales(g, 30)
    sx[3], sx[4], sw[5] = float("nan"), 0.0, float("nan")
    y = w8a8.matmul_w8a8(q, sx, w, sw)
    assert torch.isnan(y[3]).all() and torch.isnan(y[:, 5]).all()
    ok = torch.ones_like(y, dtype=torch.bool)
    ok[3], ok[:, 5] = False, False
    assert torch.isfinite(y[ok]).all() and (y[4][ok[4]] == 0).all()
    for act in (abi.ACT_RELU2, abi.ACT_SWIGLU):
        assert torch.isnan(w8a8.matmul_w8a8(q, sx, w, sw, act=act)[3]).all()
    assert torch.isinf(w8a8.matmul_w8a8(torch.full((1, 64), 127, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"), i8(g, 1, 64, lo=127), torch.ones(1, device="cuda"),
                                        out_dtype=torch.float16)).all()


# ---- grouped ----
def groups(counts, first=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]) + first, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("act", [abi.ACT_NONE, abi.ACT_SWIGLU, abi.ACT_RELU2])
@pytest.mark.parametrize("counts,K,N", [([1], 64, 64), ([0, 0, 3, 0], 100, 33), ([1, 1, 1, 1, 1, 1, 1, 1], 2048, 512), ([0] * 30 + [19, 1, 0, 8, 9], 2048, 100), ([2, 0, 0, 1], 9000, 50), ([16, 17, 0, 15, 33], 257, 130), ([300, 0, 1, 129, 64], 512, 260),
                                        ([0] * 100 + [5] + [0] * 900 + [7], 128, 40), ([2000, 3, 700], 384, 200), ([700, 0, 300, 1, 128, 129, 255, 256, 257], 512, 1024), ([3000], 100, 2000), ([40] * 64, 640, 192)])
def test_grouped(counts, K, N, act):
    g = gen(K + N + len(counts))
    M, E, R = sum(counts), len(counts), 2 * N if act == abi.ACT_SWIGLU else N
    q, w, sx, sw = i8(g, M, K), i8(g, E, R, K), scales(g, M) / K ** 0.5, scales(g, E, R)
    bias = torch.randn(E, R, generator=g, device="cuda")
    off = groups(counts)
    for dtype in TYPES:
        y = w8a8.matmul_w8a8_grouped(q, sx, w, sw, off, bias=bias, act=act, out_dtype=dtype)
        for e in range(E):
            a, b = int(off[e]), int(off[e + 1])
            if b > a:
                check(y[a:b], *product(q[a:b], sx[a:b], w[e], sw[e], bias[e], act, dtype))


@pytest.mark.parametrize("M,counts,first", [(40, [3, 0, 9, 4], 5), (500, [200, 0, 31, 170], 20), (12, [0, 0, 0, 0], 0), (300, [100, 100, 400, 1], 50)])
def test_grouped_rows_outside_every_group_stay(M, counts, first):
    g = gen(M)
    K, N = 192, 150
    q, w, sx, sw = i8(g, M, K), i8(g, 4, N, K), scales(g, M), scales(g, 4, N)
    off = groups(counts, first)          # (in the last case the ends lie behind the last row)
    out = torch.full((M, N), 7.0, device="cuda")
    w8a8.matmul_w8a8_grouped(q, sx, w, sw, off, out=out)
    seen = torch.zeros(M, dtype=torch.bool, device="cuda")
    for e in range(4):
        a, b = min(int(off[e]), M), min(int(off[e + 1]), M)
        if b > a:
            check(out[a:b], *product(q[a:b], sx[a:b], w[e], sw[e], None, abi.ACT_NONE, torch.float32))
            seen[a:b] = True
    assert (out[~seen] == 7).all()


@pytest.mark.parametrize("M", [9, 400])
def test_grouped_rows_to_other_places(M):
    g = gen(M)
    K, N, E = 128, 96, 5
    q, w, sx, sw = i8(g, M, K), i8(g, E, N, K), scales(g, M), scales(g, E, N)
    off = torch.tensor([0, M // 3, M // 3, M // 2, M - 1, M], dtype=torch.int32, device="cuda")
    y = w8a8.matmul_w8a8_grouped(q, sx, w, sw, off)
    to = torch.randperm(2 * M, generator=g, device="cuda")[:M].to(torch.int32)
    to[1], to[2] = -1, 2 * M        # nowhere
    out = torch.full((2 * M, N), 7.0, device="cuda")
    w8a8.matmul_w8a8_grouped(q, sx, w, sw, off, out_rows=to, out=out)
    want = torch.full_like(out, 7.0)
    kept = [i for i in range(M) if i not in (1, 2)]
    want[to[kept].long()] = y[kept]
    assert torch.equal(out, want)


def test_offsets_that_fall_are_empty_groups():
    g = gen(3)
    q, w, sx, sw = i8(g, 30, 64), i8(g, 4, 48, 64), scales(g, 30), scales(g, 4, 48)
    off = torch.tensor([-5, 10, 4, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")   # 0..10, none, 4..30, none
    out = torch.zeros(30, 48, device="cuda")
    w8a8.matmul_w8a8_grouped(q, sx, w, sw, off, out=out)
    check(out[10:], *product(q[10:], sx[10:], w[2], sw[2], None, abi.ACT_NONE, torch.float32))
    check(out[:4], *product(q[:4], sx[:4], w[0], sw[0], None, abi.ACT_NONE, torch.float32))


def test_stack_inside_a_wider_one():
    g = gen(4)
    W = i8(g, 9, 80, 256)
    w = W[1::2, 5:69, 16:216]
    q, sx, sw = i8(g, 50, 200), scales(g, 50), scales(g, 4, 64)
    off = groups([20, 0, 13, 17])
    y = w8a8.matmul_w8a8_grouped(q, sx, w, sw, off)
    for e in range(4):
        a, b = int(off[e]), int(off[e + 1])
        if b > a:
            check(y[a:b], *product(q[a:b], sx[a:b], w[e], sw[e], None, abi.ACT_NONE, torch.float32))


# ---- the chains ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N,act", [(1, 2048, 4096, abi.ACT_NONE), (5, 77, 130, abi.ACT_SWIGLU), (8, 3000, 515, abi.ACT_RELU2), (2, 2688, 33, abi.ACT_NONE), (7, 500, 1000, abi.ACT_SWIGLU), (6, 8192, 4100, abi.ACT_NONE), (8, 64, 20000, abi.ACT_NONE), (8, 8190, 64, abi.ACT_NONE), (3, 8192, 130, abi.ACT_SWIGLU), (1, 20000, 64, abi.ACT_NONE), (200, 1000, 640, abi.ACT_RELU2), (1025, 512, 300, abi.ACT_NONE)])
def test_linear_is_its_two_steps(M, K, N, act, dtype):
    g = gen(M + K)
    R = 2 * N if act == abi.ACT_SWIGLU else N
    x, w, sw, bias = torch.randn(M, K, generator=g, device="cuda").to(dtype), i8(g, R, K), scales(g, R), torch.randn(R, generator=g, device="cuda")
    y = w8a8.linear_w8a8(x, w, sw, bias=bias, act=act)
    assert y.dtype == dtype
    q, s = quantized(x)
    check(y, *product(q, s, w, sw, bias, act, dtype))
    q, s = w8a8.quantize_i8(x)
    assert torch.equal(y, w8a8.matmul_w8a8(q, s, w, sw, bias=bias, act=act, out_dtype=dtype))


@pytest.mark.parametrize("cfg,T", [(configs.QWEN_Q4_0, 1), (configs.QWEN_Q4_0, 9), (configs.QWEN_Q4_0_ZIPF, 200), (configs.NEMOTRON_Q4_0, 3), (configs.NEMOTRON_Q4_0, 150)])
def test_experts_behind_the_router(cfg, T):
    """Route with the package's router, then the layer's routed experts in W8A8, and the combine; against the formulas in 64 bits."""
    cfg = configs.scaled(cfg, H=512, E=32, F=192, F_s=0)
    layer = MoeWeightsTiled(configs.make_layer(cfg, device="cuda"))
    sc = MoeScratch(layer, T)
    x = configs.make_input(cfg, T, device="cuda")
    route_only(layer, sc, x)
    g, H, F, E, k = gen(T), cfg.H, cfg.F, cfg.E, cfg.top_k
    R = 2 * F if cfg.act == abi.ACT_SWIGLU else F
    w_up, s_up, w_dn, s_dn = i8(g, E, R, H), scales(g, E, R) * 0.05, i8(g, E, H, F), scales(g, E, H) * 0.05
    perm, off, ids = sc.perm(T), sc.offsets(), sc.topk_indices(T)
    y = w8a8.experts_w8a8(x, perm, off, k, w_up, s_up, w_dn, s_dn, act=cfg.act)
    assert y.shape == (T * k, H) and y.dtype == torch.float32
    # the four steps one by one
    q, s = w8a8.quantize_i8(x, perm, k)
    h = w8a8.matmul_w8a8_grouped(q, s, w_up, s_up, off, act=cfg.act)
    hq, hs = w8a8.quantize_i8(h)
    steps = w8a8.matmul_w8a8_grouped(hq, hs, w_dn, s_dn, off, out_rows=perm, out=torch.empty_like(y))
    assert torch.equal(y, steps)
    # ... and against 64 bits: the activations' bound, and behind it the second product of the rows as they were rounded
    xq, xs = quantized(x)
    for e in range(E):
        a, b = int(off[e]), int(off[e + 1])
        if b > a:
            pairs = perm[a:b].long()
            assert (ids.reshape(-1)[pairs] == e).all()
            t = pairs // k
            check(h[a:b], *product(xq[t], xs[t], w_up[e], s_up[e], None, cfg.act, torch.float32))
            rq, rs = quantized(h[a:b])
            check(y[pairs], *product(rq, rs, w_dn[e], s_dn[e], None, abi.ACT_NONE, torch.float32))
    combined = (y.reshape(T, k, H) * sc.topk_weights(T)[:, :, None]).sum(1)
    assert torch.isfinite(combined).all() and sc.status() == 0


# ---- streams, graphs, nothing to do ----
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_of_rows_at_the_ends_of_the_range(dtype):
    """What a batch of a few tokens quantises itself: the same rows, the same bits."""
    g = gen(21)
    x = torch.randn(8, 333, generator=g, device="cuda")
    x[1], x[2], x[3, 5], x[4, 332] = 0, x[2] * 1e-30, float("inf"), float("nan")
    wide = torch.zeros(8, 340, device="cuda").to(dtype)
    wide[:, 3:336] = x.to(dtype)
    w, sw = i8(g, 50, 333), scales(g, 50)
    for rows in (x.to(dtype), wide[:, 3:336]):
        q, s = w8a8.quantize_i8(rows)
        rq, rs = quantized(rows)
        assert torch.equal(q, rq) and same(s, rs)
        y = w8a8.linear_w8a8(rows, w, sw, out_dtype=torch.float32)
        assert same(y, w8a8.matmul_w8a8(q, s, w, sw)) and torch.isnan(y[3:5]).all() and (y[1] == 0).all()
        ok = [0, 1, 2, 5, 6, 7]
        check(y[ok], *product(q[ok], s[ok], w, sw, None, abi.ACT_NONE, torch.float32))


def test_experts_with_ids_outside_the_rows():
    """A permutation entry that is no pair: a row of zeros goes in, and nothing comes out for it."""
    g = gen(22)
    for T, E, H in ((6, 32, 160), (200, 4, 160), (1100, 5, 2005)):
        F, k = 64, 2
        x = torch.randn(T, H, generator=g, device="cuda")
        perm = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32)
        off = groups([T * k // E] * (E - 1) + [T * k - (E - 1) * (T * k // E)])
        wu, su, wd, sd = i8(g, E, 2 * F, H), scales(g, E, 2 * F) * 0.05, i8(g, E, H, F), scales(g, E, H) * 0.05
        want = w8a8.experts_w8a8(x, perm, off, k, wu, su, wd, sd)
        bad = perm.clone()
        bad[0], bad[3], bad[5] = -1, T * k, -2 ** 31
        out = torch.full_like(want, 7.0)
        w8a8.experts_w8a8(x, bad, off, k, wu, su, wd, sd, out=out)
        lost = perm[[0, 3, 5]].long()
        keep = torch.ones(T * k, dtype=torch.bool, device="cuda")
        keep[lost] = False
        assert torch.equal(out[keep], want[keep]) and (out[lost] == 7).all()
        if T > 1000:     # rows quantised once and copied, against a gather of the rows themselves
            q, s = w8a8.quantize_i8(x, perm, k)
            hq, hs = w8a8.quantize_i8(w8a8.matmul_w8a8_grouped(q, s, wu, su, off, act=abi.ACT_SWIGLU))
            assert torch.equal(want, w8a8.matmul_w8a8_grouped(hq, hs, wd, sd, off, out_rows=perm, out=torch.empty_like(want)))
            twice = perm.clone()
            twice[7] = twice[8]                       # one pair in two places of the same group: its row is written twice, alike
            twice[7:9] = twice[8]
            again = w8a8.experts_w8a8(x, twice, off, k, wu, su, wd, sd, out=torch.full_like(want, 7.0))
            assert torch.equal(again[twice.long()], want[twice.long()]) and (again[perm[7].long()] == 7).all()


def test_capture_and_replay_with_new_inputs():
    g = gen(6)
    x, w, sw = torch.randn(12, 500, generator=g, device="cuda"), i8(g, 300, 500), scales(g, 300)
    out = torch.empty(12, 300, device="cuda")
    perm, off = torch.randperm(24, generator=g, device="cuda").to(torch.int32), groups([10, 0, 14])
    wu, su, wd, sd = i8(g, 3, 128, 500), scales(g, 3, 128) * 0.01, i8(g, 3, 500, 64), scales(g, 3, 500) * 0.01
    rows = torch.empty(24, 500, device="cuda")
    run = lambda: (w8a8.linear_w8a8(x, w, sw, out=out), w8a8.experts_w8a8(x, perm, off, 2, wu, su, wd, sd, out=rows))   # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        run()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            run()
        with torch.cuda.graph(other, stream=stream):
            run()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in range(4):
        x.copy_(torch.randn(12, 500, generator=gen(seed), device="cuda"))
        perm.copy_(torch.randperm(24, generator=gen(seed), device="cuda").to(torch.int32))
        off.copy_(groups([seed, 20 - 5 * seed, 4 + 4 * seed]))
        (graph if seed % 2 else other).replay()
        got = out.clone(), rows.clone()
        run()
        assert torch.equal(got[0], out) and torch.equal(got[1], rows)


def test_weights_written_by_the_kernel_in_front():
    """Weights and scales that the previous launches of the stream make."""
    g = gen(7)
    x = torch.randn(4, 1024, generator=g, device="cuda")
    for i in range(20):
        wf = torch.randn(2048, 1024, generator=g, device="cuda")
        wq, ws = w8a8.quantize_i8(wf)
        y = w8a8.linear_w8a8(x, wq, ws)
        q, s = w8a8.quantize_i8(x)
        wq2, ws2 = w8a8.quantize_i8(wf)
        assert torch.equal(y, w8a8.matmul_w8a8(q, s, wq2, ws2))
        check(y, *product(*quantized(x), *quantized(wf), None, abi.ACT_NONE, torch.float32))


def test_two_streams_at_once():
    g = gen(8)
    x, w, sw = torch.randn(40, 2048, generator=g, device="cuda"), i8(g, 512, 2048), scales(g, 512)
    x2, w2, sw2 = torch.randn(700, 1024, generator=g, device="cuda"), i8(g, 3000, 1024), scales(g, 3000)
    want, want2 = w8a8.linear_w8a8(x, w, sw), w8a8.linear_w8a8(x2, w2, sw2)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got, got2 = [], []
    for _ in range(20):
        with torch.cuda.stream(a):
            got.append(w8a8.linear_w8a8(x, w, sw))
        with torch.cuda.stream(b):
            got2.append(w8a8.linear_w8a8(x2, w2, sw2))
    torch.cuda.synchronize()
    assert all(torch.equal(v, want) for v in got) and all(torch.equal(v, want2) for v in got2)


@pytest.mark.parametrize("N", [32768, 32749])
def test_more_than_2_31_results(N):
    """Offsets beyond 32 bits, in the rows that are quantised and in the results (aligned and not)."""
    M, K = (1 << 31) // 32749 + 300, 64
    g = gen(30)
    x, w, sw = torch.randn(M, K, generator=g, device="cuda"), i8(g, N, K), scales(g, N)
    y = w8a8.linear_w8a8(x, w, sw, out_dtype=torch.bfloat16)
    rows = torch.cat([torch.arange(3, device="cuda"), torch.arange(M - 290, M, device="cuda")])
    q, s = quantized(x[rows])
    check(y[rows], *product(q, s, w, sw, None, abi.ACT_NONE, torch.bfloat16))
    qy, sy = w8a8.quantize_i8(y)
    rq, rs = quantized(y[rows])
    assert torch.equal(qy[rows], rq) and torch.equal(sy[rows], rs)


def test_no_rows():
    g = gen(1)
    x, w, sw = torch.empty(0, 64, device="cuda"), i8(g, 40, 64), scales(g, 40)
    assert w8a8.linear_w8a8(x, w, sw).shape == (0, 40)
    q, s = w8a8.quantize_i8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    assert w8a8.matmul_w8a8(q, s, w, sw).shape == (0, 40)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert w8a8.experts_w8a8(x, none, torch.zeros(3, dtype=torch.int32, device="cuda"), 2, i8(g, 2, 64, 64), scales(g, 2, 64), i8(g, 2, 64, 32), scales(g, 2, 64)).shape == (0, 64)
    assert w8a8.quantize_i8(x, torch.tensor([0], dtype=torch.int32, device="cuda"))[1].item() == 0   # (an index into no rows)


def test_status_word_stays_zero():
    g = gen(2)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    w8a8.linear_w8a8(torch.randn(300, 700, generator=g, device="cuda"), i8(g, 400, 700), scales(g, 400), status=status)
    assert status.item() == 0


# ---- refusals ----
def test_arguments_that_are_refused():
    g = gen(1)
    x, w, sw = torch.randn(4, 64, generator=g, device="cuda"), i8(g, 32, 64), scales(g, 32)
    q, s = w8a8.quantize_i8(x)
    bad = [lambda: w8a8.quantize_i8(x.double()), lambda: w8a8.quantize_i8(x.cpu()), lambda: w8a8.quantize_i8(x.T), lambda: w8a8.quantize_i8(x[0]),
           lambda: w8a8.quantize_i8(x, torch.zeros(3, dtype=torch.int64, device="cuda")), lambda: w8a8.quantize_i8(x[:1].expand(4, 64)),
           lambda: w8a8.linear_w8a8(x, w[:, :60], sw), lambda: w8a8.linear_w8a8(x, w.float(), sw), lambda: w8a8.linear_w8a8(x, w, sw[:31]),
           lambda: w8a8.linear_w8a8(x, w, sw.half()), lambda: w8a8.linear_w8a8(x, w, sw, bias=torch.zeros(31, device="cuda")),
           lambda: w8a8.linear_w8a8(x, w, sw, out_dtype=torch.int32), lambda: w8a8.linear_w8a8(x, w, sw, out=torch.empty(4, 31, device="cuda")),
           lambda: w8a8.linear_w8a8(x, w[:31], sw[:31], act=abi.ACT_SWIGLU), lambda: w8a8.linear_w8a8(x, w.cpu(), sw),
           lambda: w8a8.linear_w8a8(x, w, sw, out=torch.empty(32, 4, device="cuda").T), lambda: w8a8.linear_w8a8(x, w, sw, out=torch.empty(1, 32, device="cuda").expand(4, 32)),
           lambda: w8a8.matmul_w8a8(q[:, 1:61], s, w[:, :60], sw), lambda: w8a8.matmul_w8a8(torch.zeros(4, 60, dtype=torch.int8, device="cuda"), s, w[:, :60], sw),
           lambda: w8a8.matmul_w8a8(q, s[:3], w, sw),
           lambda: w8a8.matmul_w8a8_grouped(q, s, w[None], sw[None], torch.zeros(3, dtype=torch.int32, device="cuda")),
           lambda: w8a8.matmul_w8a8_grouped(q, s, w[None], sw, torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: w8a8.experts_w8a8(x, torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), 2, w[None], sw[None], i8(g, 1, 64, 16), scales(g, 1, 64), act=abi.ACT_NONE)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError, match="bad dimension"):
        w8a8.quantize_i8(torch.zeros(1, 131072, device="cuda"))
    with pytest.raises(RuntimeError, match="bad dimension"):
        w8a8.linear_w8a8(x, w, sw, act=7)
    with pytest.raises(RuntimeError, match="bad dimension"):
        w8a8.quantize_i8(x, torch.zeros(3, dtype=torch.int32, device="cuda"), 0)
