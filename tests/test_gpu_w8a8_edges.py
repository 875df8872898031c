"""W8A8 calls at the edges of what their documentation allows."""
import pytest
import torch

from chimere_b200 import abi, w8a8

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i8(g, *shape):
    return w8a8.padded_i8(torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8))


def scales(g, *shape):
    return torch.rand(shape, generator=g, device="cuda") * 0.01 + 1e-4


def on_a_busy_gpu(fn):
    """fn on a stream of its own, while a large product holds the multiprocessors and starts its blocks late."""
    a = torch.ones(8192, 4096, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    a @ a.T
    with torch.cuda.stream(side):
        fn()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 4, 8, 9, 70])
def test_linear_over_its_own_rows(M, dtype):
    for K in (512, 2048):
        g = gen(M + K)
        w, sw = i8(g, K, K), scales(g, K) * 0.1
        for _ in range(3):
            x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
            want = w8a8.linear_w8a8(x, w, sw)
            on_a_busy_gpu(lambda: w8a8.linear_w8a8(x, w, sw, out=x))
            assert torch.equal(x, want)
            # a row further down, and beside the rows
            buf = torch.zeros(M + 1, K, device="cuda", dtype=dtype)
            buf[:M] = torch.randn(M, K, generator=g, device="cuda")
            want = w8a8.linear_w8a8(buf[:M], w, sw)
            on_a_busy_gpu(lambda: w8a8.linear_w8a8(buf[:M], w, sw, out=buf[1:]))
            assert torch.equal(buf[1:], want)
            wide = torch.zeros(M, 2 * K, device="cuda", dtype=dtype)
            wide[:, :K] = torch.randn(M, K, generator=g, device="cuda")
            want = w8a8.linear_w8a8(wide[:, :K], w, sw)
            on_a_busy_gpu(lambda: w8a8.linear_w8a8(wide[:, :K], w, sw, out=wide[:, K:]))
            assert torch.equal(wide[:, K:], want)


@pytest.mark.parametrize("T", [1, 8, 200, 5000])
def test_experts_over_their_own_rows(T):
    H, F, E = 1024, 256, 4
    g = gen(T)
    wu, su, wd, sd = i8(g, E, 2 * F, H), scales(g, E, 2 * F) * 0.01, i8(g, E, H, F), scales(g, E, H) * 0.01
    ids = torch.randint(0, E, (T,), generator=g, device="cuda")
    perm = torch.sort(ids, stable=True).indices.to(torch.int32)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(ids, minlength=E).cumsum(0)
    for _ in range(3):
        x = torch.randn(T, H, generator=g, device="cuda")
        want = w8a8.experts_w8a8(x, perm, off, 1, wu, su, wd, sd)
        on_a_busy_gpu(lambda: w8a8.experts_w8a8(x, perm, off, 1, wu, su, wd, sd, out=x))
        assert torch.equal(x, want)


def test_sizes_beyond_32_bits_are_refused():
    """What the C entry would see cut to 32 bits."""
    g = gen(3)
    x, w, sw = torch.randn(4, 64, generator=g, device="cuda"), i8(g, 32, 64), scales(g, 32)
    q, s = w8a8.quantize_i8(x)
    rows, off = torch.arange(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    wide = torch.ones(1, 2 ** 32 + 64, dtype=torch.float16, device="cuda")
    calls = [lambda: w8a8.quantize_i8(x, rows, 2 ** 32 + 1), lambda: w8a8.quantize_i8(wide), lambda: w8a8.quantize_i8(wide, rows[:1], 1),
             lambda: w8a8.linear_w8a8(x, w, sw, act=2 ** 32 + abi.ACT_RELU2), lambda: w8a8.matmul_w8a8(q, s, w, sw, act=2 ** 32 + abi.ACT_RELU2),
             lambda: w8a8.matmul_w8a8_grouped(q, s, w[None], sw[None], off, act=2 ** 32 + abi.ACT_RELU2),
             lambda: w8a8.experts_w8a8(x, rows, off, 2 ** 32 + 1, w[None], sw[None], i8(g, 1, 64, 32), scales(g, 1, 64), act=abi.ACT_RELU2)]
    for i, f in enumerate(calls):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")


# ---- weights and rows that the launches in front make ----
def weights_of(wf):
    return w8a8.quantize_i8(wf)


@pytest.mark.parametrize("M,K,N", [(7, 2688, 1000), (9, 512, 512), (61, 4096, 2048), (300, 1000, 2000), (2000, 512, 4096)])
def test_weights_made_by_the_launch_in_front(M, K, N):
    """Products in a launch of their own fetch weights and scales before the rows are there: what made the weights must be complete by then all the same."""
    g = gen(M + K)
    x = torch.randn(M, K, generator=g, device="cuda")
    q, s = w8a8.quantize_i8(x)
    for _ in range(10):
        wf = torch.randn(N, K, generator=g, device="cuda")
        y = w8a8.linear_w8a8(x, *weights_of(wf))
        wq, ws = weights_of(wf)
        torch.cuda.synchronize()
        assert torch.equal(y, w8a8.matmul_w8a8(q, s, wq, ws))


@pytest.mark.parametrize("T,E,k,H,F", [(1, 8, 2, 512, 256), (16, 32, 4, 512, 256), (200, 8, 2, 512, 320), (3000, 6, 3, 1024, 512)])
def test_experts_whose_weights_and_rows_the_launches_in_front_make(T, E, k, H, F):
    g = gen(T)
    ids = torch.randint(0, E, (T * k,), generator=g, device="cuda")
    perm = torch.sort(ids, stable=True).indices.to(torch.int32)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(ids, minlength=E).cumsum(0)

    def stack(rows, K):
        q, s = w8a8.quantize_i8(torch.randn(E * rows, K, generator=g, device="cuda"))
        return q.view(E, rows, K), s.view(E, rows) * 0.05

    for _ in range(10):
        wu, su = stack(2 * F, H)
        wd, sd = stack(H, F)
        x = torch.randn(T, H, generator=g, device="cuda")
        y = w8a8.experts_w8a8(x, perm, off, k, wu, su, wd, sd)
        torch.cuda.synchronize()
        q, s = w8a8.quantize_i8(x, perm, k)
        torch.cuda.synchronize()
        h = w8a8.matmul_w8a8_grouped(q, s, wu, su, off, act=abi.ACT_SWIGLU)
        torch.cuda.synchronize()
        hq, hs = w8a8.quantize_i8(h)
        torch.cuda.synchronize()
        assert torch.equal(y, w8a8.matmul_w8a8_grouped(hq, hs, wd, sd, off, out_rows=perm, out=torch.empty_like(y)))


# ---- the order of the roundings ----
@pytest.mark.parametrize("M,K,N", [(1, 2048, 512), (4, 4100, 515), (8, 512, 96), (17, 100, 130), (61, 4096, 2048), (300, 640, 1000), (2300, 1000, 1024)])
@pytest.mark.parametrize("act", [abi.ACT_NONE, abi.ACT_RELU2])
def test_products_round_in_the_stated_order(M, K, N, act):
    """The sum to f32, times the channel's scale, times the row's: one rounding each, the same bits in every kernel."""
    g = gen(M + K + N)
    q, w, sx, sw = i8(g, M, K), i8(g, N, K), scales(g, M), scales(g, N)
    want = (q.double() @ w.double().T).float() * sw * sx[:, None]
    if act == abi.ACT_RELU2:
        want = want.clamp_min(0).square()
    for dtype in TYPES:
        assert torch.equal(w8a8.matmul_w8a8(q, sx, w, sw, act=act, out_dtype=dtype), want.to(dtype))
    off = torch.tensor([0, M // 3, M // 3, M], dtype=torch.int32, device="cuda")
    stack, scale = w8a8.padded_i8(torch.stack([w] * 3)), torch.stack([sw] * 3).contiguous()
    assert torch.equal(w8a8.matmul_w8a8_grouped(q, sx, stack, scale, off, act=act), want)


def test_relu2_experts_are_the_formula_bit_for_bit():
    """Activations next to a half step go to one whole number or its neighbour by their last bit, so the order of the two scales decides there: channel first."""
    T, E, k, H, F = 100, 8, 3, 1344, 480
    g = gen(17)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    wu, su, wd, sd = i8(g, E, F, H), scales(g, E, F), i8(g, E, H, F), scales(g, E, H)
    ids = torch.randint(0, E, (T * k,), generator=g, device="cuda")
    perm = torch.sort(ids, stable=True).indices
    counts = torch.bincount(ids, minlength=E).tolist()
    off = torch.tensor([sum(counts[:e]) for e in range(E + 1)], dtype=torch.int32, device="cuda")
    y = w8a8.experts_w8a8(x, perm.to(torch.int32), off, k, wu, su, wd, sd, act=abi.ACT_RELU2)

    def rows(v):
        v = v.double()
        s = (v.abs().amax(1, keepdim=True) / 127).float().double()
        return (v / s).float().double().round(), s.float()

    for e in range(E):
        pairs = perm[off[e]:off[e + 1]]
        q, s = rows(x[pairs // k].float())
        h = ((q @ wu[e].double().T).float() * su[e] * s).clamp_min(0).square()
        q, s = rows(h)
        assert torch.equal(y[pairs], ((q @ wd[e].double().T).float() * sd[e] * s).to(torch.bfloat16))
