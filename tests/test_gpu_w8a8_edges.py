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
