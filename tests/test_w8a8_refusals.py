"""What the W8A8 entries refuse before anything is launched (no GPU needed)."""
import pytest

from chimere_b200 import abi, build

A = 4096   # a non-null, aligned placeholder: never dereferenced on the host


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def quantize(lib, x=A, type=abi.TYPE_F32, ldx=64, x_rows=4, rows=None, div=1, M=4, K=64, q=A, ldq=64, scale=A):
    return lib.chimere_b200_quantize_i8(x, type, ldx, x_rows, rows, div, M, K, q, ldq, scale, None)


def matmul(lib, x=A, ldx=64, sx=A, w=A, ldw=64, sw=A, bias=None, M=4, N=32, K=64, act=abi.ACT_NONE, y=A, y_type=abi.TYPE_F32, ldy=32):
    return lib.chimere_b200_matmul_w8a8(x, ldx, sx, w, ldw, sw, bias, M, N, K, act, y, y_type, ldy, None, None)


def grouped(lib, x=A, w=A, ldw=64, stride=2048, offsets=A, E=3, M=4, N=32, K=64, act=abi.ACT_NONE, y_rows=4, out_rows=None, ldy=32):
    return lib.chimere_b200_matmul_w8a8_grouped(x, 64, A, w, ldw, stride, A, None, offsets, E, M, N, K, act, A, abi.TYPE_F32, ldy, y_rows, out_rows, None, None)


def linear(lib, x=A, ldx=64, M=40, N=32, K=64, ws=A, nbytes=1 << 20, w=A):
    return lib.chimere_b200_linear_w8a8(x, abi.TYPE_BF16, ldx, w, 64, A, None, M, N, K, abi.ACT_NONE, A, abi.TYPE_BF16, N, ws, nbytes, None, None)


def experts(lib, T=4, k=2, perm=A, offsets=A, E=3, H=64, F=32, act=abi.ACT_SWIGLU, ws=A, nbytes=1 << 20, stride_up=4096):
    return lib.chimere_b200_experts_w8a8(A, abi.TYPE_F32, H, T, perm, offsets, k, E, A, 64, stride_up, A, A, 32, 2048, A, H, F, act, A, abi.TYPE_F32, H, ws, nbytes, None, None)


@pytest.mark.parametrize("want,kw", [(-2, dict(M=-1)), (-2, dict(K=0)), (-2, dict(K=131072, ldx=131072, ldq=131072)), (-2, dict(ldx=63)), (-2, dict(ldq=63)), (-2, dict(ldq=72)), (-2, dict(x_rows=3)),
                                     (-2, dict(div=0, rows=A)), (-2, dict(x_rows=-1)), (-3, dict(type=2)), (-1, dict(x=None)), (-1, dict(q=None)), (-1, dict(scale=None)),
                                     (-5, dict(x=A + 2)), (-5, dict(type=abi.TYPE_F16, x=A + 1)), (-5, dict(q=A + 8)), (-5, dict(rows=A + 2)), (0, dict(M=0, x=None, q=None, scale=None))])
def test_quantize(lib, want, kw):
    assert quantize(lib, **kw) == want


@pytest.mark.parametrize("want,kw", [(-2, dict(M=-1)), (-2, dict(N=0)), (-2, dict(K=0)), (-2, dict(K=131072, ldx=131072, ldw=131072)), (-2, dict(ldx=48)), (-2, dict(ldx=72)), (-2, dict(ldw=48)),
                                     (-2, dict(ldw=72)), (-2, dict(ldy=31)), (-2, dict(act=2)), (-2, dict(act=abi.ACT_SWIGLU, N=1 << 30, ldy=1 << 30)), (-3, dict(y_type=2)), (-1, dict(x=None)),
                                     (-1, dict(sx=None)), (-1, dict(w=None)), (-1, dict(sw=None)), (-1, dict(y=None)), (-5, dict(x=A + 8)), (-5, dict(w=A + 8)), (-5, dict(bias=A + 2)),
                                     (-5, dict(y=A + 2)), (0, dict(M=0, x=None, y=None))])
def test_matmul(lib, want, kw):
    assert matmul(lib, **kw) == want


@pytest.mark.parametrize("want,kw", [(-2, dict(E=0)), (-2, dict(E=1025)), (-2, dict(stride=2040)), (-2, dict(stride=1024)), (-2, dict(act=abi.ACT_SWIGLU)), (-2, dict(y_rows=3)), (-2, dict(y_rows=-1)),
                                     (-1, dict(offsets=None)), (-5, dict(offsets=A + 1)), (-5, dict(out_rows=A + 2)), (0, dict(M=0, offsets=None))])
def test_grouped(lib, want, kw):
    assert grouped(lib, **kw) == want


@pytest.mark.parametrize("want,kw", [(-1, dict(ws=None)), (-5, dict(ws=A + 16)), (-4, dict(nbytes=255)), (-2, dict(M=-3)), (-2, dict(K=0)), (-1, dict(w=None)), (0, dict(M=0, ws=None, x=None))])
def test_linear(lib, want, kw):
    assert linear(lib, **kw) == want


@pytest.mark.parametrize("want,kw", [(-2, dict(T=-1)), (-2, dict(k=0)), (-2, dict(T=1 << 30, k=8)), (-2, dict(E=0)), (-2, dict(act=abi.ACT_NONE)), (-2, dict(H=0)), (-2, dict(F=131072)),
                                     (-2, dict(stride_up=2048)), (-1, dict(perm=None)), (-1, dict(offsets=None)), (-1, dict(ws=None)), (-5, dict(offsets=A + 2)), (-4, dict(nbytes=512)),
                                     (0, dict(T=0, ws=None, perm=None))])
def test_experts(lib, want, kw):
    assert experts(lib, **kw) == want


def test_scratch_sizes(lib):
    linear, experts = lib.chimere_b200_linear_w8a8_bytes, lib.chimere_b200_experts_w8a8_bytes
    assert linear(-1, 32, 64) == -2 and linear(4, 32, 0) == -2 and linear(4, 32, 131072) == -2 and linear(4, 0, 64) == -2
    assert linear(0, 32, 64) == 0 and linear(1, 4096, 2048) == 0            # one launch: no scratch
    assert linear(9, 32, 2005) >= 9 * (2016 + 4) and linear(1, 32, 20000) >= 20004 and linear(70000, 32, 131071) >= 70000 * 131076
    assert experts(8, 2, 64, 0) == -2 and experts(-1, 2, 64, 64) == -2 and experts(1, 0, 64, 64) == -2 and experts(1 << 30, 8, 64, 64) == -2
    assert experts(4, 2, 64, 33) >= 8 * (64 + 4 + 48 + 4 + 33 * 4)
    assert experts(4096, 8, 2048, 64) >= 32768 * (2048 + 4 + 64 + 4 + 64 * 4) + 4096 * 2052
