"""What the balance-loss entries refuse before anything is launched (no GPU needed)."""
import pytest

from chimere_b200 import abi, build

A = 4096   # a non-null, aligned placeholder: never dereferenced on the host


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def loss(lib, logits=A, type=abi.TYPE_F32, ld=16, stride=160, ids=A, mask=None, S=2, L=10, E=16, k=2, mode=0, out=A, counts=A, prob=A, tokens=A, gl=None, d=None, ldd=16, stride_d=160, ws=A, nbytes=1 << 24):
    return lib.chimere_b200_balance_loss(logits, type, ld, stride, ids, mask, S, L, E, k, mode, 1.0, out, counts, prob, tokens, gl, d, ldd, stride_d, ws, nbytes, None)


def backward(lib, logits=A, type=abi.TYPE_BF16, ld=16, stride=160, mask=None, counts=A, tokens=A, S=2, L=10, E=16, k=2, mode=1, gl=None, d=A, ldd=16, stride_d=160):
    return lib.chimere_b200_balance_loss_backward(logits, type, ld, stride, mask, counts, tokens, S, L, E, k, mode, 1.0, gl, d, ldd, stride_d, None)


BAD = [(-2, dict(S=-1)), (-2, dict(L=-1)), (-2, dict(E=0)), (-2, dict(E=257, ld=257, ldd=257)), (-2, dict(k=0)), (-2, dict(k=257)), (-2, dict(mode=2)), (-2, dict(ld=15)), (-2, dict(stride=-1)),
       (-2, dict(S=1 << 20, L=1 << 12)), (-2, dict(L=1 << 24, k=128, S=1)), (-3, dict(type=2)), (-1, dict(logits=None)), (-1, dict(counts=None)), (-1, dict(tokens=None)), (-5, dict(logits=A + 1)),
       (-5, dict(counts=A + 2)), (-5, dict(gl=A + 2)), (-2, dict(d=A, ldd=15)), (-2, dict(d=A, stride_d=159)), (-5, dict(d=A + 1)), (0, dict(S=0))]


@pytest.mark.parametrize("want,kw", BAD + [(-1, dict(ids=None)), (-1, dict(out=None)), (-1, dict(prob=None)), (-1, dict(ws=None, L=100000, stride=1600000)), (-5, dict(ws=A + 64)), (-5, dict(ids=A + 2)),
                                           (-4, dict(L=100000, nbytes=4096, stride=1600000))])
def test_loss(lib, want, kw):
    assert loss(lib, **kw) == want


@pytest.mark.parametrize("want,kw", BAD + [(-1, dict(d=None)), (0, dict(L=0, logits=None))])
def test_backward(lib, want, kw):
    assert backward(lib, **kw) == want


def test_scratch_sizes(lib):
    f = lib.chimere_b200_balance_loss_bytes
    assert f(0, 10, 16, 2) == 0 and f(1, 0, 16, 2) == 0 and f(1, 10, 16, 2) == 0 and f(1, 10, 0, 2) == -2 and f(1, 10, 257, 2) == -2 and f(1, 10, 16, 0) == -2 and f(-1, 10, 16, 2) == -2
    assert f(1, 1 << 20, 256, 8) > f(1, 1 << 10, 256, 8) and f(16, 8192, 256, 8) < 1 << 22
