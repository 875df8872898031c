"""Results over the rows they come from: where one launch reads and stores, the C entry refuses, and the Python call takes two steps (no GPU needed)."""
import pytest
import torch

from chimere_b200 import abi, build, w8a8

A = 1 << 20   # a non-null, aligned placeholder: never dereferenced on the host
REFUSED = -2


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def linear(lib, x, ldx, y, ldy, M=8, N=64, K=64, ws=None, nbytes=0, x_type=abi.TYPE_BF16, y_type=abi.TYPE_BF16):
    return lib.chimere_b200_linear_w8a8(x, x_type, ldx, A, 64, A, None, M, N, K, abi.ACT_NONE, y, y_type, ldy, ws, nbytes, None, None)


# (x, ldx, y, ldy) of eight rows of 64 values of two bytes
SHARED = [(A, 64, A, 64), (A, 64, A + 2, 64), (A, 64, A + 2 * (7 * 64 + 63), 64), (A + 2 * (7 * 64 + 63), 64, A, 64), (A, 128, A + 126, 128), (A, 128, A + 130, 128), (A + 130, 128, A, 128), (A, 200, A + 2 * 64, 128),
          (A, 64, A - 2, 100)]
APART = [(A, 64, A + 2 * 512, 64), (A + 2 * 512, 64, A, 64), (A, 128, A + 128, 128), (A + 128, 128, A, 128), (A, 128, A + 128 + 256 * 3, 128), (A, 200, A + 2 * 1600, 64)]


@pytest.mark.parametrize("args", SHARED)
def test_one_launch_over_its_own_rows_is_refused(lib, args):
    assert lib.chimere_b200_linear_w8a8_bytes(8, 64, 64) == 0
    assert linear(lib, *args) == REFUSED
    x, ldx, y, ldy = args
    assert linear(lib, y, ldy, x, ldx) == REFUSED


def test_one_row_of_other_types(lib):
    assert linear(lib, A, 64, A + 254, 64, M=1, x_type=abi.TYPE_F32) == REFUSED           # (x: 256 bytes)
    assert linear(lib, A + 254, 64, A, 64, M=1, y_type=abi.TYPE_F32) == REFUSED


def test_what_needs_scratch_is_not_refused_for_it(lib):
    """Its rows have been read when results are stored: the next error in line answers."""
    assert linear(lib, A, 64, A, 64, M=9, ws=A, nbytes=0) == -4


def views(x, ldx, y, ldy):
    buf = torch.empty(4000, dtype=torch.bfloat16)
    low = min(x, y)
    return [torch.as_strided(buf, (8, 64), (ld, 1), (at - low) // 2) for at, ld in ((x, ldx), (y, ldy))]


@pytest.mark.parametrize("args,want", [(a, True) for a in SHARED] + [(a, False) for a in APART])
def test_the_python_call_sees_the_same(args, want):
    a, b = views(*args)
    assert w8a8._share_memory(a, args[1], b, args[3]) is want and w8a8._share_memory(b, args[3], a, args[1]) is want
    used = [set((t.storage_offset() + i * ld + j) for i in range(8) for j in range(64)) for t, ld in ((a, args[1]), (b, args[3]))]
    assert not (used[0] & used[1]) or want          # (never apart where an element is shared)


def test_nothing_is_shared_with_no_rows():
    a = torch.empty(4, 64)
    assert not w8a8._share_memory(a[:0], 64, a, 64) and not w8a8._share_memory(a, 64, a[:0], 64)
