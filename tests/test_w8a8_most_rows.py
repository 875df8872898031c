"""The most rows that a product takes: beyond, the number of its tiles would not fit 32 bits (no GPU needed)."""
import pytest

from chimere_b200 import abi, build

A = 1 << 20   # a non-null, aligned placeholder: never dereferenced on the host
MOST = 0x7FFFFF00


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


@pytest.mark.parametrize("M", [MOST + 1, 2 ** 31 - 64, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1])
def test_products(lib, M):
    assert lib.chimere_b200_matmul_w8a8(A, 16, A, A, 16, A, None, M, 1, 16, abi.ACT_NONE, A, abi.TYPE_F32, 1, None, None) == -2
    assert lib.chimere_b200_matmul_w8a8_grouped(A, 16, A, A, 16, 16, A, None, A, 1, M, 1, 16, abi.ACT_NONE, A, abi.TYPE_F32, 1, M, None, None, None) == -2
    assert lib.chimere_b200_linear_w8a8_bytes(M, 1, 16) == -2
    assert lib.chimere_b200_linear_w8a8(A, abi.TYPE_F32, 16, A, 16, A, None, M, 1, 16, abi.ACT_NONE, A, abi.TYPE_F32, 1, A, 1 << 60, None, None) == -2


@pytest.mark.parametrize("T,k", [(MOST + 1, 1), (2 ** 31 - 1, 1), (MOST // 3 + 1, 3)])
def test_experts(lib, T, k):
    assert lib.chimere_b200_experts_w8a8_bytes(T, k, 16, 16) == -2
    assert lib.chimere_b200_experts_w8a8(A, abi.TYPE_F32, 16, T, A, A, k, 1, A, 16, 512, A, A, 16, 256, A, 16, 16, abi.ACT_SWIGLU, A, abi.TYPE_F32, 16, A, 1 << 60, None, None) == -2


def test_the_most_has_a_size(lib):
    assert lib.chimere_b200_linear_w8a8_bytes(MOST, 1, 16) >= MOST * 20 and lib.chimere_b200_experts_w8a8_bytes(MOST, 1, 16, 16) > MOST * 20
