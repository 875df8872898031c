"""linear_w8a8's scratch: asked for where the size function names some, and no address made up where it names none (no GPU needed)."""
import os
import re

import pytest

from chimere_b200 import abi, build

A = 1 << 20   # a non-null, aligned placeholder: never dereferenced on the host


@pytest.fixture(scope="module")
def lib():
    build.build()
    return abi.load()


def test_no_address_is_made_up():
    """A pointer that must not be used is null, which the launch refuses: an address of one's own would be written to if two places ever decided differently."""
    with open(os.path.join(build.CSRC, "w8a8.cu")) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\(\s*\w+\s*\*\s*\)\s*(0x)?\d", code) and not re.search(r"reinterpret_cast<[^>]*\*>\(\s*\d", code)


@pytest.mark.parametrize("M", [1, 2, 5, 8, 9, 300])
@pytest.mark.parametrize("K", [1, 16, 2048, 2049, 8192, 8193, 131071])
@pytest.mark.parametrize("N", [1, 64, 4736, 4737, 40000])
def test_what_needs_scratch_is_refused_without(lib, M, N, K):
    need, ld = lib.chimere_b200_linear_w8a8_bytes(M, N, K), (K + 15) // 16 * 16
    linear = lambda ws, n: lib.chimere_b200_linear_w8a8(A, abi.TYPE_F32, K, A, ld, A, None, M, N, K, abi.ACT_NONE, A, abi.TYPE_F32, N, ws, n, None, None)   # noqa: E731
    assert need == 0 or need >= M * (ld + 4)
    if need:
        assert linear(None, 0) == -1 and linear(None, need) == -1 and linear(A, need - 1) == -4
    else:
        assert M <= 8 and linear(None, 0) == -2        # (one launch; x and y are the same memory here)
