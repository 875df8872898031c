"""padded_i8: rows on 16-byte boundaries, whatever the matrix lies in (no GPU needed)."""
import pytest
import torch

from chimere_b200 import w8a8


@pytest.mark.parametrize("shape", [(4, 64), (1, 16), (3, 5), (1, 1), (2, 3, 32), (2, 3, 33)])
@pytest.mark.parametrize("at", [0, 1, 8, 16, 24])
def test_rows_start_on_boundaries(shape, at):
    n = 1
    for s in shape:
        n *= s
    q = torch.arange(n + at, dtype=torch.int32).to(torch.int8)[at:].view(shape)        # contiguous, from an odd address on
    for m in (q, q.transpose(-1, -2)):
        p = w8a8.padded_i8(m)
        assert torch.equal(p, m) and p.data_ptr() % 16 == 0 and p.stride(-1) == 1
        assert all(d % 16 == 0 for s, d in zip(p.shape[:-1], p.stride()) if s > 1)
    whole = torch.zeros(4, 64, dtype=torch.int8)
    assert w8a8.padded_i8(whole).data_ptr() == whole.data_ptr()
