"""Training-block operators on the GPU where a rule of their launches ends: empty tables, the
largest rows and widths, several host threads, sizes whose races or rounding small ones hide."""

import pytest
import torch

import block_refs as R
from flashcart_b200 import ops

pytestmark = pytest.mark.gpu

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("dim", [3, 5, 8, 63, 64])
def test_embedding_in_an_empty_table(cuda_device, dtype, dim):
    """No row to read: zeros, the status bit, and a gradient without rows."""
    ops.check_device_status()
    table = torch.empty(0, dim, dtype=dtype, device="cuda", requires_grad=True)
    for rows in (1, 259):
        idx = torch.arange(rows, device="cuda") - 1
        y = ops.embedding(table, idx, 2.0, 1.0)
        assert torch.equal(y, torch.zeros(rows, dim, dtype=dtype, device="cuda"))
        (g,) = torch.autograd.grad(y, table, torch.ones_like(y))
        assert g.shape == (0, dim)
        with pytest.raises(RuntimeError, match="outside"):
            ops.check_device_status()
    assert ops.embedding(table, idx[:0]).shape == (0, dim)
    ops.check_device_status()
