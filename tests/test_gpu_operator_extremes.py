"""The embedding, list and AdamW operators at the far ends of what they accept, and in the calls that programs make
around them: other streams and threads, repeated backward passes, transforms of torch.func."""
import pytest
import torch

from recommend_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,D", [(torch.float32, (1 << 27) + 5), (torch.bfloat16, (1 << 28) + 9)])
@pytest.mark.parametrize("n", [0, 1])
def test_rows_whose_vectors_pass_32_bits(dtype, D, n):
    """64 rows of more than 2^25 vectors of 16 bytes have more than 2^31 of them.  Rows without an id are zeros, in memory
    that held something else; factors of two round nothing."""
    ids = torch.ones(n, dtype=torch.int64, device=DEV)
    table = torch.empty(3, D, dtype=dtype, device=DEV)
    table[0], table[1], table[2] = 3.0, 1.5, 5.0
    table[1, 7::11] = -0.25
    table.requires_grad_(True)
    out = ops.embedding_lookup(table, ids, scale=2.0)
    grad = torch.full((n, D), 0.5, dtype=dtype, device=DEV)
    grad[:, ::13] = -4.0
    for i in range(n):
        assert torch.equal(out[i], 2 * table.detach()[1])
    torch.full((3, D), float("nan"), dtype=dtype, device=DEV)          # (the next tensor of this size gets its memory)
    dw, = torch.autograd.grad(out, table, grad)
    assert bool((dw[0] == 0).all()) and bool((dw[2] == 0).all())
    assert torch.equal(dw[1], 2 * grad[0] if n else torch.zeros_like(dw[1]))
