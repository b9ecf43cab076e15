"""Rows of gated_linear's operands and gradients that end inside a 16-byte block of a stride of whole blocks: what follows
a row in memory takes no part in the products and is left as it was (a TMA store cuts whole blocks only)."""
import pytest

from test_gpu_gated_linear import ACTS, check_backward, check_forward, forward, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("m,d,f", [(3, 5, 17), (2, 13, 46), (72, 61, 18), (300, 541, 261), (130, 257, 1039), (600, 2049, 9)])
@pytest.mark.parametrize("more", [0, 8])
def test_rows_end_inside_a_block(cuda, m, d, f, trans, dtype, more):
    torch = cuda
    act = ACTS[(m + d + f) % 3]
    extra = -(d if trans else f) % 8 + more  # the weights' strides, and those of their gradients, are whole blocks
    x, wg, wu, dout = make(torch, m, d, f, dtype, trans, 7, extra=extra)
    assert wg.stride(0) % 8 == 0 and wg.shape[1] % 8 != 0
    check_forward(torch, x, wg, wu, act, trans)
    _, g, u = forward(torch, x, wg, wu, act, trans)
    check_backward(torch, x, wg, wu, g, u, dout, act, trans, extra)
