"""Single derivatives and values of gated_linear's activations in their tails, each relative to itself.

With one row x = 1 and u = dout = 1, dwg is the derivative of every gate and dwu its activation.  Both are rounded to
bf16 (half a step, 2^-8 of the value; the products with 1 are exact).  Before that they hold e to the power of an argument
of at most 87, whose roundings (four at most, 2^-24 of it each) are below 2^-15 of the value, and factors good to 2^-20.
The gates end where the values leave the normal range."""
import pytest

from test_gpu_gated_linear import act_and_grad

pytestmark = pytest.mark.gpu

GATES = {"silu": [-20.0, -31.0, -32.0, -33.0, -35.0, -40.0, -50.0, -64.5, -80.0, -86.0, -1.25, 33.0, 50.0, 100.0],
         "gelu": [-3.0, -5.0, -7.0, -9.0, -11.0, -12.0, -12.75, -1.25, 5.0, 9.0, 31.0, 33.0, 50.0, 100.0],
         "gelu_tanh": [-3.0, -5.0, -6.5, -7.0, -8.0, -9.0, -9.5, -1.25, 5.0, 9.0, 31.0, 33.0, 50.0, 100.0]}


@pytest.mark.parametrize("act", list(GATES))
def test_tails(cuda, act):
    torch = cuda
    from bee_b200 import tensor_cuda as tc
    g = torch.tensor([GATES[act]]).bfloat16().cuda()
    n = g.shape[1]
    one, x, w = torch.ones_like(g), torch.ones(1, 8, dtype=g.dtype, device="cuda"), torch.zeros(8, n, dtype=g.dtype, device="cuda")
    dwg, dwu = torch.empty_like(w), torch.empty_like(w)
    tc.gated_linear_backward(x, w, w, g, one, one, None, dwg, dwu, act=act)
    for got, want in zip((dwu, dwg), act_and_grad(g.double(), act)):
        off = ((got.double() - want) / want).abs()
        assert (off <= 2.0 ** -8 + 2.0 ** -14).all(), (act, off.max(0).values.tolist())
