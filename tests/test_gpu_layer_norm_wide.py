"""Layer norm of the widest rows: launches, and sums of 2^26 terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
D = (1 << 26) + 17


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from maskplanner_amd import ops as O
    return O


def make(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((2, D), generator=gen, device="cuda")


def test_parameter_gradients_of_2_26_columns(ops):
    """more columns than one grid of the last reduction covers.  With weight 1 and bias 0 the result is z itself, formed by the backward pass in the
    same way: a product and a sum a row, one rounding at the end, 2 x 2 + 1 roundings (2^-24) of the absolute terms"""
    x, dy = make(1), make(2)
    w, b = torch.ones(D, device="cuda", requires_grad=True), torch.zeros(D, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    y.backward(dy)
    z, g = y.detach().double(), dy.double()
    assert ((w.grad.double() - (g * z).sum(0)).abs() <= 5 * U * (g * z).abs().sum(0)).all()
    assert ((b.grad.double() - g.sum(0)).abs() <= 5 * U * g.abs().sum(0)).all()
