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


def test_sums_of_2_26_terms(ops):
    """Thread sums in fp64, then a tree of eight fp32 sums and a division: the mean is off by at most 12 U of itself and rstd by 12 U, so z by
    12 U |mean| rstd + 14 U |z| (the difference's and the product's own roundings among them).  The means of g and g z likewise 12 U of the mean
    of their absolute terms (and of z's error), dx with its three products and two differences within 40 U of its terms' sizes.  y below: z itself."""
    x = (make(3) + 3.0).requires_grad_(True)
    dy = make(4) + 0.5
    y = ops.layer_norm(x)
    y.backward(dy)
    xd, g = x.detach().double(), dy.double()
    mean = xd.mean(1, keepdim=True)
    rstd = 1.0 / (((xd - mean) ** 2).mean(1, keepdim=True) + 1e-5).sqrt()
    z = (xd - mean) * rstd
    tol = U * (12 * mean.abs() * rstd + 14 * z.abs() + 1)
    assert ((y.detach().double() - z).abs() <= tol).all()
    means = [(g.mean(1, keepdim=True), g.abs().mean(1, keepdim=True)), ((g * z).mean(1, keepdim=True), (g * z).abs().mean(1, keepdim=True))]
    want = rstd * (g - means[0][0] - z * means[1][0])
    size = rstd * (g.abs() + means[0][1] + (z.abs() + mean.abs() * rstd + 1) * means[1][1])
    assert ((x.grad.double() - want).abs() <= 40 * U * size).all()
