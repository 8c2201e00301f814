"""How exact 16-bit Newton-Schulz results are, over the spectra that weight gradients have: full rank, rank of a batch, one dominating direction.

Tolerance.  A 16-bit result is off by its own rounding, r = |round(exact) - exact|_F, and by what the evaluation adds in front of it; the
library states that this is less than r.  The two are independent (the rounding takes whatever value it is given), so they add in squares:
    |out - exact|_F <= sqrt(2) r.
r is formed from the exact result itself, 1e-3 (bfloat16) or 2e-4 (float16) of its norm: a wrong tile, a missing step or a zero is hundreds of
times as far off, which every check asserts.  At most five steps: further ones multiply by 3.4 each what any fp32 arithmetic leaves in
directions that the matrix does not have (2^-24 to begin with).  Below 256 elements r is a matter of luck: there half a step of every element is taken for it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)
HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from maskplanner_amd import ops as O
    return O


def normal(*shape, seed):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def make(rows, cols, kind, dtype, seed=7):
    """kind: "full", "dominated" (one direction 100 times the rest), "decay" (singular values like 1 / k), or the rank"""
    k = min(rows, cols)
    if kind == "full":
        g = normal(rows, cols, seed=seed)
    elif kind == "dominated":
        g = normal(rows, 1, seed=seed) * normal(1, cols, seed=seed + 1) + 1e-2 * normal(rows, cols, seed=seed + 2)
    elif kind == "decay":
        g = (normal(rows, k, seed=seed) / torch.arange(1, k + 1, device="cuda")) @ normal(k, cols, seed=seed + 1)
    else:
        k = min(k, kind)
        g = normal(rows, k, seed=seed) @ normal(k, cols, seed=seed + 1)
    return (1e-3 * g).to(dtype)


def exact(u, steps=5, eps=1e-7):
    """float64, from the definition"""
    u = u.double()
    x = u.t().contiguous() if u.shape[0] > u.shape[1] else u
    x = x / max(float(x.norm()), eps)
    for _ in range(steps):
        a = x @ x.t().contiguous()
        x = COEF[0] * x + (COEF[1] * a + COEF[2] * (a @ a)) @ x
    return x.t().contiguous() if u.shape[0] > u.shape[1] else x


def check(out, want, what):
    dtype, norm = out.dtype, float(want.norm())
    r = float((want.to(dtype).double() - want).norm()) if want.numel() >= 256 else torch.finfo(dtype).eps / 2 * norm
    assert r <= 0.01 * norm, what
    assert float((out.double() - want).norm()) <= 2 ** 0.5 * r, (what, float((out.double() - want).norm()) / r)


def both_forms(ops, g, steps, what):
    want = exact(g, steps)
    check(ops.orthogonalize([g], steps=steps)[0], want, what)
    p, m = torch.zeros_like(g), g.float()                     # the momentum is the gradient and stays so: p = -orthogonalize(g), rounded once
    ops.muon_step([p], [g], [m], lr=1.0, scale=None, steps=steps)
    check(-p, want, (what, "muon"))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ["full", "dominated", "decay", 1, 8, 32, 128])
@pytest.mark.parametrize("rows,cols", [(16, 1100), (100, 300), (256, 512), (512, 512), (1024, 1024), (1500, 700), (300, 3000)])
def test_spectra_of_gradients(ops, rows, cols, kind, dtype):
    both_forms(ops, make(rows, cols, kind, dtype), 5, (rows, cols, kind, dtype))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", ["full", "dominated", 1, 32])
@pytest.mark.parametrize("steps", [1, 2, 3, 4])
def test_step_counts(ops, steps, kind, dtype):
    for rows, cols in ((512, 512), (128, 131), (60, 60)):
        both_forms(ops, make(rows, cols, kind, dtype), steps, (rows, cols, kind, dtype, steps))


SIZES = [(1, 7), (9, 1), (3, 64), (31, 33), (32, 32), (63, 65), (64, 64), (65, 64), (100, 300), (300, 100), (128, 131), (128, 128), (129, 1000), (257, 255),
         (2100, 65), (40, 9000), (640, 500), (8, 4096), (4097, 3), (9, 500), (1000, 20), (1500, 1700)]


@pytest.mark.parametrize("dtype", HALF)
def test_sizes_alone_and_in_one_list(ops, dtype):
    gs = [make(r, c, "full", dtype, 3 * i) for i, (r, c) in enumerate(SIZES)]
    for size, g, out in zip(SIZES, gs, ops.orthogonalize(gs)):
        want = exact(g)
        check(out, want, (size, "list"))
        check(ops.orthogonalize([g])[0], want, (size, "alone"))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["original", "match_rms", None])
def test_muon_step_with_everything(ops, dtype, nesterov, scale):
    """Momentum of its own, decay and step factors: the weight is rounded once, r its rounding; what is added in front of it (momentum and
    direction in fp32, the factors) is again less than the rounding, as the step is as large as the decayed weight here (lr s = 0.5, weights of
    an orthogonal matrix's size).  The lists take the one-launch kernels (first) and the chain."""
    for sizes in ([(64, 3), (64, 64), (5, 100), (8, 4096), (200, 40)], [(64, 64), (128, 131), (256, 128), (70, 500), (6, 1024), (512, 512)]):
        gs = [make(r, c, "full", dtype, 3 * i) for i, (r, c) in enumerate(sizes)]
        ms = [1e-3 * normal(r, c, seed=100 + i) for i, (r, c) in enumerate(sizes)]
        ps = [(normal(r, c, seed=200 + i) / max(r, c) ** 0.5).to(dtype) for i, (r, c) in enumerate(sizes)]
        old, before = [p.double() for p in ps], [m.double() for m in ms]
        ops.muon_step(ps, gs, ms, lr=0.5, momentum=0.9, nesterov=nesterov, weight_decay=0.2, scale=scale)
        for (r, c), p, g, m, p0, m0 in zip(sizes, ps, gs, ms, old, before):
            gd = g.double()
            mean = m0 + 0.1 * (gd - m0)
            s = {"original": max(1.0, r / c) ** 0.5, "match_rms": 0.2 * max(r, c) ** 0.5, None: 1.0}[scale]
            want = 0.9 * p0 - 0.5 * s * exact(gd + 0.9 * (mean - gd) if nesterov else mean)
            check(p, want, (r, c, dtype, nesterov, scale))
            # a difference, a product with a rounded factor, a sum: four roundings of the operands' size
            assert ((m.double() - mean).abs() <= 4 * 2.0 ** -24 * (gd.abs() + m0.abs())).all()


@pytest.mark.parametrize("rows,cols", [(64, 600), (600, 64), (32, 1100), (16, 2000)])
def test_small_float32_squares_keep_the_low_planes_in_any_company(ops, rows, cols):
    """A^2 of fewer than 128 rows takes the product of the low planes too, whatever tiles the launch has because of other matrices in it.  A case
    that is exact in binary: rows of 2^-4 (1, 2^-6, 2^-6, 0, ..), eps = 1 above the norm, so X is the matrix itself; the entries of A are
    2^-8 (1 + 2^-11), high plane 1, low plane 2^-11; those of A^2 are m 2^-16 (1 + 2^-10 + 2^-22) with the low planes' product, without it the
    2^-22 is missing from the result X <- A^2 X (coefficients 0, 0, 1).
    Tolerance, half of that: the last product sums m entries 1 + 2^-10 (high) and 2^-22 (low), 16 at a time.  fp32 steps are 2^-19 from 16 on,
    2^-18 from 32 on; 16 low products are 2^-18, but where the matrix instruction adds them in two parts each part is half a step from 32 on
    and may round away: for m = 64 the last two groups of four, 2 x 2^-18 of 64, or 2^-23 of the result; none for m <= 32."""
    m = min(rows, cols)
    g = torch.zeros(m, max(rows, cols), device="cuda")
    g[:, 5] = 2.0 ** -4
    g[:, 100] = g[:, 101] = 2.0 ** -10
    gd = g.double()
    a = gd @ gd.t().contiguous()
    want = (a @ a) @ gd
    assert torch.equal(want.float().double(), want)
    if rows > cols:
        g, want = g.t().contiguous(), want.t().contiguous()
    for others in ([], [normal(2048, 2048, seed=99)], [normal(300, 3000, seed=98)], [normal(1024, 1024, seed=90), normal(150, 130, seed=91)]):
        out = ops.orthogonalize([g] + others, steps=1, coefficients=(0.0, 0.0, 1.0), eps=1.0)[0]
        assert ((out.double() - want).abs() <= 2.0 ** -23 * want).all(), [o.shape for o in others]


@pytest.mark.parametrize("rows,cols", [(8, 20), (40, 50), (20, 900), (70, 90), (90, 70), (300, 900), (1000, 9)])
def test_norms_far_below_eps(ops, rows, cols):
    """X = G / eps is tiny and stays so: the steps multiply it by a each (A is next to nothing).  Half a step of X's planes (2^-23), a product and a
    scale a step: 4 x 2^-23 x 5 = 2.4e-6 of the result, however small it is."""
    for scale, eps in ((1e-12, 1e-3), (1e-14, 1e-7), (1e-16, 1e-7), (1e-20, 1e-7), (1e-24, 1e-7), (1e-3, 1e9), (1e-18, 1.0)):
        g = scale * normal(rows, cols, seed=2)
        want = exact(g, eps=eps)
        got = [ops.orthogonalize([g], eps=eps)[0], ops.orthogonalize([g, normal(400, 300, seed=3)], eps=eps)[0]]
        p, m = torch.zeros_like(g), g.clone()
        ops.muon_step([p], [g], [m], lr=1.0, scale=None, eps=eps)
        for out in got + [-p]:
            assert float((out.double() - want).norm()) <= 2.4e-6 * float(want.norm()), (scale, eps)
        h = g.to(torch.bfloat16)
        check(ops.orthogonalize([h], eps=eps)[0], exact(h, eps=eps), (scale, eps))


@pytest.mark.parametrize("rows,cols", [(40, 50), (70, 90), (300, 900)])
def test_norms_around_eps(ops, rows, cols):
    """From |X| = 1 down to where the steps are linear.  A step is off by at most 2^-22 (1.4 x 13 + 8) of |X| (two steps on the Gram matrix), and what
    it leaves grows by 485 at most, as X itself does at 0."""
    for ratio in (2.0, 1.0, 0.3, 3e-2, 3e-3, 1e-3, 3e-4, 1e-5):
        g = normal(rows, cols, seed=4)
        g = g / g.norm() * 1e-7 * ratio
        want = exact(g)
        bound = 5 * 2.0 ** -22 * (1.4 * 13 + 8) * 485 * min(ratio, 1.0)
        assert float((ops.orthogonalize([g])[0].double() - want).norm()) <= bound, ratio
        h = g.to(torch.bfloat16)
        check(ops.orthogonalize([h])[0], exact(h), ratio)
