"""Layer normalisation on the HIP kernels against a plain implementation in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and h = half a step of the storage type (finfo.eps / 2):

* y: x - mean carries the rounding of the mean, which is an fp32 sum of D terms (a tree over threads: at most ~log2 D + 64 roundings in a
  row, together below 80 u) relative to max|x|; rstd is relative to the same order.  |dy| <= (160 u (1 + max|x| rstd) + h) max(1, |y|, |w|).
* dx: a difference of three terms of the size of rstd * max|g| and the means' sums: 400 u of that size, plus h.
* every result: below the storage type's smallest normal number n the step no longer shrinks: a rounding is off by up to n * h absolutely
  (fp16: n = 2^-14, so 2^-25; a weight gradient of one row has entries that small).
* dw, db: sums over the rows: 80 u + (rows / partial sums <= 512) u / 2 of the sum of absolute terms, plus h of the result.  The error of
  z = (x - mean) rstd is absolute (the mean's, see y: a z near 0 keeps it), so the terms of dw count with |dy| (|z| + 1).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from maskplanner_amd import ops as O
    return O


def reference(x, w, b, dy, eps):
    """value and gradients in float64 on the CPU."""
    x, w, b, dy = (None if t is None else t.detach().double().cpu() for t in (x, w, b, dy))
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    z = (x - mean) * rstd
    y = z * (1.0 if w is None else w) + (0.0 if b is None else b)
    g = dy * (1.0 if w is None else w)
    dx = rstd * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, x.shape[-1]).sum(0)                                     # noqa: E731
    return dict(y=y, dx=dx, dw=flat(dy * z), db=flat(dy), z=z, rstd=rstd, g=g, dw_abs=flat((dy * z).abs() + dy.abs()), db_abs=flat(dy.abs()), x=x)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def low(dtype):
    """half the step of subnormal results"""
    return torch.finfo(dtype).tiny * half_step(dtype)


def check(x, w, b, dy, eps, got):
    r = reference(x, w, b, dy, eps)
    y, dx, dw, db = got
    h = half_step(x.dtype)
    wmax = 1.0 if w is None else float(w.detach().abs().max())
    cond = (1.0 + r["x"].abs().amax(-1, keepdim=True) * r["rstd"])
    big = torch.maximum(r["y"].abs(), torch.full_like(r["y"], max(1.0, wmax)))
    assert ((y.double().cpu() - r["y"]).abs() <= (160 * U * cond + h) * big + low(x.dtype)).all()
    if dx is not None:
        size = r["rstd"] * r["g"].abs().amax(-1, keepdim=True) * (1.0 + r["z"].abs()) * cond
        assert ((dx.double().cpu() - r["dx"]).abs() <= 400 * U * size + h * r["dx"].abs() + low(x.dtype)).all()
    for name, t in (("dw", dw), ("db", db)):
        if t is None:
            continue
        hw = half_step(t.dtype)
        tol = 400 * U * r[name + "_abs"] * (float(cond.max()) if name == "dw" else 1.0) + hw * r[name].abs() + low(t.dtype)
        assert ((t.double().cpu() - r[name]).abs() <= tol).all(), name


def run(ops, x, w, b, dy, eps=1e-5):
    x = x.detach().requires_grad_(True)
    ws = [None if t is None else t.detach().requires_grad_(True) for t in (w, b)]
    y = ops.layer_norm(x, *ws, eps=eps)
    leaves = [x] + [t for t in ws if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, dy))
    dx = next(grads)
    return y.detach(), dx, next(grads) if w is not None else None, next(grads) if b is not None else None


def make(shape, dtype, wdtype, seed, affine="wb"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    D = shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * 1.5 + 0.5).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(wdtype) if "w" in affine else None
    b = (0.3 * torch.randn(D, generator=g, device="cuda")).to(wdtype) if "b" in affine else None
    return x, w, b, torch.randn(shape, generator=g, device="cuda").to(dtype)


# every (threads a row, vectors a thread) form on both sides of its limits, for 4- and 2-byte rows; the loop form behind 8192 / 16384
WIDTHS = [1, 2, 3, 7, 8, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 500, 511, 512, 513, 999, 1000, 1023, 1024, 1025, 2048, 2049,
          4095, 4097, 8191, 8192, 8193, 16385]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_every_width(ops, D, dtype):
    rows = 37 if D > 600 else 300
    x, w, b, dy = make((rows, D), dtype, torch.float32, D)
    check(x, w, b, dy, 1e-5, run(ops, x, w, b, dy))


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 999), (3, 128), (1023, 700), (1024, 700), (1025, 1500), (5000, 300), (20001, 64), (9000, 999),
                                    (70, 16400)])
@pytest.mark.parametrize("affine", ["wb", "w", "b", ""])
def test_row_counts_types_and_missing_parameters(ops, rows, D, dtype, wdtype, affine):
    x, w, b, dy = make((rows, D), dtype, wdtype, rows + D, affine)
    check(x, w, b, dy, 1e-5, run(ops, x, w, b, dy))


def test_leading_shapes(ops):
    for shape in ((129,), (2, 3, 129), (2, 0, 129), (0, 129), (1, 1, 1, 5)):
        x, w, b, dy = make(shape, torch.float32, torch.float32, 3)
        got = run(ops, x, w, b, dy)
        assert got[0].shape == x.shape and got[1].shape == x.shape
        if x.numel():
            check(x, w, b, dy, 1e-5, got)
        else:
            assert not got[2].any() and not got[3].any()


def test_strided_rows_columns_and_upstream_gradients(ops):
    x, w, b, dy = make((60, 300), torch.float32, torch.float32, 5)
    for xv, dyv in ((x[:, 17:250], dy[:, 3:236]), (x[::3, :233], dy[::3, 40:273]), (x.t()[:233, :].t().expand(60, 233), dy[:1, :233].expand(60, 233)),
                    (x[:60, :120].t(), dy[:60, :120].t()), (x[:, ::2], dy[:, ::2]), (x[:1, :7].expand(60, 7), dy[:, :7])):
        D = xv.shape[-1]
        check(xv, w[:D], b[:D], dyv, 1e-5, run(ops, xv, w[:D], b[:D], dyv))
    # sum(): the upstream gradient is one number expanded over everything
    xv = x.detach().requires_grad_(True)
    ops.layer_norm(xv, w, b).sum().backward()
    r = reference(x, w, b, torch.ones_like(x), 1e-5)
    assert ((xv.grad.double().cpu() - r["dx"]).abs() <= 400 * U * r["rstd"] * 3 * (1 + r["z"].abs())).all()


def test_odd_addresses(ops):
    """views that start at every element offset of a 16-byte vector."""
    for dtype in (torch.float32, torch.bfloat16):
        flat, w, b, dyf = make((4000,), dtype, torch.float32, 9)
        w, b = w[:61].contiguous(), b[:61].contiguous()
        for off in range(9):
            x, dy = flat[off:off + 61 * 61].view(61, 61), dyf[off:off + 61 * 61].view(61, 61)
            check(x, w, b, dy, 1e-5, run(ops, x, w, b, dy))


def test_constant_rows_and_offsets(ops):
    """variance 0: z is 0 exactly, rstd = 1 / sqrt(eps); a large common offset must not cancel the variance away."""
    x = torch.full((5, 256), 3.0, device="cuda")
    w, b = torch.full((256,), 2.0, device="cuda"), torch.full((256,), 0.25, device="cuda")
    dy = torch.randn(5, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    got = run(ops, x, w, b, dy)
    assert torch.equal(got[0], torch.full_like(x, 0.25))
    check(x, w, b, dy, 1e-5, got)
    x2 = torch.randn(64, 500, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) + 1000.0
    dy2 = torch.randn(64, 500, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    check(x2, None, None, dy2, 1e-5, run(ops, x2, None, None, dy2))


def test_infinities_and_nan_stay_in_their_rows(ops):
    for D in (40, 700, 20000):
        x, w, b, dy = make((6, D), torch.float32, torch.float32, D)
        want = run(ops, x, w, b, dy)
        bad = x.clone()
        bad[1, D // 2] = float("inf")
        bad[4, 0] = float("nan")
        got = run(ops, bad, w, b, dy)
        keep = [0, 2, 3, 5]
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
        assert got[0][[1, 4]].isnan().all() and got[1][[1, 4]].isnan().all()
        assert torch.equal(got[3], want[3])                     # db does not read x
        assert got[2].isnan().all()


def test_gradient_against_differences(ops):
    """central differences of the kernel's own forward pass in a direction: f'(t) of sum(y dy).  Truncation O(t^2) relative 1e-4 at t = 1e-2,
    rounding 2^-24 * sqrt(n) * |y dy| / t: 1e-3 of the derivative's scale covers both."""
    x, w, b, dy = make((40, 96), torch.float32, torch.float32, 11)
    dirs = [torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(20 + i)) for i, t in enumerate((x, w, b))]
    _, dx, dw, db = run(ops, x, w, b, dy)
    t = 1e-2
    for k, grad in enumerate((dx, dw, db)):
        def f(sign):
            a = [x, w, b]
            a[k] = a[k] + sign * t * dirs[k]
            return float((ops.layer_norm(*a).double() * dy.double()).sum())
        num, ana = (f(1) - f(-1)) / (2 * t), float((grad.double() * dirs[k].double()).sum())
        scale = float((grad.double().norm() * dirs[k].double().norm()))
        assert abs(num - ana) <= 1e-3 * scale


def test_reproducible_and_partial_gradients(ops):
    x, w, b, dy = make((30000, 200), torch.bfloat16, torch.float32, 4)
    a, c = run(ops, x, w, b, dy), run(ops, x, w, b, dy)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        t = [v.detach().requires_grad_(n) for v, n in zip((x, w, b), need)]
        g = torch.autograd.grad(ops.layer_norm(*t), [v for v, n in zip(t, need) if n], dy)
        assert all(torch.equal(p, q) for p, q in zip(g, [q for q, n in zip(a[1:], need) if n]))
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b), a[0])


def test_side_stream_and_replayed_graph(ops):
    x, w, b, dy = make((500, 333), torch.float32, torch.float32, 6)
    want = run(ops, x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(ops, x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    xs, dys = x.clone(), dy.clone()
    with torch.cuda.stream(s):
        run(ops, xs, w, b, dys)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(ops, xs, w, b, dys)
    for k in range(3):
        x2, _, _, dy2 = make((500, 333), torch.float32, torch.float32, 60 + k)
        xs.copy_(x2)
        dys.copy_(dy2)
        g.replay()
        eager = run(ops, x2, w, b, dy2)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_refusals(ops):
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (lambda: ops.layer_norm(x, w[:7]), lambda: ops.layer_norm(x, w.half()), lambda: ops.layer_norm(x, w, w.double()),
                lambda: ops.layer_norm(x.double(), None), lambda: ops.layer_norm(x.half(), w, w.half()), lambda: ops.layer_norm(x, w, eps=-1.0),
                lambda: ops.layer_norm(x, w, eps=float("nan")), lambda: ops.layer_norm(x[:, :0], None), lambda: ops.layer_norm(x[0, 0], None)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.layer_norm(x, w.cpu())
    xg = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(ops.layer_norm(xg, w).square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


# vectors of a row (16 bytes each) on both sides of every form's limits; rows enough for the register form of the backward pass, and for some
# workgroups to walk several of them
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("vecs,rows", [(65, 1100), (128, 6200), (129, 1100), (192, 3300), (193, 1100), (256, 1700), (257, 700), (512, 600), (513, 300),
                                       (768, 300), (769, 300), (1024, 300), (1025, 300), (1536, 300), (1537, 300), (2047, 270), (2048, 65)])
@pytest.mark.parametrize("off", [0, 1])
def test_every_form_backward(ops, vecs, rows, off, dtype, wdtype):
    V = 16 // dtype.itemsize
    x, w, b, dy = make((rows, vecs * V - off), dtype, wdtype, vecs + off)
    check(x, w, b, dy, 1e-5, run(ops, x, w, b, dy))


def test_offsets_beyond_32_bits(ops):
    """2^31 elements and more, 4.3 GB a tensor: first, middle and last rows against 64 bits, the others zeros (y = b, dx = 0, nothing in dw)"""
    rows, D = (1 << 21) + 3, 1100
    x = torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros_like(x)
    at = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    xs, w, b, dys = make((len(at), D), torch.bfloat16, torch.float32, 5)
    x[at], dy[at] = xs, dys
    y, dx, dw, db = run(ops, x, w, b, dy)
    check(xs, w, b, dys, 1e-5, (y[at], dx[at], dw, db))
    for r in (2, rows // 2 + 1, rows - 3):
        assert torch.equal(y[r], b.to(torch.bfloat16)) and not dx[r].any()
