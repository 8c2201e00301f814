"""Newton-Schulz orthogonalisation and the Muon update on the HIP kernels against 64 bits.

Tolerance.  One step's rounding: operands kept to 2^-22 (two fp16 planes), products accumulated in fp32; in a hop of h steps on the Gram
matrix the smallest eigenvalues' relative error grows by a^2 < 12 per further step.  So a step's result is off by at most
e_h = 2^-22 * 1.4 * (1 + 12 + .. + 12^(h-1)) + 8 * 2^-22 of its norm (1.4 = |b| / a: how an eigenvalue's error enters a I + b A + c A^2; 8: the
product itself, three plane products and the fp32 sums): fp32 takes h <= 2, the 16-bit types h <= 5.  What a step leaves is carried by the
polynomial of the steps behind it, whose largest slope over the singular values that occur is `sens` (at most a^5 = 485, at 0).  Five steps:
    |out - exact|_F <= 5 e_h (sens |X_0|_F + |exact|_F) + h |exact|_F,      h half a step of the result's type.
A wrong tile, row or element is off by the size of the entries themselves.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    from maskplanner_amd import ops as O
    return O


def f_of(s, steps, coef):
    for _ in range(steps):
        s = s * (coef[0] + coef[1] * s ** 2 + coef[2] * s ** 4)
    return s


def reference(g, steps=5, coef=COEF, eps=1e-7):
    """float64 on the CPU, from the definition"""
    g = g.detach().double().cpu()
    x = g.t() if g.shape[0] > g.shape[1] else g
    x = x / max(float(x.norm()), eps)
    x0 = x
    for _ in range(steps):
        a = x @ x.t()
        x = coef[0] * x + (coef[1] * a + coef[2] * (a @ a)) @ x
    return (x.t() if g.shape[0] > g.shape[1] else x), x0


def tolerance(want, x0, dtype, steps=5, coef=COEF):
    s = torch.linspace(0, 1, 4001, dtype=torch.float64)
    lo = float(torch.linalg.svdvals(x0).min()) if min(x0.shape) <= 512 else 0.0
    s = s[s >= lo * 0.999] if lo < 0.999 else torch.tensor([lo], dtype=torch.float64)
    s = torch.cat([s, torch.tensor([max(lo, 1e-9)], dtype=torch.float64)])
    d = 1e-7
    sens = max(float((f_of(s, steps, coef) / s.clamp_min(1e-9)).abs().max()), float(((f_of(s + d, steps, coef) - f_of(s - d, steps, coef)) / (2 * d)).abs().max()))
    hop = min(steps, 2 if dtype == torch.float32 else 5)
    e = 2.0 ** -22 * (1.4 * sum(12.0 ** k for k in range(hop)) + 8)
    return steps * e * (sens * float(x0.norm()) + float(want.norm())) + torch.finfo(dtype).eps / 2 * float(want.norm()) + torch.finfo(dtype).tiny


def check(got, g, **kw):
    want, x0 = reference(g, **kw)
    kw.pop("eps", None)
    assert got.shape == g.shape and got.dtype == g.dtype
    err = (got.double().cpu() - want).norm()
    assert float(err) <= tolerance(want, x0, g.dtype, **kw), (float(err), float(want.norm()))


def make(rows, cols, dtype=torch.float32, seed=0, kind="gradient"):
    gen = torch.Generator(device="cuda").manual_seed(seed * 100003 + rows * 131 + cols)
    g = torch.randn((rows, cols), generator=gen, device="cuda")
    if kind == "gradient":
        g += torch.randn((rows, 1), generator=gen, device="cuda") * torch.randn((1, cols), generator=gen, device="cuda")
    if kind == "lowrank":
        g = torch.randn((rows, 1), generator=gen, device="cuda") * torch.randn((1, cols), generator=gen, device="cuda") + 1e-2 * g
    return (1e-3 * g).to(dtype)


def dirty(mb=64):
    """leave NaN bits in the allocator's free blocks: nothing may depend on what a workspace holds"""
    t = torch.full((mb * 262144,), float("nan"), device="cuda")
    del t


SIZES = [(1, 1), (1, 7), (9, 1), (2, 2), (3, 64), (64, 3), (31, 33), (32, 32), (33, 31), (63, 65), (64, 64), (65, 64), (100, 300), (300, 100),
         (127, 129), (128, 131), (128, 128), (129, 1000), (257, 255), (300, 3000), (2100, 65), (40, 9000), (640, 500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_one_matrix(ops, rows, cols, dtype):
    dirty()
    g = make(rows, cols, dtype)
    (out,) = ops.orthogonalize([g])
    check(out, g)


@pytest.mark.parametrize("kind", ["plain", "gradient", "lowrank"])
def test_spectra(ops, kind):
    for dtype in (torch.float32, torch.bfloat16):
        g = make(150, 260, dtype, 5, kind)
        check(ops.orthogonalize([g])[0], g)


def test_a_list_of_many_sizes(ops):
    """more matrices than one pass takes, sizes and hop lengths mixed, empty ones among them: each as if alone, bit for bit where the split of the
    work is the same, and within the tolerance everywhere"""
    sizes = SIZES + [(0, 5), (5, 0)] + [(20 + i, 30 + 3 * i) for i in range(15)]
    for dtype in (torch.float32, torch.bfloat16):
        gs = [make(r, c, dtype, 3) for r, c in sizes]
        dirty()
        outs = ops.orthogonalize(gs)
        assert len(outs) == len(gs)
        for g, o in zip(gs, outs):
            if g.numel():
                check(o, g)
            else:
                assert o.shape == g.shape
    assert ops.orthogonalize([]) == []


def test_batched_tensor_and_strides(ops):
    g = torch.stack([make(48, 80, seed=i) for i in range(6)]).view(2, 3, 48, 80)
    out = ops.orthogonalize(g)
    for i in range(2):
        for j in range(3):
            check(out[i, j], g[i, j])
    assert ops.orthogonalize(g[:0]).shape == (0, 3, 48, 80)
    base = make(200, 300)
    for v in (base.t(), base[:, 5:90], base[::2, ::3], base[3:4].expand(9, 300)):
        check(ops.orthogonalize([v])[0], v)


def test_large_tiles_and_split_products(ops):
    """enough work for the 128 x 128 tiles, and a long K over few tiles"""
    for dtype in (torch.float32, torch.float16):
        g = make(1500, 1700, dtype, 2)
        check(ops.orthogonalize([g])[0], g)
    g = make(130, 20000, torch.float32, 2)
    check(ops.orthogonalize([g])[0], g)


def test_magnitudes(ops):
    """norms whose squares leave fp32, and below eps: X = G / eps there"""
    for scale in (1e30, 1e-20, 1e-30):
        g = make(70, 90) * scale
        kw = {} if scale > 1 else {"eps": 0.0}
        check(ops.orthogonalize([g], **kw)[0], g, **kw)
    g = make(70, 90) * 1e-12
    check(ops.orthogonalize([g])[0], g)
    z = torch.zeros(40, 50, device="cuda")
    assert not ops.orthogonalize([z])[0].any()
    one = torch.zeros(40, 50, device="cuda")
    one[7, 9] = -3.0
    check(ops.orthogonalize([one])[0], one)


def test_not_finite_stays_in_its_matrix(ops):
    gs = [make(60, 70, seed=i) for i in range(3)]
    want = ops.orthogonalize(gs)
    for bad in (float("nan"), float("inf")):
        hs = [g.clone() for g in gs]
        hs[1][5, 6] = bad
        got = ops.orthogonalize(hs)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        assert got[1].isnan().any()


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (3, COEF), (8, (1.875, -1.25, 0.375)), (16, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(ops, steps, coef):
    for dtype in (torch.float32, torch.bfloat16):
        for size in ((90, 90), (64, 500)):
            g = make(*size, dtype, 8)
            (out,) = ops.orthogonalize([g], steps=steps, coefficients=coef)
            want, x0 = reference(g, steps, coef)
            # a of these is 1.5 to 3.45: eigenvalues grow by a^2 <= 12 a step, sens as computed
            assert float((out.double().cpu() - want).norm()) <= tolerance(want, x0, dtype, steps, coef)


def test_same_bits_twice_side_stream_and_replayed_graph(ops):
    gs = [make(r, c, torch.float32, 4) for r, c in ((64, 3), (128, 131), (256, 5000), (300, 200))]
    want = ops.orthogonalize(gs)
    dirty()
    assert all(torch.equal(a, b) for a, b in zip(want, ops.orthogonalize(gs)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.orthogonalize(gs)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    static = [g.clone() for g in gs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(static)
    for k in range(3):
        new = [make(*g.shape, torch.float32, 40 + k) for g in gs]
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        eager = ops.orthogonalize(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


# ------------------------------------------------------------------------------------------------------------ Muon
def muon_reference(p, g, m, lr, mu, nesterov, wd, scale):
    p, g, m = (t.double().cpu() for t in (p, g, m))
    m = m + (1 - mu) * (g - m)
    u = g + mu * (m - g) if nesterov else m
    u2 = u.flatten(1)
    o, x0 = reference(u2)
    r, c = u2.shape
    s = {"original": max(1.0, r / c) ** 0.5, "match_rms": 0.2 * max(r, c) ** 0.5, None: 1.0}[scale]
    return (1 - lr * wd) * p - lr * s * o.view_as(p), m, lr * s, o, x0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["original", "match_rms", None])
def test_muon_step(ops, dtype, nesterov, scale):
    u = 2.0 ** -24
    shapes = [(64, 3, 1, 1), (64, 64, 1, 1), (128, 131, 1, 1), (256, 128), (500, 70), (1, 40), (33, 1), (6, 1024)]
    ps = [torch.randn(s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(dtype) for i, s in enumerate(shapes)]
    gs = [make(s[0], p.numel() // s[0], dtype, 6).view(s) for s, p in zip(shapes, ps)]
    ms = [make(s[0], p.numel() // s[0], torch.float32, 7).view(s) for s, p in zip(shapes, ps)]
    for _ in range(2):
        want = [muon_reference(p, g, m, 0.05, 0.9, nesterov, 0.1, scale) for p, g, m in zip(ps, gs, ms)]
        before = [(p._version, m._version) for p, m in zip(ps, ms)]
        old = [m.clone() for m in ms]
        ops.muon_step(ps, gs, ms, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
        for p, g, m, o, w, b in zip(ps, gs, ms, old, want, before):
            # momentum: a difference, a product with a rounded 1 - mu and a sum: 4 roundings of the operands' size
            assert ((m.double().cpu() - w[1]).abs() <= 4 * u * (g.double().abs().cpu() + o.double().abs().cpu())).all()
            # weight: decay and step factors rounded, product, difference (4 u |p|, 4 u of the step), the orthogonalisation's own error
            # in fp32 form (u is formed in fp32 from a gradient and a momentum of its size), one rounding to the weight's type
            hop5 = dtype != torch.float32
            tol_o = tolerance(w[3], w[4], torch.float32) * (2700 if hop5 else 1)      # e_5 / e_2 = 1.4 (12^5 - 1) / 11 / (1.4 * 13 + 8) < 1212
            h = torch.finfo(dtype).eps / 2
            err = (p.double().cpu() - w[0]).norm()
            assert float(err) <= w[2] * (tol_o + 4 * u * float(w[3].norm())) + (4 * u + h) * float(w[0].norm() + w[2] * w[3].norm()) + torch.finfo(dtype).tiny
            assert p._version > b[0] and m._version > b[1]


def test_muon_step_in_a_graph(ops):
    def state(seed):
        return [[make(r, c, seed=seed + k) for r, c in ((64, 3), (128, 131), (256, 512))] for k in (0, 1, 2)]
    a, b = state(1), state(1)
    ops.muon_step(*a, lr=0.1, weight_decay=0.01)
    graph = torch.cuda.CUDAGraph()
    c = state(1)
    with torch.cuda.graph(graph):
        ops.muon_step(*b, lr=0.1, weight_decay=0.01)
    for k in range(3):
        for t, s in zip(b[0] + b[2], c[0] + c[2]):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(a[0] + a[2], b[0] + b[2]))


def test_refusals(ops):
    g = make(8, 9)
    ok = dict(lr=0.1)
    for bad in (lambda: ops.orthogonalize([g, g.half()]), lambda: ops.orthogonalize([g.double()]), lambda: ops.orthogonalize([g[0]]),
                lambda: ops.orthogonalize(g[0]), lambda: ops.orthogonalize([g], steps=0), lambda: ops.orthogonalize([g], steps=17),
                lambda: ops.orthogonalize([g], coefficients=(1.0, 2.0)), lambda: ops.orthogonalize([g], eps=-1.0),
                lambda: ops.orthogonalize([g], coefficients=(float("nan"), 0.0, 0.0)),
                lambda: ops.muon_step([g], [g], [], **ok), lambda: ops.muon_step([g], [g], [g.half()], **ok),
                lambda: ops.muon_step([g], [g.half()], [g.clone()], **ok), lambda: ops.muon_step([g.t()], [g.t()], [g.t().contiguous()], **ok),
                lambda: ops.muon_step([g[0]], [g[0]], [g[0].clone()], **ok), lambda: ops.muon_step([g], [g], [g.clone()], scale="other", **ok),
                lambda: ops.muon_step([g, g], [g, g], [g.clone(), g.clone()], **ok)):
        with pytest.raises(ValueError):
            bad()
    from maskplanner_amd._lib import MaskPlannerHipError
    with pytest.raises(MaskPlannerHipError):
        ops.orthogonalize([g], coefficients=(30.0, 0.0, 0.0))       # singular values grow by 30 a step
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.orthogonalize([g.cpu()])
    ops.muon_step([], [], [], **ok)


@pytest.mark.parametrize("kind", ["plain", "gradient", "lowrank"])
@pytest.mark.parametrize("rows,cols", [(256, 256), (700, 700), (1000, 1300), (1300, 1000)])
def test_bfloat16_steps_on_one_plane(ops, rows, cols, kind):
    """The last two bf16 steps round X, A and Q to fp16: each is off by an rms of 2^-12 / sqrt(3) of its entries, six such roundings, the first
    three carried through a step of slope <= a = 3.45 whose rms over singular values near 1 is about 1: they add at most 0.5 of the result's own
    rounding (rms 2^-9 / sqrt(3), 8 times as large), the Gram-side hop before them 0.4.  In 2-norm together with it: sqrt(1 + 0.25 + 0.16) = 1.19."""
    g = make(rows, cols, torch.bfloat16, 11, kind)
    want, _ = reference(g)
    rounding = float((want.to(torch.bfloat16).double() - want).norm())
    p, m = torch.zeros_like(g), g.float()
    outs = [ops.orthogonalize([g])[0], ops.orthogonalize([g, make(90, 120, torch.bfloat16), g])[2]]
    ops.muon_step([p], [g], [m], lr=1.0, scale=None)         # the momentum is the gradient: p = -orthogonalize(g)
    for out in outs + [-p]:
        assert float((out.double().cpu() - want).norm()) <= 1.19 * rounding


def test_offsets_beyond_32_bits(ops):
    """more than 2^31 elements: columns of the result from the small side in float64, R = Q_5 .. Q_1 of A = X X^T.  Tolerance as above."""
    m, n = 1040, (1 << 21) - 5
    gen = torch.Generator(device="cuda").manual_seed(9)
    g = torch.empty((m, n), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    gram = torch.zeros((m, m), dtype=torch.float64, device="cuda")
    for c in range(0, n, 1 << 18):
        part = g[:, c:c + (1 << 18)].double()
        gram += part @ part.t()
        del part
    norm = float(gram.trace().sqrt())
    a, r = gram / norm ** 2, torch.eye(m, dtype=torch.float64, device="cuda")
    for _ in range(5):
        q = COEF[0] * torch.eye(m, dtype=torch.float64, device="cuda") + COEF[1] * a + COEF[2] * a @ a
        a, r = q @ a @ q, q @ r
    cols = torch.tensor([0, 1, 12345, n // 2, n - 700, n - 2, n - 1], device="cuda")
    want = r @ (g[:, cols].double() / norm)
    tol = tolerance(want.cpu(), (g[:, cols].double() / norm).cpu(), torch.bfloat16)
    (out,) = ops.orthogonalize([g])
    assert float((out[:, cols].double() - want).norm()) <= tol
    del out
    tall = g.t().contiguous()
    del g
    (out,) = ops.orthogonalize([tall])
    assert float((out[cols].t().double() - want).norm()) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 2), (8, 8), (3, 5), (8, 1024), (1024, 8), (7, 1025), (1025, 7), (5, 2000), (1, 4096), (4096, 8), (8, 4096),
                                       (8, 4097), (4097, 3), (9, 500), (500, 9), (32, 1000), (1000, 20)])
def test_thin_matrices(ops, rows, cols, dtype):
    """both sides of the limits of the one-launch forms for up to 8, 32 and 64 rows, alone and in one list"""
    dirty()
    g = make(rows, cols, dtype, 4)
    other = make(cols, rows, dtype, 5)
    for got, want in zip(ops.orthogonalize([g]) + ops.orthogonalize([other, g, make(40, 60, dtype, 6)]), (g, other, g, make(40, 60, dtype, 6))):
        check(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_of_small_matrices(ops, dtype, nesterov):
    """lists that take the one-launch forms only: update and momentum as in test_muon_step, same tolerances"""
    u = 2.0 ** -24
    shapes = [(64, 3, 1, 1), (64, 64, 1, 1), (5, 100), (100, 5), (8, 4096), (3000, 7), (33, 200), (1, 1), (200, 40), (20, 900)]
    ps = [torch.randn(s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(dtype) for i, s in enumerate(shapes)]
    gs = [make(s[0], p.numel() // s[0], dtype, 6).view(s) for s, p in zip(shapes, ps)]
    ms = [make(s[0], p.numel() // s[0], torch.float32, 7).view(s) for s, p in zip(shapes, ps)]
    for _ in range(2):
        want = [muon_reference(p, g, m, 0.05, 0.9, nesterov, 0.1, "original") for p, g, m in zip(ps, gs, ms)]
        old = [m.clone() for m in ms]
        ops.muon_step(ps, gs, ms, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
        for p, g, m, o, w in zip(ps, gs, ms, old, want):
            assert ((m.double().cpu() - w[1]).abs() <= 4 * u * (g.double().abs().cpu() + o.double().abs().cpu())).all()
            tol_o, h = tolerance(w[3], w[4], torch.float32), torch.finfo(dtype).eps / 2
            err = (p.double().cpu() - w[0]).norm()
            assert float(err) <= w[2] * (tol_o + 4 * u * float(w[3].norm())) + (4 * u + h) * float(w[0].norm() + w[2] * w[3].norm()) + torch.finfo(dtype).tiny
