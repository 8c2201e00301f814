"""Layer norm and Muon as a model uses them: the module, the segmenters with point_norm="layer", the optimizer classes, TrainStep, and all of them in
one training loop -- each against the same step in 64 bits."""
import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_layer_norm_module_over_one_and_two_axes():
    """difference from float64: 160 roundings (2^-24) of values of order |z| (1 + |x| rstd) <= 40 here"""
    from maskplanner_amd.layer_norm import LayerNorm
    for shape, affine in (((96,), True), ((4, 6), True), ((96,), False)):
        m = LayerNorm(shape, elementwise_affine=affine).cuda()
        if affine:
            torch.nn.init.normal_(m.weight)
            torch.nn.init.normal_(m.bias)
        x = torch.randn(7, 5, *shape, device="cuda", generator=gen(1), requires_grad=True)
        y = m(x)
        y.square().sum().backward()
        xd = x.detach().double().cpu().requires_grad_(True)
        w, b = (m.weight.detach().double().cpu().requires_grad_(True), m.bias.detach().double().cpu().requires_grad_(True)) if affine else (None, None)
        yd = F.layer_norm(xd, shape, w, b, m.eps)
        yd.square().sum().backward()
        tol = 160 * 2.0 ** -24 * 40
        assert (y.double().cpu() - yd).abs().max() <= tol
        assert (x.grad.double().cpu() - xd.grad).abs().max() <= 8 * tol * float(yd.abs().max())
        if affine:
            for p, q in ((m.weight, w), (m.bias, b)):      # sums of 35 such terms
                assert (p.grad.double().cpu() - q.grad).abs().max() <= 35 * 4 * tol * float(yd.abs().max())


@pytest.mark.parametrize("cls", ["PointNet2Segmenter_v1", "PointNet2Segmenter_PaintNet_v1"])
def test_segmenter_with_layer_norm_matches_64_bits(cls):
    """Head only: the encoder's output is taken from the model itself.  fp32 Linears over 1027, 512 and 256 terms and three norms: each stage
    is off by at most (K + 160) 2^-24 of its inputs' absolute sums, a few 1e-4 of the features' size (1 behind a norm) in all."""
    from maskplanner_amd import pointnet2_seg
    torch.manual_seed(0)
    model = getattr(pointnet2_seg, cls)(point_norm="layer").cuda().eval()
    pts = torch.randn(3, 3, 700, device="cuda", generator=gen(2))
    kept = {}
    model.sa3.register_forward_hook(lambda mod, args, out: kept.__setitem__("g", out[1].detach()))
    trunk = []
    inner = model._trunk
    model._trunk = lambda *a: trunk.append(inner(*a)) or trunk[-1]
    with torch.no_grad():
        model(pts)
    d = {k: v.double().cpu() for k, v in model.state_dict().items()}
    g, x = kept["g"].double().cpu().reshape(3, 1024), pts.double().cpu()
    h = torch.cat([g[:, :, None].expand(-1, -1, 700), x], 1).transpose(1, 2)
    for k, c in ((1, 512), (2, 256), (3, 128)):
        h = F.relu(F.layer_norm(F.linear(h, d[f"conv{k}.weight"][:, :, 0], d[f"conv{k}.bias"]), (c,), d[f"bn{k}.weight"], d[f"bn{k}.bias"], 1e-5))
    assert (trunk[0].double().cpu() - h.transpose(1, 2)).abs().max() <= 1e-3
    # a cloud's result does not depend on its neighbours in the batch, in training mode either
    model.train()
    x1, x2 = (torch.randn(2, 50, 512, device="cuda", generator=gen(s)) for s in (3, 3))
    assert torch.equal(model.bn1(x1)[:1], model.bn1(x2[:1]))


def test_muon_optimizer_equals_the_formula():
    """two steps of two groups and three types against float64; the bound is the update's: see the orthogonalisation's own tests -- here 1e-3 of
    the step plus the weight type's half step, over ten times what those bounds come to for these sizes in fp32"""
    from maskplanner_amd.muon import Muon
    ps = [torch.randn(s, device="cuda", generator=gen(i)).to(t).requires_grad_(True)
          for i, (s, t) in enumerate((((40, 30), torch.float32), ((64, 16, 1, 1), torch.float32), ((50, 80), torch.bfloat16), ((30, 30), torch.float16)))]
    opt = Muon([{"params": ps[:1], "lr": 0.1, "nesterov": False}, {"params": ps[1:], "weight_decay": 0.1}], lr=0.05, scale="match_rms")
    ref = [p.detach().double().cpu() for p in ps]
    mom = [torch.zeros_like(r) for r in ref]
    for step in range(2):
        for i, p in enumerate(ps):
            p.grad = (1e-2 * torch.randn(p.shape, device="cuda", generator=gen(50 + 10 * step + i))).to(p.dtype)
        ps[3].grad = None if step == 1 else ps[3].grad                     # a parameter without a gradient is left alone
        opt.step()
        for i, p in enumerate(ps):
            if p.grad is None:
                continue
            lr, nest, wd = (0.1, False, 0.0) if i == 0 else (0.05, True, 0.1)
            g = p.grad.double().cpu()
            mom[i] = mom[i] + 0.05 * (g - mom[i])
            u = (g + 0.95 * (mom[i] - g) if nest else mom[i]).flatten(1)
            x = u.t() if u.shape[0] > u.shape[1] else u
            x = x / x.norm()
            for _ in range(5):
                a = x @ x.t()
                x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
            o = (x.t() if u.shape[0] > u.shape[1] else x).reshape(p.shape)
            ref[i] = (1 - lr * wd) * ref[i] - lr * 0.2 * max(u.shape) ** 0.5 * o
            err = (p.detach().double().cpu() - ref[i]).abs()
            assert (err <= 1e-3 * lr * 0.2 * max(u.shape) ** 0.5 + (step + 1) * torch.finfo(p.dtype).eps / 2 * (ref[i].abs() + 1)).all(), i
        assert all(opt.state[p]["momentum_buffer"].dtype == torch.float32 for p in ps)


def test_muon_notices_a_stale_graph():
    """the update is in place: a backward pass through what a weight was must raise"""
    from maskplanner_amd.muon import Muon
    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    x = torch.randn(8, 8, device="cuda", requires_grad=True)
    loss = (x @ w).sum()
    w.grad = torch.randn(8, 8, device="cuda")
    Muon([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_muon_recorded_after_one_step_and_refused_before():
    from maskplanner_amd.muon import Muon

    def make():
        w = torch.randn(70, 90, device="cuda", generator=gen(1)).requires_grad_(True)
        w.grad = torch.randn(70, 90, device="cuda", generator=gen(2))
        return w, Muon([w], lr=0.1)
    w, opt = make()
    with pytest.raises(RuntimeError, match="before recording"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    (a, oa), (b, ob) = make(), make()
    oa.step()
    ob.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
    for k in range(3):
        for t in (a, b):
            t.grad.copy_(torch.randn(70, 90, device="cuda", generator=gen(20 + k)))
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, b) and torch.equal(oa.state[a]["momentum_buffer"], ob.state[b]["momentum_buffer"])


def test_train_step_with_muon_eager_and_replayed():
    """the replayed step makes the eager step's updates: Muon on the encoder's matrices, Adam on the rest"""
    from maskplanner_amd.harness import TrainStep
    from maskplanner_amd.muon import MuonAdam
    kw = dict(B=2, N=1024, hidden_size=(128, 128), optimizer="muon", muon={"weight_decay": 0.01})
    a, b = TrainStep("cuboids", graph=False, **kw), TrainStep("cuboids", graph=True, **kw)
    for t in (a, b):
        assert isinstance(t.opt, MuonAdam) and len(t.opt.muon.param_groups[0]["params"]) == 9
        t.model.dropout.p = 0.0
    before = copy.deepcopy(a.model.state_dict())
    losses = [[float(t.step()) for _ in range(7)] for t in (a, b)]
    torch.cuda.synchronize()
    assert b._graph is not None
    assert all(x == x for row in losses for x in row)
    # atomics and arg-max routing make two runs differ (see the gradient tests); the first step starts from the same weights
    assert abs(losses[0][0] - losses[1][0]) <= 1e-4 * abs(losses[0][0])
    for n, p in a.model.named_parameters():
        assert torch.isfinite(p).all(), n
        if n.startswith("sa") and p.ndim > 1:
            moved = [(t.model.state_dict()[n] - before[n]).flatten(1) for t in (a, b)]
            # seven steps of an orthogonalised direction (singular values 0.68 .. 1.2, 1.21 bound) of size lr sqrt(max(1, rows / columns))
            r, c = moved[0].shape
            bound = 7 * 0.02 * max(1.0, r / c) ** 0.5 * 1.25 * min(r, c) ** 0.5 + 7 * 0.02 * 0.01 * float(before[n].norm()) * 1.2
            for m in moved:
                assert 0 < float(m.norm()) <= bound, n


def test_layer_norm_model_trained_by_muon_and_adam_in_one_loop():
    """a normalised two-layer head, three steps: forward, loss, backward, MuonAdam; every weight against the same loop in float64.  Per step an
    entry of a matrix moves by at most lr, off by 1e-3 of that (orthogonalisation of a gradient that is itself off by ~1e-5 relative, amplified
    by at most 485 / its rank's root); Adam's first steps are lr sign-like: 1e-2 lr where |g| is small against eps."""
    from maskplanner_amd.layer_norm import LayerNorm
    from maskplanner_amd.muon import MuonAdam
    torch.manual_seed(5)
    net = torch.nn.Sequential(torch.nn.Linear(24, 48), LayerNorm(48), torch.nn.ReLU(), torch.nn.Linear(48, 16), LayerNorm(16)).cuda()
    ref = torch.nn.Sequential(torch.nn.Linear(24, 48), torch.nn.LayerNorm(48), torch.nn.ReLU(), torch.nn.Linear(48, 16), torch.nn.LayerNorm(16)).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    mats = [p for p in net.parameters() if p.ndim > 1]
    opt = MuonAdam(mats, [p for p in net.parameters() if p.ndim == 1], lr=1e-3, muon_lr=0.02)
    mom = {n: torch.zeros_like(p) for n, p in ref.named_parameters()}
    sq = {n: torch.zeros_like(p) for n, p in ref.named_parameters()}
    for step in range(3):
        x = torch.randn(333, 24, device="cuda", generator=gen(step))
        y = torch.randn(333, 16, device="cuda", generator=gen(10 + step))
        opt.zero_grad()
        (net(x) - y).square().mean().backward()
        opt.step()
        ref.zero_grad()
        (ref(x.double().cpu()) - y.double().cpu()).square().mean().backward()
        with torch.no_grad():
            for n, p in ref.named_parameters():
                g = p.grad
                if p.ndim > 1:
                    mom[n] += 0.05 * (g - mom[n])
                    u = g + 0.95 * (mom[n] - g)
                    z = (u.t() if u.shape[0] > u.shape[1] else u)
                    z = z / z.norm()
                    for _ in range(5):
                        a = z @ z.t()
                        z = 3.4445 * z + (-4.7750 * a + 2.0315 * (a @ a)) @ z
                    p -= 0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * (z.t() if u.shape[0] > u.shape[1] else z)
                else:
                    mom[n] += 0.1 * (g - mom[n])
                    sq[n] = 0.999 * sq[n] + 0.001 * g * g
                    p -= 1e-3 / (1 - 0.9 ** (step + 1)) * mom[n] / (sq[n].sqrt() / (1 - 0.999 ** (step + 1)) ** 0.5 + 1e-8)
    for (n, p), q in zip(net.named_parameters(), ref.parameters()):
        tol = 3 * 0.02 * 1.5 * 1e-3 if p.ndim > 1 else 3 * 1e-3 * 1e-2
        assert float((p.detach().double().cpu() - q.detach()).abs().max()) <= tol + 2.0 ** -22, n


def test_layer_norm_module_keeps_the_input_type_under_autocast():
    """the output has the input's type; its values are those of the same numbers in float32, rounded (2^-11), each of the two within 160 roundings of
    2^-24 (1 + max|x| / std) <= 10 of the exact one"""
    from maskplanner_amd.layer_norm import LayerNorm
    m = LayerNorm(300).cuda()
    x = (3 + torch.randn(50, 300, device="cuda", generator=gen(1))).half()
    with torch.autocast("cuda", dtype=torch.float16):
        y, z = m(x), m(x.float())
    assert y.dtype == torch.float16 and z.dtype == torch.float32 and torch.equal(z, m(x.float()))
    assert ((y.float() - z).abs() <= 2.0 ** -11 * z.abs() + 2 * 160 * 2.0 ** -24 * 10).all()
