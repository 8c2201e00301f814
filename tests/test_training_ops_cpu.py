"""Layer norm, orthogonalisation and Muon without a GPU: argument checks before the device is touched, module and optimizer bookkeeping."""
import ctypes

import pytest
import torch


def _arr(t, v):
    return (t * len(v))(*v)


def test_c_entries_check_before_they_launch():
    from maskplanner_amd import _lib
    lib = _lib.load()
    i64 = ctypes.c_int64
    # layer norm: null pointers, dtype, widths, missing half of the statistics, workspace
    assert lib.mp_layer_norm_fwd(None, 0, 4, 8, 8, None, None, 0, 1e-5, None, None, None, None) == _lib.MP_EINVAL
    assert lib.mp_layer_norm_fwd(None, 0, 0, 8, 8, None, None, 0, 1e-5, None, None, None, None) == _lib.MP_OK
    assert lib.mp_layer_norm_fwd(64, 0, 4, 0, 8, None, None, 0, 1e-5, 64, None, None, None) == _lib.MP_EINVAL
    assert lib.mp_layer_norm_fwd(64, 7, 4, 8, 8, None, None, 0, 1e-5, 64, None, None, None) == _lib.MP_EUNSUPPORTED
    assert lib.mp_layer_norm_fwd(64, 0, 4, 8, 8, None, None, 1, 1e-5, 64, None, None, None) == _lib.MP_EUNSUPPORTED      # fp16 parameters of fp32 rows
    assert lib.mp_layer_norm_fwd(64, 0, 4, 8, 8, None, None, 0, 1e-5, 64, 64, None, None) == _lib.MP_EINVAL
    assert lib.mp_layer_norm_fwd(64, 0, 4, 8, 8, None, None, 0, float("nan"), 64, None, None, None) == _lib.MP_EINVAL
    assert lib.mp_layer_norm_fwd(64, 0, 1 << 31, 8, 8, None, None, 0, 1e-5, 64, None, None, None) == _lib.MP_EUNSUPPORTED
    need = lib.mp_layer_norm_bwd_workspace_bytes(1000, 70, 0)
    assert need > 0 and lib.mp_layer_norm_bwd_workspace_bytes(0, 70, 0) == 0
    assert lib.mp_layer_norm_bwd(64, 70, 64, 70, 0, 1000, 70, None, 0, 64, 64, None, 64, None, None, 0, None) == _lib.MP_EWORKSPACE
    assert lib.mp_layer_norm_bwd(64, 70, 64, 70, 0, 1000, 70, None, 0, 64, 64, None, 64, None, 64, need - 1, None) == _lib.MP_EWORKSPACE
    assert lib.mp_layer_norm_bwd(None, 70, 64, 70, 0, 1000, 70, None, 0, 64, 64, 64, None, None, None, 0, None) == _lib.MP_EINVAL
    # orthogonalisation
    rows, cols = _arr(i64, [80]), _arr(i64, [90])
    coef = _arr(ctypes.c_double, [3.4445, -4.7750, 2.0315])
    ptr = _arr(ctypes.c_void_p, [1 << 20])
    need = lib.mp_orthogonalize_workspace_bytes(1, rows, cols, 0, 5)
    assert need > 0
    assert lib.mp_orthogonalize_workspace_bytes(1, _arr(i64, [0]), cols, 0, 5) == 0
    assert lib.mp_orthogonalize_workspace_bytes(2, _arr(i64, [64, 3]), _arr(i64, [64, 64]), 0, 5) == 0        # small ones need none
    assert lib.mp_orthogonalize_workspace_bytes(2, _arr(i64, [64, 80]), _arr(i64, [64, 90]), 0, 5) > need     # unless they go with others
    ok = (1, ptr, ptr, rows, cols, 0, 5, coef, 1e-7, 1 << 20, need, None)

    def call(**kw):
        names = ("count", "in", "out", "rows", "cols", "dtype", "steps", "coef", "eps", "ws", "nbytes", "stream")
        a = list(ok)
        for k, v in kw.items():
            a[names.index(k)] = v
        return lib.mp_orthogonalize(*a)
    assert call(nbytes=need - 1) == _lib.MP_EWORKSPACE
    assert call(ws=None) == _lib.MP_EWORKSPACE
    assert call(ws=(1 << 20) + 16) == _lib.MP_EWORKSPACE          # not 256-byte aligned
    assert call(steps=0) == _lib.MP_EINVAL
    assert call(steps=17) == _lib.MP_EUNSUPPORTED
    assert call(dtype=3) == _lib.MP_EUNSUPPORTED
    assert call(eps=-1.0) == _lib.MP_EINVAL
    assert call(coef=None) == _lib.MP_EINVAL
    assert call(coef=_arr(ctypes.c_double, [float("inf"), 0.0, 0.0])) == _lib.MP_EINVAL
    assert call(coef=_arr(ctypes.c_double, [30.0, 0.0, 0.0])) == _lib.MP_EUNSUPPORTED        # the singular values would grow by 30 a step
    assert call(rows=_arr(i64, [-1])) == _lib.MP_EINVAL
    assert call(rows=_arr(i64, [70000]), cols=_arr(i64, [70000])) == _lib.MP_EUNSUPPORTED
    assert call(cols=_arr(i64, [(1 << 21) + 1])) == _lib.MP_EUNSUPPORTED
    assert call(**{"in": _arr(ctypes.c_void_p, [0])}) == _lib.MP_EINVAL
    assert call(count=-1) == _lib.MP_EINVAL
    assert call(count=0) == _lib.MP_OK
    assert lib.mp_muon_step(1, ptr, ptr, None, rows, cols, 0, 0.1, 0.9, 1, 0.0, 1, 5, coef, 1e-7, 1 << 20, need, None) == _lib.MP_EINVAL
    assert lib.mp_muon_step(1, ptr, ptr, ptr, rows, cols, 0, 0.1, 0.9, 1, 0.0, 9, 5, coef, 1e-7, 1 << 20, need, None) == _lib.MP_EINVAL
    # large shapes are accepted as far as the arguments go: the size of the workspace is computed in 64 bits
    assert lib.mp_orthogonalize_workspace_bytes(1, _arr(i64, [40000]), _arr(i64, [40000]), 0, 5) > 1 << 33


def test_operators_refuse_cpu_tensors():
    from maskplanner_amd import ops
    x = torch.zeros(3, 4)
    for call in (lambda: ops.layer_norm(x), lambda: ops.orthogonalize([x]), lambda: ops.orthogonalize(x),
                 lambda: ops.muon_step([x], [x], [x.clone()], lr=0.1)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_layer_norm_module_bookkeeping():
    from maskplanner_amd.layer_norm import LayerNorm
    a, b = LayerNorm((4, 6), eps=1e-3), torch.nn.LayerNorm((4, 6), eps=1e-3)
    assert list(a.state_dict()) == list(b.state_dict()) and all(p.shape == q.shape for p, q in zip(a.parameters(), b.parameters()))
    b.load_state_dict(a.state_dict())
    with pytest.raises(ValueError):
        a(torch.zeros(2, 4, 5))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        a(torch.zeros(2, 4, 6))


def test_segmenter_point_norm_parameters():
    from maskplanner_amd.pointnet2_seg import PointNet2Segmenter_PaintNet_v1, PointNet2Segmenter_v1
    for cls in (PointNet2Segmenter_v1, PointNet2Segmenter_PaintNet_v1):
        batch, layer = cls(), cls(point_norm="layer")
        stats = ("running_mean", "running_var", "num_batches_tracked")
        want = [k for k in batch.state_dict() if not (k.startswith("bn") and k.endswith(stats))]
        assert list(layer.state_dict()) == want
        assert all(batch.state_dict()[k].shape == v.shape for k, v in layer.state_dict().items())
        with pytest.raises(ValueError):
            cls(point_norm="group")


def test_muon_checks_its_parameters():
    from maskplanner_amd.muon import Muon
    w = torch.nn.Parameter(torch.zeros(4, 5))
    for bad in (lambda: Muon([torch.nn.Parameter(torch.zeros(4))]), lambda: Muon([w], lr=-1.0), lambda: Muon([w], momentum=1.0),
                lambda: Muon([w], scale="x"), lambda: Muon([w], weight_decay=-0.1), lambda: Muon([torch.nn.Parameter(torch.zeros(4, 5).double())]),
                lambda: Muon([torch.nn.Parameter(torch.zeros(4, 5).t())])):
        with pytest.raises(ValueError):
            bad()
    opt = Muon([w])
    opt.step()                                    # no gradient: nothing to do
    w.grad = torch.zeros(4, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()


def test_muon_momentum_stays_in_32_bits_through_a_checkpoint():
    from maskplanner_amd.muon import Muon
    w = torch.nn.Parameter(torch.zeros(4, 5, dtype=torch.bfloat16))
    opt = Muon([w], lr=0.03, scale="match_rms")
    opt.state[w]["momentum_buffer"] = torch.full((4, 5), 1.0 + 2.0 ** -20)
    sd = opt.state_dict()
    other = Muon([w])
    other.load_state_dict(sd)
    m = other.state[w]["momentum_buffer"]
    assert m.dtype == torch.float32 and torch.equal(m, opt.state[w]["momentum_buffer"]) and m.data_ptr() != opt.state[w]["momentum_buffer"].data_ptr()
    assert other.param_groups[0]["lr"] == 0.03 and other.param_groups[0]["scale"] == "match_rms"


def test_train_step_refuses_unknown_optimizers():
    from maskplanner_amd.harness import TrainStep
    with pytest.raises(ValueError):
        TrainStep("cuboids", B=2, N=256, device="cpu", optimizer="sgd")
    with pytest.raises(RuntimeError, match="MI355X"):
        TrainStep("cuboids", B=2, N=256, device="cpu", optimizer="muon", hidden_size=(64, 64))


def test_muon_step_finds_shared_memory():
    from maskplanner_amd.ops import _no_overlap
    buf, g = torch.zeros(64, 8), torch.zeros(32, 8)
    p, q, m, n = buf[:16], buf[16:32], buf[32:48], buf[48:]
    _no_overlap([p, q, m, n], [g, g])                       # neighbours in one buffer, one gradient for two parameters
    _no_overlap([p, q, m, n, buf[:0]], [buf[:0], buf[:0]])  # nothing to share
    for written, read in (([p, p, m, n], [g]), ([p, m, m], [g]), ([p, buf[15:31], m, n], [g]), ([p, m], [p]), ([p, m], [buf[40:56]]),
                          ([buf, m], [g]), ([buf[60:], p], [buf[:64]]), ([p, m, n], [g, buf[20:40], g])):
        with pytest.raises(ValueError, match="shares memory"):
            _no_overlap(written, read)


def test_recorded_reductions_have_counters_of_their_own(monkeypatch):
    """Two recordings replayed on two streams at once must not count each other's workgroups (a loss term came out partial)."""
    from maskplanner_amd import ops
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": 7})())
    monkeypatch.setattr(ops, "_REDUCE_COUNTERS", {})
    monkeypatch.setattr(ops, "_RECORDED_COUNTERS", {})
    monkeypatch.setattr(ops, "_COUNTER_POOL", 8)
    d = torch.device("cpu")
    eager = ops._reduce_counter(d)
    assert ops._reduce_counter(d) is eager
    capturing[0] = True
    taken = [ops._reduce_counter(d) for _ in range(10)]           # the last two beyond the pool
    assert len({t.data_ptr() for t in taken + [eager]}) == 11 and all(int(t) == 0 and t.numel() == 1 for t in taken)
    capturing[0] = False
    assert ops._reduce_counter(d) is eager
    capturing[0] = True
    assert ops._reduce_counter(d).data_ptr() not in {t.data_ptr() for t in taken}
