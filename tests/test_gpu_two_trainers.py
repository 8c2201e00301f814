"""Training steps compared without the noise of training: at a learning rate of 0 the weights stay as they are, so that the run-to-run noise of
atomic sums has nothing to grow in -- the losses of two runs of one seed are the same to the bit, step for step (dropout masks included), and
gradients differ by the order of their sums only: 1e-5 of their norm, or of next to nothing where a following BatchNorm takes the shift out
(norms of 1e-4 beside 1e4).  A partial sum, another trainer's or another step's gradient is off by its own size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def make(seed, **kw):
    from maskplanner_amd.harness import TrainStep
    return TrainStep("cuboids", B=4, N=1024, seed=seed, lr=0.0, **kw)


def gradients(ts):
    return {n: p.grad.clone() for n, p in ts.model.named_parameters() if p.grad is not None}


def close(got, want):
    assert got.keys() == want.keys()
    floor = 1e-6 * max(float(g.norm()) for g in want.values())
    for n, g in want.items():
        assert float((got[n] - g).norm()) <= 1e-3 * float(g.norm()) + floor, n


def test_two_trainers_on_two_streams_each_as_alone():
    """eager steps, the recording and replays of two trainers, interleaved on two streams of one process"""
    steps, seeds = 9, (11, 12)

    def solo(seed, graph):
        ts = make(seed, graph=graph)
        losses = [ts.step().clone() for _ in range(steps)]
        torch.cuda.synchronize()
        ts.check()
        return [float(x) for x in losses], gradients(ts)
    want = {s: solo(s, True) for s in seeds}
    eager, grads = solo(11, False)
    assert eager == want[11][0] and len(set(eager)) == steps           # (every step has dropout masks of its own)
    close(grads, want[11][1])
    streams = {s: torch.cuda.Stream() for s in seeds}
    pair, losses = {}, {s: [] for s in seeds}
    for s in seeds:
        with torch.cuda.stream(streams[s]):
            pair[s] = make(s, graph=True)
    for _ in range(steps):
        for s in seeds:
            with torch.cuda.stream(streams[s]):
                losses[s].append(pair[s].step().clone())
    torch.cuda.synchronize()
    for s in seeds:
        pair[s].check()
        assert pair[s]._graph is not None and [float(x) for x in losses[s]] == want[s][0], s
        close(gradients(pair[s]), want[s][1])


MUON = dict(hidden_size=(128, 128), optimizer="muon")


def momentum(ts):
    return {i: ts.opt.muon.state[p]["momentum_buffer"].clone() for i, p in enumerate(ts.opt.muon.param_groups[0]["params"])}


def test_replayed_muon_steps_see_the_gradients_of_their_own_step():
    """momentum over nine steps of different dropout masks, eager against eager and replayed: a gradient of another step would stay in it"""
    runs = []
    for graph in (False, True):
        ts = make(5, graph=graph, muon={"muon_lr": 0.0}, **MUON)
        losses = [ts.step().clone() for _ in range(9)]
        torch.cuda.synchronize()
        assert (ts._graph is not None) == graph
        runs.append(([float(x) for x in losses], momentum(ts), gradients(ts)))
    assert runs[0][0] == runs[1][0] and len(set(runs[0][0])) == 9
    close(runs[1][1], runs[0][1])
    close(runs[1][2], runs[0][2])
    last = runs[0][2]
    first = make(5, graph=False, muon={"muon_lr": 0.0}, **MUON)
    first.step()
    other = gradients(first)
    assert any(float((other[n] - g).norm()) > 0.1 * float(g.norm()) for n, g in last.items() if n.startswith("sa") and g.ndim > 1)


@pytest.mark.parametrize("graph", [False, True])
def test_muon_steps_of_the_trainer_are_muon_steps(graph):
    """each step's update of the encoder's matrices, to the bit: ops.muon_step on what weights and momentum were before, with the step's gradients"""
    from maskplanner_amd import ops
    ts = make(6, graph=graph, muon={"muon_lr": 0.02, "weight_decay": 0.01}, **MUON)
    ps = ts.opt.muon.param_groups[0]["params"]
    ts.step()
    for k in range(8):
        torch.cuda.synchronize()
        before, m = [p.detach().clone() for p in ps], [ts.opt.muon.state[p]["momentum_buffer"].clone() for p in ps]
        ts.step()
        torch.cuda.synchronize()
        ops.muon_step(before, [p.grad for p in ps], m, lr=0.02, weight_decay=0.01)
        for p, q, n in zip(ps, before, m):
            assert torch.equal(p, q) and torch.equal(ts.opt.muon.state[p]["momentum_buffer"], n), k
    assert (ts._graph is not None) == graph
