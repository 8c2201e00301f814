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
