"""What a cloud's segmentation depends on, with a layer norm and with the reference's BatchNorm in the point head."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def clouds(seed):
    return torch.randn(1, 3, 700, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def run(model, first, second):
    """the first cloud's result in a batch of two; sampling starts fixed"""
    from maskplanner_amd.pointnet2_utils import fps_start_override
    with torch.no_grad(), fps_start_override([torch.zeros(2, dtype=torch.long)] * 2):
        return model(torch.cat([first, second]))[0]


@pytest.mark.parametrize("cls", ["PointNet2Segmenter_v1", "PointNet2Segmenter_PaintNet_v1"])
def test_neighbours_of_a_cloud(cls):
    """Rows of a product and of a norm do not meet: with batches of one shape the results are the same to the bit, or they depend on the neighbour."""
    from maskplanner_amd import pointnet2_seg
    a, b, c = (clouds(s) for s in (1, 2, 3))
    for norm in ("layer", "batch"):
        torch.manual_seed(0)
        model = getattr(pointnet2_seg, cls)(point_norm=norm).cuda()
        model.eval()
        assert torch.equal(run(model, a, b), run(model, a, c)), norm                # evaluation: neither norm looks at the batch
        model.train()
        assert not torch.equal(run(model, a, b), run(model, a, c)), norm            # training: the encoder's BatchNorm does, with either
        # the head alone: the encoder's features of the first cloud held fixed, the second one's its own
        fixed = torch.randn(1, 1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))

        def hold(mod, args, out):
            points = out[1].clone()
            points.reshape(2, 1024)[0] = fixed[0]
            return (out[0], points)
        handle = model.sa3.register_forward_hook(hold)
        same = torch.equal(run(model, a, b), run(model, a, c))
        handle.remove()
        assert same == (norm == "layer"), norm
