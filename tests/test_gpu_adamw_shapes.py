"""AdamW takes a gradient for its parameter's elements in their order, and no other of the same size."""
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu


def test_a_gradient_of_another_shape_is_refused():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.optim import AdamW
    p = torch.zeros(6, 4, device=DEV)
    opt = AdamW([p, torch.zeros((), device=DEV)])
    one = torch.ones((), device=DEV)
    for shape in ((4, 6), (2, 3, 4), (6, 4, 1), (6, 5), (24, 1)):
        with pytest.raises(MqganHipError, match="gradient 0"):
            opt.step(grads=[torch.ones(shape, device=DEV), one])
    with pytest.raises(MqganHipError, match="gradient 1"):
        opt.step(grads=[p, torch.ones(1, 1, device=DEV)])
    assert not bool(p.any()) and opt._steps() == ([0, 0], 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_flat_and_transposed_gradients_step_alike(dtype):
    from mqgan_amd.optim import AdamW
    g = torch.randn(6, 4, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    ps = [torch.zeros(6, 4, device=DEV) for _ in range(4)]
    given = [g, g.reshape(-1), g.t().contiguous().t(), torch.cat([g, g], 1)[:, :4]]
    for p, x in zip(ps, given):
        AdamW([p], lr=0.1).step(grads=[x])
    assert bool(ps[0].all()) and all(torch.equal(p, ps[0]) for p in ps)


def test_a_parameter_that_was_reshaped_takes_gradients_of_its_new_shape():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(6, 4, device=DEV))
    opt = AdamW([p], lr=0.1)
    p.data = p.data.view(8, 3)
    opt.step(grads=[torch.ones(8, 3, device=DEV)])
    assert bool((p != 0).all())
    with pytest.raises(MqganHipError):
        opt.step(grads=[torch.ones(4, 6, device=DEV)])
