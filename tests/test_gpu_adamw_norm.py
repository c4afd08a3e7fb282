"""AdamW.grad_norm(): the norm of the last step that clipped, with that step's scale, whatever was stepped or replayed since."""
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu
H32 = 2.0 ** -24


def check(opt, norm):
    got = opt.grad_norm()
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - norm) <= 2 * H32 * norm          # squares and their sum in 64 bits, rounded once


def test_the_norm_keeps_the_scale_it_was_taken_with():
    from mqgan_amd.optim import AdamW
    p = torch.zeros(1000, device=DEV)
    opt = AdamW([p])
    g = torch.full((1000,), 0.5, device=DEV)
    norm = 0.5 * 1000 ** 0.5
    assert float(opt.grad_norm()) == 0.0
    opt.step(max_norm=1.0, grads=[g])
    check(opt, norm)
    opt.step(grad_scale=0.5, grads=[g * 3])                  # no clipping: no norm
    check(opt, norm)
    opt.step(max_norm=1.0, grad_scale=-0.25, grads=[g])
    check(opt, norm / 4)
    opt.step(grads=[g])
    check(opt, norm / 4)


def test_the_norm_of_a_replayed_step():
    from mqgan_amd.optim import AdamW
    p = torch.zeros(1000, device=DEV)
    opt = AdamW([p])
    g = torch.full((1000,), 0.5, device=DEV)
    norm = 0.5 * 1000 ** 0.5
    opt.step(max_norm=1.0, grad_scale=0.5, grads=[g])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(max_norm=1.0, grad_scale=0.5, grads=[g])
    for r in range(3):
        opt.step(max_norm=1.0, grad_scale=2.0, grads=[g])
        check(opt, norm * 2)
        graph.replay()
        check(opt, norm / 2)
