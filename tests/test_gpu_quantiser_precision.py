"""L2Quantizer's scores, draws and balance loss inside bf16 layers: the distances stay exact f32 products, as in the nearest-code search."""
import contextlib

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def layers(name, storage):
    from mqgan_amd import ops
    with ops.conv_precision(name), ops.act_storage(storage):
        yield


MODES = [("f32", False), ("bf16", False), ("bf16", True), ("f32x3", False)]


@pytest.mark.parametrize("rows,D", [(40, 24), (2500, 64)])
@pytest.mark.parametrize("mode", MODES, ids=str)
def test_scores_and_their_gradient_are_f32_in_every_mode(mode, rows, D):
    from mqgan_amd.quantizer import L2Quantizer
    torch.manual_seed(1)
    K, T = 128, 0.5
    q = L2Quantizer(K, D).to(DEV)
    x = torch.randn(rows, D, device=DEV, requires_grad=True)
    idx = q.indices(x)
    with layers(*mode):
        s = q.scores(x, T)
        loss, counts = q.balance_loss(x, idx, temperature=T)
        (dx,) = torch.autograd.grad(loss, x)
    x64, c64 = x.detach().double(), q.codebook.double()
    want = (2 * x64 @ c64.t() - c64.square().sum(1)) / T
    # D products and a norm's D squares, each sum rounding at every step: D half steps of the terms' magnitudes
    room = (D + 8) * 2.0 ** -24 * (2 * x64.abs() @ c64.abs().t() + c64.square().sum(1)) / T
    assert s.dtype == torch.float32 and float(((s.double() - want).abs() - room).max()) <= 0
    y = x64.clone().requires_grad_(True)
    f = torch.bincount(idx.long(), minlength=K).double()
    ref = K * (f / f.sum() * torch.softmax((2 * y @ c64.t() - c64.square().sum(1)) / T, -1).mean(0)).sum()
    (dy,) = torch.autograd.grad(ref, y)
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-5 * float(ref.detach())
    # an error of the scores is one of the shares: room at its largest, relative, in every term of the gradient
    assert float((dx.double() - dy).norm() / dy.norm()) <= 4 * float(room.max()) + 1e-5


@pytest.mark.parametrize("mode", MODES, ids=str)
def test_sharp_draws_are_the_nearest_codes_in_every_mode(mode):
    from mqgan_amd.quantizer import L2Quantizer
    torch.manual_seed(2)
    q = L2Quantizer(256, 64).to(DEV)
    x, u = torch.randn(2500, 64, device=DEV), torch.rand(2500, device=DEV)
    with layers(*mode):
        sharp = q.draw(x, u, temperature=1e-4)
    two = torch.cdist(x.double(), q.codebook.double()).topk(2, dim=-1, largest=False).values
    clear = (two[..., 1] ** 2 - two[..., 0] ** 2) > 0.01                # 100 temperatures: e^-100 for the second
    assert int(clear.sum()) > 2000 and torch.equal(sharp[clear], q.indices(x)[clear])
