"""Codes drawn, kept in use and trained on, as a program uses them together: the quantiser's draw and balance loss under an AdamW step,
draws decoded to spectrograms, and the trainer's AdamW."""
import math

import pytest
import torch

from conftest import load_golden
from gpu_util import DEV, t
from test_gpu_trainstep import make_trainer

pytestmark = pytest.mark.gpu


def test_quantiser_scores_and_their_balance_gradient():
    """Scores against the distances in 64 bits, and the loss's gradient through them to the vectors."""
    from mqgan_amd.quantizer import L2Quantizer
    torch.manual_seed(1)
    K, D, T = 96, 24, 2.5
    q = L2Quantizer(K, D).to(DEV)
    x = torch.randn(4, 17, D, device=DEV, requires_grad=True)
    padded = torch.rand(4, 17, device=DEV) < 0.3
    idx = q.indices(x)
    s = q.scores(x, T)
    x64, c64 = x.detach().double(), q.codebook.double()
    want = (2 * x64 @ c64.t() - c64.square().sum(1)) / T
    # D products and a norm's D squares, each sum rounding at every step: D half steps of the terms' magnitudes
    room = (D + 8) * 2.0 ** -24 * (2 * x64.abs() @ c64.abs().t() + c64.square().sum(1)) / T
    assert float(((s.double() - want).abs() - room).max()) <= 0
    loss, counts = q.balance_loss(x, idx, padded, temperature=T)
    (dx,) = torch.autograd.grad(loss, x)
    y = x64.clone().requires_grad_(True)
    z = ((2 * y @ c64.t() - c64.square().sum(1)) / T)[~padded]
    f = torch.bincount(idx[~padded].long(), minlength=K).double()
    assert torch.equal(counts.long(), f.long())
    ref = K * (f / f.sum() * torch.softmax(z, -1).mean(0)).sum()
    (dy,) = torch.autograd.grad(ref, y)
    assert abs(float(loss.detach()) - float(ref.detach())) <= 1e-5 * float(ref.detach())
    assert float((dx.double() - dy).norm() / dy.norm()) <= 1e-5 and not bool(dx[padded].any())


def test_draws_from_the_quantiser_follow_the_distances():
    from mqgan_amd import ops
    from mqgan_amd.quantizer import L2Quantizer
    torch.manual_seed(2)
    q = L2Quantizer(64, 16).to(DEV)
    x, u = torch.randn(5, 40, 16, device=DEV), torch.rand(5, 40, device=DEV)
    padded = torch.rand(5, 40, device=DEV) < 0.2
    got = q.draw(x, u, temperature=3.0, top_k=4, padded=padded)
    assert got.dtype == torch.int32 and got.shape == (5, 40) and bool((got[padded] == -1).all())
    near = q.scores(x).topk(4, dim=-1).indices
    assert bool((near == got.long()[..., None]).any(-1)[~padded].all())
    assert torch.equal(got, ops.sample_codes(q.scores(x, 3.0), u, top_k=4, padded=padded).int())
    sharp = q.draw(x, u, temperature=1e-4)
    d = torch.cdist(x.double(), q.codebook.double())
    two = d.topk(2, dim=-1, largest=False).values
    clear = (two[..., 1] ** 2 - two[..., 0] ** 2) > 0.01                # 100 temperatures: e^-100 for the second
    assert torch.equal(sharp[clear], q.indices(x)[clear])


@pytest.mark.parametrize("bits", [32, 8])
def test_an_encoder_learns_to_use_its_codebook(bits):
    """An encoder in front of a quantiser, stepped on the balance loss of codes it draws: one step against the 64-bit gradient and the
    formula, then the run goes on (EMA codebook beside it) with everything finite and in range."""
    from mqgan_amd import ops
    from mqgan_amd.nn_base import ConvParams, linear
    from mqgan_amd.optim import AdamW
    from mqgan_amd.quantizer import L2Quantizer
    torch.manual_seed(3)
    enc = ConvParams(16, 12, ()).to(DEV)
    q = L2Quantizer(40, 16, decay=0.9).to(DEV)
    opt = AdamW(list(enc.parameters()), lr=1e-2, weight_decay=0.0, state_bits=bits)
    for step in range(6):
        x = torch.randn(3, 30, 12, device=DEV)
        padded = torch.arange(30, device=DEV)[None] >= torch.tensor([30, 17, 9], device=DEV)[:, None]
        h = linear(x, enc)
        codes = q.draw(h, torch.rand(3, 30, device=DEV), temperature=4.0, padded=padded)
        assert bool(((codes >= 0) & (codes < 40))[~padded].all()) and bool((codes[padded] == -1).all())
        loss, counts = q.balance_loss(h, codes, padded, temperature=4.0)
        assert int(counts.sum()) == int((~padded).sum())
        opt.zero_grad()
        loss.backward()
        if step == 0:
            w = enc.weight.detach().double().requires_grad_(True)
            b = enc.bias.detach().double().requires_grad_(True)
            y = x.double() @ w.t() + b
            c = q.codebook.double()
            p = torch.softmax((2 * y @ c.t() - c.square().sum(1)) / 4.0, -1)[~padded].mean(0)
            ref = 40 * (counts.double() / counts.sum() * p).sum()
            gw, gb = torch.autograd.grad(ref, (w, b))
            assert float((enc.weight.grad.double() - gw).norm() / gw.norm()) <= 1e-4 and float((enc.bias.grad.double() - gb).norm() / gb.norm()) <= 1e-4
            before = enc.weight.detach().clone()
        opt.step(max_norm=1.0)
        if step == 0:                                   # the first step of a bias-corrected average is lr sign(g)
            moved = (before - enc.weight.detach()) / 1e-2
            sure = gw.abs() > gw.abs().max() * 1e-2
            assert float((moved.double() - gw.sign())[sure].abs().max()) <= (1e-3 if bits == 32 else 0.2)
        q.ema_update(h.detach()[~padded], codes[~padded])
        assert all(bool(torch.isfinite(v).all()) for v in (loss.detach(), enc.weight.detach(), q.codebook))


def test_sampled_indices_decode():
    from mqgan_amd.preencoder import PreEncoder
    torch.manual_seed(4)
    m = PreEncoder(mel_channels=16, channels=[16, 16, 24], kernel_sizes=[3, 5], fsq_levels=[8, 5, 5], dropout=0.0, refiner_base_channels=8).to(DEV).eval()
    B, T, V = 2, 21, m.codebook_size + 3                # a token model's head: the codes, then its special tokens
    logits, u = torch.randn(B, T, V, device=DEV), torch.rand(B, T, device=DEV)
    logits[..., m.codebook_size:] = 50.0                # never drawn, however likely
    mask = (torch.arange(T, device=DEV)[None] >= torch.tensor([T, 13], device=DEV)[:, None]).unsqueeze(1)
    idx = m.sample(logits, u, mask, temperature=0.9, top_k=20, top_p=0.95, min_p=0.01)
    assert idx.shape == (B, T) and idx.dtype == torch.int64 and int(idx.max()) < m.codebook_size and int(idx.min()) >= 0
    assert not bool(idx[mask[:, 0]].any())
    top = logits[..., :m.codebook_size].topk(20, dim=-1).indices
    assert bool((top == idx[..., None]).any(-1)[~mask[:, 0]].all())
    mel = m.decode(idx, mask)
    assert mel.shape == (B, T, 16) and bool(torch.isfinite(mel).all())
    assert torch.equal(m.sample(logits, u, temperature=0.0), logits[..., :m.codebook_size].argmax(-1))
    with pytest.raises(ValueError):
        m.sample(logits[..., :50], u)


def _trainer(kind, **training):
    tr = make_trainer(load_golden("g7_trainstep.npz"), False)
    from mqgan_amd.train import WarmupLR
    tr.config["training"] = {**tr.config["training"], "optimizer": kind, **training}
    tr.optimizer_g, tr.optimizer_d = tr._init_optimizers()
    tr.scheduler_g = WarmupLR(tr.optimizer_g, tr.config["training"]["warmup_steps"])
    return tr


@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
def test_trainer_steps_with_adamw_and_resumes(kind, tmp_path):
    g = load_golden("g7_trainstep.npz")
    tr = _trainer(kind, weight_decay=0.1)
    tr.generator.eval()
    assert type(tr.optimizer_g).__name__ == "AdamW" and tr.optimizer_g.state_bits == (8 if kind.endswith("8bit") else 32)
    old = [p.detach().double().clone() for p in tr.arena_g.params]
    lr = tr.optimizer_g.lr
    tr.train_step(t(g["s0/x"]), t(g["lens"]))
    grads = [p.grad for p in tr.arena_g.params]
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in grads if x is not None))
    assert abs(float(tr.optimizer_g.grad_norm()) / norm - 1) < 1e-6
    decayed = 0
    for p, before, x in zip(tr.arena_g.params, old, grads):
        if x is None:                                   # no gradient: neither stepped nor decayed
            assert torch.equal(p.detach().double(), before)
            continue
        c = x.double() * min(1.0, 1.0 / (norm + 1e-6))
        wd = 0.1 if p.dim() > 1 and p.numel() > p.shape[0] else 0.0
        decayed += wd > 0
        want = before * (1 - lr * wd) - lr * c / (c.abs() + 1e-8)
        # f32: two roundings of the parameter; the step itself relative 1e-5 (eps next to a gradient), or 3 % a moment in 8 bits' first rounding:
        # m and v are used before they are rounded, so the first step is exact in both
        assert float((p.detach().double() - want).abs().max()) <= 3 * 2.0 ** -24 * float(before.abs().max()) + 1e-5 * lr
    assert decayed > 5
    tr.config["data"] = {"output_dir": str(tmp_path)}
    tr._save_checkpoint(1)
    from mqgan_amd.train import Trainer
    two = Trainer(dict(tr.config), device=DEV, build_data=False)
    assert two.start_epoch == 2 and type(two.optimizer_g).__name__ == "AdamW"
    two.generator.eval()
    for a in (tr, two):
        a.patch_discriminator.eval()
        a.multibin_discriminator.eval()
        a.epoch = 1
        a.train_step(t(g["s0/x"]), t(g["lens"]))
    # the step's own kernels may add in another order (atomics are not used on this path): weights agree bit for bit
    for p, r in zip(tr.arena_g.params + tr.arena_d.params, two.arena_g.params + two.arena_d.params):
        assert torch.equal(p, r)
    for o, r in ((tr.optimizer_g, two.optimizer_g), (tr.optimizer_d, two.optimizer_d)):
        assert o._steps() == r._steps()
        for a, b in zip(o.moments(), r.moments()):
            assert torch.equal(a, b)


def test_trainer_refuses_an_unknown_optimizer():
    with pytest.raises(ValueError, match="optimizer"):
        _trainer("sgd")
