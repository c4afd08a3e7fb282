"""AdamW under data parallelism on one GPU: two ranks whose gradients differ in which tensors they reach, against one process, bit for bit."""
import threading

import pytest
import torch

from conftest import load_golden
from gpu_util import DEV
from test_gpu_dp import _Shared, _trainer, make_comm

pytestmark = pytest.mark.gpu


def ranks(fn, world=2):
    """fn(rank, communicator) in one thread a rank, which take turns and meet in every sum; the results."""
    shared = _Shared(world)
    got, errors = [None] * world, []

    def main(r):
        shared.run.acquire()
        try:
            torch.cuda.set_device(0)
            got[r] = fn(r, make_comm(shared, r))
        except BaseException as e:               # noqa: BLE001
            errors.append(e)
        finally:
            shared.run.release()
    threads = [threading.Thread(target=main, args=(r,)) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    return got


class Branches(torch.nn.Module):
    """First `a`; behind it `b` on the rank that takes it; `never` has no consumer."""

    def __init__(self):
        super().__init__()
        self.a = torch.nn.Parameter(torch.linspace(-1, 1, 5000).view(50, 100))
        self.b = torch.nn.Parameter(torch.linspace(1, 2, 777))
        self.never = torch.nn.Parameter(torch.full((300,), 3.0))

    def forward(self, x, whole):
        y = (self.a * x).pow(2).sum()
        return y + (self.b * x.sum()).pow(2).sum() if whole else y


# per step: who takes `b`
STEPS = [(True, False), (True, True), (False, False), (False, True)]


@pytest.mark.parametrize("bits", [32, 8])
def test_two_ranks_stay_equal_where_one_lacks_a_gradient(bits):
    from mqgan_amd.ddp import FlatArena, GradReducer
    from mqgan_amd.optim import AdamW
    x = [[torch.randn(50, 100, generator=torch.Generator().manual_seed(10 * s + r)).to(DEV) for r in range(2)] for s in range(len(STEPS))]

    def run(rank, comm):
        net = Branches().to(DEV)
        arena = FlatArena([net], gather=True)
        opt = AdamW(arena, lr=1e-2, weight_decay=0.1, state_bits=bits, seed=4)
        red = GradReducer(arena, comm=comm)
        norms, sums = [], []
        for s, who in enumerate(STEPS):
            opt.zero_grad()
            red.start()
            net(x[s][rank], who[rank]).backward()
            red.finish()
            opt.step(max_norm=0.5)
            norms.append(float(opt.grad_norm()))
            sums.append(arena.flat_grad.clone())
        return [p.detach().clone() for p in arena.params], opt.moments(), opt._steps(), norms, sums
    (p0, m0, s0, n0, sums), (p1, m1, s1, n1, _) = ranks(run)
    assert s0 == s1 and n0 == n1 and s0[0] == [4, 3, 0]      # b: three of four steps; never: none
    for a, b in zip(p0 + list(m0), p1 + list(m1)):
        assert torch.equal(a, b)
    assert bool((p0[2] == 3.0).all())                        # no gradient anywhere: not decayed either

    # one process on the summed gradients, whose optimiser is told by None what has no gradient
    net = Branches().to(DEV)
    ps = list(net.parameters())
    one = AdamW(ps, lr=1e-2, weight_decay=0.1, state_bits=bits, seed=4)
    arena = FlatArena([Branches()], gather=True)             # for its offsets
    for s, who in enumerate(STEPS):
        views = [sums[s][o:o + p.numel()].view_as(p) for p, o in zip(ps, arena.offsets)]
        one.step(max_norm=0.5, grads=[views[0], views[1] if any(who) else None, None])
    for a, b in zip(p0 + list(m0), ps + list(one.moments())):
        assert torch.equal(a, b.detach())
    assert one._steps()[0] == s0[0]


@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
def test_trainer_ranks_with_adamw_equal_the_global_batch(kind):
    """Two Trainers on the halves of a ragged batch against one on the whole of it: what no rank has a gradient for stays as it was in both."""
    import numpy as np
    from mqgan_amd.train import WarmupLR, synthetic_mel
    g = load_golden("g7_trainstep.npz")
    xs = torch.from_numpy(np.stack([synthetic_mel(40, 16, 500 + b) for b in range(4)])).to(DEV)
    lens = torch.tensor([40, 23, 31, 17], dtype=torch.int32, device=DEV)
    for b in range(4):
        xs[b, int(lens[b]):] = 0.0

    def make(comm=None):
        tr = _trainer(g, False, comm)
        tr.config["training"] = {**tr.config["training"], "optimizer": kind, "weight_decay": 0.1}
        tr.optimizer_g, tr.optimizer_d = tr._init_optimizers()
        tr.scheduler_g = WarmupLR(tr.optimizer_g, tr.config["training"]["warmup_steps"])
        return tr
    ref = make()
    before = [p.detach().clone() for p in ref.arena_g.params]
    ref.train_step(xs, lens)
    absent = [i for i, p in enumerate(ref.arena_g.params) if p.grad is None]
    assert absent

    def run(rank, comm):
        tr = make(comm)
        tr.train_step(xs[2 * rank:2 * rank + 2].contiguous(), lens[2 * rank:2 * rank + 2].contiguous())
        return tr
    two = ranks(run)
    for name in ("arena_g", "arena_d"):
        a, b, r = (getattr(t, name).flat_param for t in (*two, ref))
        assert torch.equal(a, b)
        # a first step moves a weight by lr times the sign of its gradient, so gradients that round apart about 0 move apart: few, and by 2 lr
        off = (a - r).abs()
        assert float(off.max()) <= 2.1 * max(two[0].optimizer_g.lr, two[0].optimizer_d.lr) and float((off > 1e-6).float().mean()) < 0.02
    for i in absent:
        assert torch.equal(two[0].arena_g.params[i].detach(), before[i]) and torch.equal(ref.arena_g.params[i].detach(), before[i])
    assert two[0].optimizer_g._steps() == two[1].optimizer_g._steps() == ref.optimizer_g._steps()
