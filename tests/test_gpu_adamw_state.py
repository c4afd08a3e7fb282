"""AdamW's state dictionaries: parameter groups, their settings and the seed go with the moments, to torch.optim.AdamW and back."""
import math

import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu
H32 = 2.0 ** -24
SIZES = [(6, 4), (4,), (300, 5), (300,), (2, 3, 7)]


def leaves(like=None):
    ps = [torch.nn.Parameter(torch.linspace(-1, 1, math.prod(s), device=DEV).view(s)) for s in SIZES]
    for p, q in zip(ps, like or []):
        p.data.copy_(q.data)
    return ps


def give(ps, seed):
    for i, p in enumerate(ps):
        g = torch.Generator().manual_seed(100 * seed + i)
        p.grad = torch.randn(p.shape, generator=g).to(DEV)


def same(ps, qs):
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)


def near(ps, qs, lr, steps=1):
    """Steps of two implementations in f32: 64 half steps of the update (at most about lr), 4 of the parameter."""
    for p, q in zip(ps, qs):
        assert float((p.detach() - q.detach()).abs().max()) <= steps * (lr * 64 * H32 + 4 * H32)


def groups_of(ps, kind):
    decayed, rest = [p for p in ps if p.dim() > 1], [p for p in ps if p.dim() == 1]
    if kind == "torch":
        return [{"params": decayed, "weight_decay": 0.1}, {"params": rest, "weight_decay": 0.0, "lr": 5e-3}]
    return [{"params": decayed, "weight_decay": 0.1}, {"params": rest, "weight_decay": 0.0, "lr_scale": 0.5}]


@pytest.mark.parametrize("bits", [32, 8])
def test_two_groups_move_to_torch_and_back_unmodified(bits):
    """Decays and scales are the state's: the receiving optimisers are built with others."""
    from mqgan_amd.optim import AdamW
    ps = leaves()
    opt = AdamW(groups_of(ps, "own"), lr=1e-2, betas=(0.8, 0.95), eps=1e-6, state_bits=bits)
    for t in range(3):
        give(ps, t)
        opt.step()
    sd = opt.state_dict()
    assert [g["params"] for g in sd["param_groups"]] == [[0, 1, 2], [3, 4]]
    assert [(g["lr"], g["weight_decay"]) for g in sd["param_groups"]] == [(1e-2, 0.1), (5e-3, 0.0)]
    qs = leaves(ps)
    decayed = [q for q in qs if q.dim() > 1]
    theirs = torch.optim.AdamW([{"params": decayed}, {"params": [q for q in qs if q.dim() == 1]}], lr=1.0, weight_decay=0.7)
    theirs.load_state_dict(sd)
    assert [g["weight_decay"] for g in theirs.param_groups] == [0.1, 0.0] and theirs.param_groups[0]["betas"] == (0.8, 0.95)
    rs = leaves(ps)
    two = AdamW([{"params": [r for r in rs if r.dim() > 1]}, {"params": [r for r in rs if r.dim() == 1]}], lr=1.0, weight_decay=0.7, state_bits=bits)
    two.load_state_dict(sd)
    assert two.weight_decays == opt.weight_decays and two.lr_scales == opt.lr_scales and (two.lr, two.betas, two.eps) == (1e-2, (0.8, 0.95), 1e-6)
    for t in range(3, 5):
        for x in (ps, qs, rs):
            give(x, t)
        opt.step()
        two.step()
        same(ps, rs)
        if t == 3:                                       # with 8 bits torch's moments part after a step: the first step's are the same
            theirs.step()
            near(ps, qs, 1e-2)
    if bits == 32:
        give(qs, 4)
        theirs.step()
        near(ps, qs, 1e-2, 2)
        xs = leaves(qs)
        back = AdamW([{"params": [x for x in xs if x.dim() > 1]}, {"params": [x for x in xs if x.dim() == 1]}], lr=3.0)
        back.load_state_dict(theirs.state_dict())        # torch numbers its tensors group by group
        assert back.weight_decays == opt.weight_decays and abs(back.lr - 1e-2) < 1e-15 and back._steps()[0] == [5] * 5
        for x in (xs, qs):
            give(x, 9)
        back.step()
        theirs.step()
        near(xs, qs, 1e-2)


def test_a_state_of_torch_sets_decays_and_rates():
    from mqgan_amd.optim import AdamW
    qs = leaves()
    theirs = torch.optim.AdamW(groups_of(qs, "torch"), lr=1e-2, betas=(0.7, 0.9))
    for t in range(2):
        give(qs, t)
        theirs.step()
    ps = leaves(qs)
    opt = AdamW(groups_of(ps, "own"), lr=9.0)
    opt.load_state_dict(theirs.state_dict())
    assert opt.weight_decays == [0.1] * 3 + [0.0] * 2 and opt.betas == (0.7, 0.9)
    assert abs(opt.lr - 1e-2) < 1e-12 and [round(s, 6) for s in opt.lr_scales] == [1.0] * 3 + [0.5] * 2
    for t in range(2, 4):
        for x in (ps, qs):
            give(x, t)
        opt.step()
        theirs.step()
    near(ps, qs, 1e-2, 2)


@pytest.mark.parametrize("bits", [32, 8])
def test_an_arena_whose_tensors_decay_in_part(bits):
    """The trainer's set-up: the state has a group for what decays and one for the rest, by position in the arena."""
    from mqgan_amd.ddp import FlatArena
    from mqgan_amd.optim import AdamW

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.ParameterList(leaves())
    decays = lambda p: p.dim() > 1  # noqa: E731
    make = lambda **kw: AdamW(FlatArena([Net()], gather=True), decays=decays, state_bits=bits, **kw)  # noqa: E731
    opt = make(lr=1e-2, weight_decay=0.2, seed=6)
    for t in range(2):
        opt.zero_grad()
        give(opt.params, t)
        opt.step()
    sd = opt.state_dict()
    assert [g["params"] for g in sd["param_groups"]] == [[0, 2, 4], [1, 3]]
    assert [g["weight_decay"] for g in sd["param_groups"]] == [0.2, 0.0]
    qs = leaves(opt.params)
    theirs = torch.optim.AdamW([{"params": [qs[i] for i in (0, 2, 4)]}, {"params": [qs[i] for i in (1, 3)]}])
    theirs.load_state_dict(sd)
    two = make(lr=1.0, weight_decay=0.0)
    for p, q in zip(two.params, opt.params):
        p.data.copy_(q.data)
    two.load_state_dict(sd)
    for o in (opt, two):
        o.zero_grad()
        give(o.params, 7)
        o.step()
    give(qs, 7)
    theirs.step()
    same(opt.params, two.params)
    near(opt.params, qs, 1e-2)
    # through torch, whose numbers follow its groups
    three = make(lr=1.0)
    three.load_state_dict(theirs.state_dict())
    assert three._steps()[0] == [3] * 5 and three.weight_decays == opt.weight_decays
    for i, (a, n) in enumerate(zip(three.positions, three._sizes)):
        assert torch.equal(theirs.state[qs[i]]["exp_avg"].reshape(-1), three.moments()[0][a:a + n]) or bits == 8


def test_eight_bits_go_on_bit_for_bit_under_another_seed():
    from mqgan_amd.optim import AdamW
    ps = leaves()
    opt = AdamW(ps, lr=1e-2, state_bits=8, seed=3)
    for t in range(3):
        give(ps, t)
        opt.step()
    qs = leaves(ps)
    two = AdamW(qs, lr=1e-2, state_bits=8, seed=99)
    two.load_state_dict(opt.state_dict())
    for t in range(3, 6):
        for x in (ps, qs):
            give(x, t)
        opt.step()
        two.step()
    same(ps, qs)
    same(opt.moments(), two.moments())


def test_states_of_other_groups_give_lr_and_moments_only():
    from mqgan_amd.ddp import FlatArena
    from mqgan_amd.optim import AdamW
    from mqgan_amd.train import FlatAdam

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.ParameterList(leaves())
    adam = FlatAdam(FlatArena([Net()]), 2e-3)
    adam.exp_avg.fill_(0.25)
    adam.exp_avg_sq.fill_(0.5)
    adam.step_count = 4
    opt = AdamW(FlatArena([Net()]), lr=1.0, weight_decay=0.3, decays=lambda p: p.dim() > 1)
    opt.load_state_dict(adam.state_dict())
    assert opt.lr == 2e-3 and opt.weight_decays == [0.3, 0.0, 0.3, 0.0, 0.3] and opt._steps()[0] == [4] * 5
    m, v = opt.moments()
    for a, n in zip(opt.positions, opt._sizes):
        assert bool((m[a:a + n] == 0.25).all()) and bool((v[a:a + n] == 0.5).all())
    opt.lr = 7e-4
    adam.load_state_dict(opt.state_dict())
    assert adam.lr == 7e-4 and adam.step_count == 4


@pytest.mark.parametrize("kind", ["torch.optim.Adam", "FlatAdam"])
def test_the_decay_of_adam_is_not_taken_for_a_decoupled_one(kind):
    from mqgan_amd.ddp import FlatArena
    from mqgan_amd.optim import AdamW
    from mqgan_amd.train import FlatAdam

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.ParameterList(leaves())
    if kind == "FlatAdam":
        adam = FlatAdam(FlatArena([Net()]), 2e-3, (0.6, 0.8))
        adam.step_count = 1
    else:
        qs = leaves()
        adam = torch.optim.Adam(qs, lr=2e-3, betas=(0.6, 0.8), weight_decay=0.5)
        give(qs, 0)
        adam.step()
    opt = AdamW(leaves(), lr=1.0, weight_decay=0.3)
    opt.load_state_dict(adam.state_dict())
    assert opt.weight_decays == [0.3] * 5 and (opt.lr, opt.betas) == (2e-3, (0.6, 0.8)) and opt._steps()[0] == [1] * 5


def test_a_state_with_one_group_for_all_gives_lr_and_moments():
    """As this class wrote them at first: whatever the groups, one with the largest decay and the lr before scaling."""
    from mqgan_amd.optim import AdamW
    ps = leaves()
    opt = AdamW([{"params": ps, "lr_scale": 0.5}], lr=1e-2, weight_decay=0.1)
    give(ps, 0)
    opt.step()
    sd = opt.state_dict()
    del sd["mqgan_amd_lr"], sd["param_groups"][0]["lr_scale"]
    sd["param_groups"][0].update(lr=3e-2, weight_decay=0.9)
    two = AdamW([{"params": leaves(ps), "lr_scale": 0.5}], lr=1.0, weight_decay=0.1)
    two.load_state_dict(sd)
    assert two.lr == 3e-2 and two.lr_scales == [0.5] * 5 and two.weight_decays == [0.1] * 5
    same(two.moments(), opt.moments())


def test_states_that_do_not_fit_change_nothing():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.optim import AdamW
    ps = leaves()
    opt = AdamW(ps, lr=1e-2, state_bits=8, seed=3)
    give(ps, 0)
    opt.step()
    sd = opt.state_dict()
    kept = [x.clone() for x in opt.moments()]
    group = sd["param_groups"][0]
    short = tuple(c[:256].clone() for c in sd["mqgan_amd_moments8"]["codes"])
    entry = {**sd["state"][0], "exp_avg": torch.ones(3)}
    for bad in ({**sd, "param_groups": [{**group, "amsgrad": True}]}, {**sd, "param_groups": [{**group, "maximize": True}]},
                {**sd, "mqgan_amd_moments8": {**sd["mqgan_amd_moments8"], "codes": short}}, {**sd, "state": {**sd["state"], 0: entry}}):
        bad = {**bad, "mqgan_amd_lr": 5.0}
        with pytest.raises(MqganHipError):
            opt.load_state_dict(bad)
        assert opt.lr == 1e-2 and opt._steps() == ([1] * 5, 1)
        same(opt.moments(), kept)
    two = AdamW([{"params": ps[:2]}, {"params": ps[2:]}], lr=1e-2)
    mixed = two.state_dict()
    mixed["param_groups"][1]["betas"] = (0.5, 0.6)
    with pytest.raises(MqganHipError, match="betas"):
        two.load_state_dict(mixed)
