"""mqgan_amd.optim.AdamW against the formulas in 64 bits, its 8-bit moments bit for bit against the format, and the life of a state."""
import math

import numpy as np
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu
H32 = 2.0 ** -24                     # half a step of f32, relative
SIZES = [1, 3, 255, 256, 257, 1024, 4096, 4097, 10007]


def _leaves(sizes, seed=0, unaligned=False):
    """Parameters (views one element off 16-byte alignment where asked) with one guard value before and behind each."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        buf = torch.full((n + 12,), 7.25, device=DEV)
        o = 5 if unaligned else 4
        buf[o:o + n] = (torch.randn(n, generator=g) * 0.1).to(DEV)
        out.append((buf, buf[o:o + n], o))
    return out


def _grads(sizes, seed, dtype=torch.float32, scale=1e-2):
    g = torch.Generator().manual_seed(1000 + seed)
    return [(torch.randn(n, generator=g) * scale * 10.0 ** (i % 3 - 1)).to(dtype).to(DEV) for i, n in enumerate(sizes)]


def _ref_step(p, m, v, g, t, lr, b1, b2, eps, wd, coef):
    g = g * coef
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - lr * wd * p - lr / (1 - b1 ** t) * m / (torch.sqrt(v / (1 - b2 ** t)) + eps), m, v


def _near(got, want, bound, what):
    off = (got.double().cpu() - want).abs()
    worst = float((off - bound).max())
    assert worst <= 0, f"{what}: off by {float(off.max()):.3e}, {worst:.3e} over the bound"


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("unaligned", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("max_norm,grad_scale", [(0.0, 1.0), (0.05, 0.5), (1e6, -1.0)])
def test_step_follows_the_formula(grad, unaligned, max_norm, grad_scale):
    from mqgan_amd.optim import AdamW
    leaves = _leaves(SIZES, 1, unaligned)
    ps = [x[1] for x in leaves]
    cut = len(SIZES) // 2
    lr, b1, b2, eps = 3e-3, 0.9, 0.99, 1e-8
    opt = AdamW([{"params": ps[:cut], "weight_decay": 0.1}, {"params": ps[cut:], "lr_scale": 0.5}], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0)
    ref = [(p.double().cpu(), torch.zeros(p.numel(), dtype=torch.float64), torch.zeros(p.numel(), dtype=torch.float64)) for p in ps]
    for t in range(1, 4):
        gs = _grads(SIZES, 10 * t, grad)
        if unaligned:
            gs = [torch.cat([g.new_zeros(1), g])[1:] for g in gs]
        opt.step(max_norm=max_norm, grad_scale=grad_scale, grads=gs)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in gs)) * abs(grad_scale)
        coef = grad_scale * (min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0)
        if max_norm:
            assert abs(float(opt.grad_norm()) - norm) <= 4 * H32 * norm
        m_all, v_all = opt.moments()
        for i, (p, g) in enumerate(zip(ps, gs)):
            rate, wd = (lr, 0.1) if i < cut else (lr * 0.5, 0.0)
            g64 = g.double().cpu()
            old_p, old_m, old_v = ref[i]
            p64, m64, v64 = _ref_step(old_p, old_m, old_v, g64, t, rate, b1, b2, eps, wd, coef)
            at = opt.positions[i]
            # m: the factor, the product, the difference, its product and the sum round once each, t steps add up; v likewise (six roundings)
            em = t * 6 * H32 * (old_m.abs() + (g64 * coef).abs() + m64.abs())
            ev = t * 7 * H32 * (old_v + v64 + (1 - b2) * (g64 * coef) ** 2)
            _near(m_all[at:at + p.numel()], m64, em + 1e-44, f"step {t} tensor {i} exp_avg")
            _near(v_all[at:at + p.numel()], v64, ev + 1e-44, f"step {t} tensor {i} exp_avg_sq")
            # the update: m's and half of v's error, six roundings (both factors, product, sum, two products), and one ulp - two half steps -
            # each of the root and the reciprocal; p: two roundings a step
            upd = rate / (1 - b1 ** t) * m64.abs() / (torch.sqrt(v64 / (1 - b2 ** t)) + eps)
            e_upd = rate / (1 - b1 ** t) * em / (torch.sqrt(v64 / (1 - b2 ** t)) + eps) + upd * (ev / v64.clamp(min=1e-60) + 10 * H32)
            _near(p, p64, 3 * H32 * (old_p.abs() + p64.abs() + upd) + e_upd, f"step {t} tensor {i} parameter")
            ref[i] = (p.double().cpu(), m_all[at:at + p.numel()].double().cpu(), v_all[at:at + p.numel()].double().cpu())
    for buf, p, o in leaves:                          # the neighbours of every parameter stay as they were
        assert bool((buf[:o] == 7.25).all()) and bool((buf[o + p.numel():] == 7.25).all())


# ----------------------------------------------------------------------------- 8-bit moments, restated in numpy
def np_mix(x):
    x = np.asarray(x, np.uint32)
    x = x ^ (x >> np.uint32(16))
    x = x * np.uint32(0x7FEB352D)
    x = x ^ (x >> np.uint32(15))
    x = x * np.uint32(0x846CA68B)
    return x ^ (x >> np.uint32(16))


def np_words(n, seed, calls):
    s = (seed + calls * 0xD1B54A32D192ED03) & (2 ** 64 - 1)
    lo, hi = np.uint32(s & 0xFFFFFFFF), np.uint32(s >> 32)
    with np.errstate(over="ignore"):
        k0 = lo ^ np_mix(hi ^ np.uint32(0x85EBCA6B))
        k1 = np_mix(hi + np_mix(lo ^ np.uint32(0xC2B2AE35)))
        return np_mix(np.arange(n, dtype=np.uint32) ^ k0) + k1


def np_encode(x, ebits, rnd=None):
    b = (x.view(np.uint32) & 0x7FFFFFFF).astype(np.int64).reshape(-1, 256)
    top = np.where(b < 0x7F800000, b, 0).max(1) >> 23
    base = np.maximum(0, top + 1 - (2 ** ebits - 1))
    add = 0x7FFFF + ((b >> 20) & 1) if rnd is None else rnd.astype(np.int64).reshape(-1, 256) << 4
    most = 2 ** (ebits + 3)
    c = ((b + add) >> 20) - 8 * base[:, None]
    c = np.where(c < 1, np.where(b > 0, 1, 0) if ebits == 5 else 0, c)
    c = np.where(b >= 0x7F800000, np.where(b == 0x7F800000, most - 2, most - 1), c)
    if ebits == 4:
        c = c | np.where((np.signbit(x).reshape(-1, 256)) & (c > 0), 128, 0)
    return c.astype(np.uint8).reshape(-1), base.astype(np.uint8)


def np_decode(c, base, ebits):
    most = 2 ** (ebits + 3)
    c = c.astype(np.int64).reshape(-1, 256)
    k = c & (most - 1)
    b = np.where(k > 0, (k + 8 * base.astype(np.int64)[:, None]) << 20, 0)
    b = np.where(k >= most - 2, np.where(k == most - 2, 0x7F800000, 0x7FC00000), b)
    if ebits == 4:
        b = b | ((c & 0x80) << 24)
    return b.astype(np.uint32).view(np.float32).reshape(-1)


def test_eight_bit_steps_are_the_format_bit_for_bit():
    """Codes and bases after each of five steps equal numpy's f32 arithmetic on the decoded moments and the hash's bits."""
    from mqgan_amd.optim import AdamW
    f = np.float32
    ps = [x[1] for x in _leaves(SIZES, 2)]
    opt = AdamW(ps, lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=77)
    total = opt.positions[-1]
    rows = total // 256
    mc, mb, vc, vb = np.zeros(total, np.uint8), np.zeros(rows, np.uint8), np.zeros(total, np.uint8), np.zeros(rows, np.uint8)
    for t in range(1, 6):
        gs = _grads(SIZES, 100 + t, scale=10.0 ** (t - 4))
        opt.step(grads=gs)
        g = np.zeros(total, f)
        for a, x in zip(opt.positions, gs):
            g[a:a + x.numel()] = x.cpu().numpy()
        m, v = np_decode(mc, mb, 4), np_decode(vc, vb, 5)
        m = m + (g - m) * f(1 - 0.9)
        v = v * f(0.999) + f(1 - 0.999) * g * g
        w = np_words(total, 77, t)
        mc, mb = np_encode(m, 4, w >> np.uint32(16))
        vc, vb = np_encode(v, 5, w & np.uint32(0xFFFF))
        for got, want, what in ((opt.exp_avg, mc, "m"), (opt._bases[0], mb, "m base"), (opt.exp_avg_sq, vc, "v"), (opt._bases[1], vb, "v base")):
            d = got.cpu().numpy() != want
            assert not d.any(), f"step {t}: {int(d.sum())} of {d.size} {what} differ, first at {int(d.argmax())}"
    dm, dv = opt.moments()
    assert np.array_equal(dm.cpu().numpy(), np_decode(mc, mb, 4)) and np.array_equal(dv.cpu().numpy(), np_decode(vc, vb, 5))
    bm, bv = opt.moments(torch.bfloat16)
    assert torch.equal(bm.float(), dm) and torch.equal(bv.float(), dv)


def test_format_holds_specials_and_its_whole_range():
    from mqgan_amd.optim import AdamW
    r = np.random.RandomState(3)
    x = np.zeros((12, 256), np.float32)
    x[0] = r.randn(256)
    x[1, :4] = [np.inf, -np.inf, np.nan, 1.0]
    x[2] = 2.0 ** np.arange(-149.0, 107.0).clip(-149, 100)            # denormals to 2^100 in one group
    x[3, 0] = 3.4028234e38
    x[4, 7] = 1.4e-45
    x[5] = 1e-40 * r.randn(256)
    x[6] = np.float32(1.9999999) * 2.0 ** r.randint(-40, 0, 256)
    x[7] = -np.abs(r.randn(256)) * 10.0 ** r.uniform(-12, 0, 256)
    x[8] = -0.0
    x[9:] = r.randn(3, 256) * 10.0 ** r.uniform(-30, 30, (3, 1))
    m, v = x.reshape(-1).astype(np.float32), np.abs(x).reshape(-1).astype(np.float32)
    opt = AdamW([torch.zeros(m.size, device=DEV)], state_bits=8)
    opt.load_moments(torch.from_numpy(m).to(DEV), torch.from_numpy(v).to(DEV))
    (mc, mb), (vc, vb) = np_encode(m, 4), np_encode(v, 5)
    assert np.array_equal(opt.exp_avg.cpu().numpy(), mc) and np.array_equal(opt._bases[0].cpu().numpy(), mb)
    assert np.array_equal(opt.exp_avg_sq.cpu().numpy(), vc) and np.array_equal(opt._bases[1].cpu().numpy(), vb)
    dm, dv = (a.cpu().numpy().reshape(12, 256) for a in opt.moments())
    np.testing.assert_array_equal(dm[1, :4], [np.inf, -np.inf, np.nan, 1.0])
    np.testing.assert_array_equal(dv[1, :4], [np.inf, np.inf, np.nan, 1.0])
    for d, want, span in ((dm, x, 14), (dv, np.abs(x), 30)):           # to nearest: 2^-4 relative over `span` binades under the largest
        for row in (0, 6, 9, 10, 11):
            big = np.abs(want[row]).max()
            fine = np.abs(want[row]) >= big * 2.0 ** -(span - 1)
            assert (np.abs(d[row] - want[row])[fine] <= 2.0 ** -4 * np.abs(want[row])[fine]).all()
    assert (dv[np.abs(x) > 0] > 0).all(), "a positive second moment became 0"


def test_random_rounding_lets_a_slow_average_move():
    """Constant gradients with g^2 = 4 v0: in 400 steps v goes to v0 (4 - 3 b2^400).  Each rounding is unbiased, so the mean over 65536 elements
    follows; one step's noise is at most the root of (change x step) = sqrt(0.003 / 8) of v, 400 of them at most 20 times that: 39 % an
    element, 0.15 % the mean.  To nearest nothing would move (0.3 % a step against 3-6 % half a step)."""
    from mqgan_amd.optim import AdamW
    n = 65536
    p = torch.zeros(n, device=DEV)
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), state_bits=8, seed=5)
    v0 = 1.0 + torch.rand(n, generator=torch.Generator().manual_seed(1)).to(DEV)
    opt.load_moments(torch.zeros(n, device=DEV), v0, step=0)
    v0 = opt.moments()[1]
    g = 2 * v0.sqrt()
    for _ in range(400):
        opt.step(grads=[g])
    got = float((opt.moments()[1] / v0).double().mean())
    want = 4 - 3 * 0.999 ** 400
    assert abs(got / want - 1) < 0.01, (got, want)


def test_a_poisoned_gradient_stays_with_its_element():
    from mqgan_amd.optim import AdamW
    for bits in (32, 8):
        p = torch.ones(600, device=DEV)
        opt = AdamW([p], lr=0.1, state_bits=bits)
        g = torch.full((600,), 0.5, device=DEV)
        g[17], g[300] = float("nan"), float("inf")
        opt.step(grads=[g])
        bad = ~torch.isfinite(p)
        assert bad.nonzero().reshape(-1).tolist() == [17, 300], bits
        m, v = opt.moments()
        assert bool(torch.isnan(m[17])) and bool(torch.isinf(m[300])) and bool(torch.isfinite(m[:17]).all()) and bool(torch.isfinite(v[301:]).all())


def test_many_tensors_take_more_than_one_launch_and_absent_gradients_are_left_out():
    from mqgan_amd.optim import AdamW
    for bits in (32, 8):
        n = 1000
        sizes = [1 + (i * 37) % 700 for i in range(n)]
        ps = [torch.ones(s, device=DEV) for s in sizes]
        opt = AdamW(ps, lr=0.01, weight_decay=0.0, state_bits=bits)
        for t in range(2):
            gs = [None if (i % 7 == 3 and t == 0) else torch.full((s,), 1.0 if i % 2 else -2.0, device=DEV) for i, s in enumerate(sizes)]
            opt.step(max_norm=1e9, grads=gs)
            total = sum(s * (1.0 if i % 2 else 4.0) for i, s in enumerate(sizes) if gs[i] is not None)
            assert abs(float(opt.grad_norm()) ** 2 / total - 1) < 1e-6
        steps, calls = opt._steps()
        assert calls == 2 and steps == [1 if i % 7 == 3 else 2 for i in range(n)]
        for i, p in enumerate(ps):                     # a constant gradient's bias-corrected step is lr, rounding of the moments apart
            want = 1 - (0.01 if i % 7 == 3 else 0.02) * (1 if i % 2 else -1)
            assert float((p - want).abs().max()) <= (1e-6 if bits == 32 else 0.02 * 0.13), (bits, i)


def test_no_gradient_at_all_changes_nothing():
    from mqgan_amd.optim import AdamW
    p, empty = torch.ones(300, device=DEV), torch.zeros(0, device=DEV)
    opt = AdamW([p, empty], lr=0.1, weight_decay=0.5)
    opt.step(grads=[None, None])
    opt.step(max_norm=1.0, grads=[None, empty])
    assert bool((p == 1).all()) and opt._steps() == ([0, 0], 2) and float(opt.grad_norm()) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_counts_on(bits):
    """Replays against the same steps taken eagerly, with eager work of the program between them: bit for bit."""
    from mqgan_amd.optim import AdamW
    sizes = [5, 300, 5000]

    def fresh():
        ps = [torch.linspace(-1, 1, s, device=DEV) for s in sizes]
        return ps, AdamW(ps, lr=1e-2, state_bits=bits, seed=9)
    ps, opt = fresh()
    qs, ref = fresh()
    gs = _grads(sizes, 5)
    opt.step(max_norm=0.5, grads=gs)
    ref.step(max_norm=0.5, grads=gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(max_norm=0.5, grads=gs)
    for r in range(4):
        for g, new in zip(gs, _grads(sizes, 50 + r)):
            g.copy_(new)
        graph.replay()
        ref.step(max_norm=0.5, grads=gs)
        assert float(torch.ones(1000, device=DEV).sum()) == 1000.0
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q), r
        for a, b in zip(opt.moments(), ref.moments()):
            assert torch.equal(a, b), r
    assert opt._steps() == ref._steps() == ([5, 5, 5], 5)


def test_capture_refuses_a_parameter_that_moved():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(64, device=DEV))
    opt = AdamW([p])
    g = torch.ones(64, device=DEV)
    opt.step(grads=[g])
    p.data = torch.ones(64, device=DEV) * 2
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(MqganHipError, match="moved"):
        with torch.cuda.graph(graph):
            opt.step(grads=[g])
    opt.step(grads=[g])                                # eagerly the table is made anew
    assert float(p.detach().max()) < 2


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_on_bit_for_bit_and_moves_between_optimisers(bits):
    from mqgan_amd.optim import AdamW
    sizes = [(3, 5), (257,), (40, 30)]
    make = lambda: [torch.nn.Parameter(torch.linspace(-1, 1, math.prod(s), device=DEV).view(s)) for s in sizes]  # noqa: E731
    ps = make()
    opt = AdamW(ps, lr=1e-2, state_bits=bits, seed=3)

    def steps(o, p, ts):
        for t in ts:
            g = _grads([x.numel() for x in p], t)
            for x, y in zip(p, g):
                x.grad = y.view_as(x)
            o.step(max_norm=1.0)
    steps(opt, ps, (1, 2, 3))
    qs = make()
    for p, q in zip(ps, qs):
        q.data.copy_(p.data)
    two = AdamW(qs, lr=1e-2, state_bits=bits, seed=3)
    two.load_state_dict(opt.state_dict())
    steps(opt, ps, (4, 5))
    steps(two, qs, (4, 5))
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    for a, b in zip(opt.moments(), two.moments()):
        assert torch.equal(a, b)
    # torch.optim.AdamW takes the state and takes the same next step
    rs = make()
    for p, r in zip(ps, rs):
        r.data.copy_(p.data)
    theirs = torch.optim.AdamW(rs, lr=1e-2, weight_decay=0.01)
    sd = opt.state_dict()
    theirs.load_state_dict({"state": sd["state"], "param_groups": [{**theirs.state_dict()["param_groups"][0]}]})
    g = _grads([x.numel() for x in ps], 6)
    for p, r, x in zip(ps, rs, g):
        p.grad, r.grad = x.view_as(p), x.view_as(r).clone()
    opt.step()
    theirs.step()
    for p, r in zip(ps, rs):
        assert float((p - r).abs().max()) <= 1e-2 * 64 * H32 + 4 * H32


def test_gradients_default_to_the_parameters_own_and_may_lie_strided():
    from mqgan_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(6, 4, device=DEV))
    q = torch.nn.Parameter(torch.zeros(6, 4, device=DEV))
    g = torch.arange(24.0, device=DEV).view(4, 6)
    a, b = AdamW([p], lr=0.1), AdamW([q], lr=0.1)
    p.grad = g.t()
    a.step()
    b.step(grads=[g.t().contiguous()])
    assert torch.equal(p, q) and float(p.detach().abs().max()) > 0
    a.zero_grad()
    assert p.grad is None


def test_a_step_on_another_stream():
    from mqgan_amd.optim import AdamW
    p, q = torch.ones(100_000, device=DEV), torch.ones(100_000, device=DEV)
    g = torch.randn(100_000, device=DEV)
    a, b = AdamW([p], state_bits=8), AdamW([q], state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step(max_norm=1.0, grads=[g])
    torch.cuda.current_stream().wait_stream(side)
    b.step(max_norm=1.0, grads=[g])
    assert torch.equal(p, q)


def test_refusals():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.optim import AdamW
    p = torch.zeros(8, device=DEV)
    for bad in (lambda: AdamW([]), lambda: AdamW([p], state_bits=16), lambda: AdamW([p], lr=-1.0), lambda: AdamW([p], betas=(0.9, 1.0)),
                lambda: AdamW([p, p]), lambda: AdamW([{"params": [p], "momentum": 1}]), lambda: AdamW([p], weight_decay=-0.1),
                lambda: AdamW([p]).step(max_norm=-1.0), lambda: AdamW([p]).step(max_norm=float("nan"))):
        with pytest.raises(ValueError):
            bad()
    opt = AdamW([p])
    for bad in (lambda: AdamW([torch.zeros(8)]), lambda: AdamW([p.half()]), lambda: AdamW([torch.zeros(8, 8, device=DEV).t()]),
                lambda: AdamW([p[:5], p[4:]]), lambda: AdamW([p, p.detach()]),
                lambda: opt.step(grads=[]), lambda: opt.step(grads=[torch.zeros(7, device=DEV)]), lambda: opt.step(grads=[torch.zeros(8)]),
                lambda: opt.step(grads=[torch.zeros(8, device=DEV, dtype=torch.float64)]), lambda: opt.load_moments(p, p),
                lambda: AdamW([p], state_bits=8).moments(torch.float16)):
        with pytest.raises(MqganHipError):
            bad()
    assert opt._steps() == ([0], 0)
    AdamW([p[:4], p[4:], torch.zeros(0, device=DEV)])      # halves of one buffer are two parameters
