"""Drawing codes from scores and the codebook's balance loss, against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu
INF = float("inf")
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ----------------------------------------------------------------------------- sampling
def ref_row(z, u, T=1.0, k=0, p=1.0, mp=0.0):
    """(code, log of its share, distance of u from the nearest border) of one row of f32 scores, in f64 from the definition."""
    z = np.where(np.isnan(z), -np.inf, z).astype(np.float64) + 0.0
    if not np.isfinite(z).any() and not (z == np.inf).any():
        return -1, 0.0, 1.0
    order = np.argsort(-z, kind="stable")
    top = z[order[0]]
    if not T > 0:
        return int(order[0]), 0.0, 1.0
    w = (z == np.inf) * 1.0 if top == np.inf else np.exp((z - top) / T)
    w = w[order]
    alive = w > 0
    if k > 0:
        alive &= np.arange(len(w)) < k
    w = np.where(alive, w, 0.0)
    margin = 1.0
    if p < 1:
        before = np.cumsum(w) - w
        goal = p * w.sum()
        keep = before < goal
        keep[0] = True
        near = np.abs(before - goal)[1:]
        if len(near) and goal > 0:
            margin = min(margin, float(near.min() / w.sum()))
        w = np.where(keep, w, 0.0)
    if mp == mp:
        w = np.where(w < min(mp, 1.0), 0.0, w)
    by = np.zeros_like(w)
    by[order] = w
    reach = np.cumsum(by)
    u = min(max(float(u), 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    at = u * reach[-1]
    i = int(np.argmax((reach > at) & (by > 0)))
    if u > 0:
        margin = min(margin, float(np.abs(reach - at).min() / reach[-1]))
    return i, float(np.log(by[i] / reach[-1])), margin


def check_draws(z, u, **kw):
    """Every row against ref_row; rows whose u (or top-p cut) lies within 1e-9 of a border may fall on either side, and are few.  ON a border
    (equal scores: weights of 1 and sums of them are exact in both) they may not."""
    from mqgan_amd import ops
    idx, logp = ops.sample_codes(z, u, return_logp=True, **kw)
    assert idx.dtype == torch.int64 and idx.shape == z.shape[:-1] and logp.dtype == torch.float32
    rows = z.float().cpu().numpy().reshape(-1, z.shape[-1])
    idx, logp, u = idx.cpu().numpy().reshape(-1), logp.cpu().numpy().reshape(-1), u.cpu().numpy().reshape(-1)
    name = {"temperature": "T", "top_k": "k", "top_p": "p", "min_p": "mp"}
    edge = 0
    for n in range(len(rows)):
        s = {name[a]: (v.reshape(-1)[n].item() if torch.is_tensor(v) else v) for a, v in kw.items() if a != "padded"}
        i, lp, margin = ref_row(rows[n], u[n], **s)
        if 0 < margin < 1e-9:
            edge += 1
            continue
        assert idx[n] == i, (n, idx[n], i, s, float(u[n]), margin)
        # the log of a quotient of f64 sums, rounded once; the units' own rounding is 2^-36 of the mass
        assert abs(logp[n] - lp) <= 2.0 ** -24 * abs(lp) + 2e-10, (n, logp[n], lp)
    assert edge <= max(2, len(rows) // 50), edge


SETTINGS = [{}, {"temperature": 1e-310}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 5}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_p": 0.0}, {"temperature": 0.0},
            {"temperature": 1.3, "top_k": 40, "top_p": 0.8, "min_p": 0.02}, {"temperature": 3.0, "top_k": 300, "top_p": 0.999}]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 64, 65, 255, 256, 257, 1000, 1024, 2049, 4097, 8003, 8192, 20001, 65536])
def test_draws_follow_the_definition(V, dtype):
    g = torch.Generator().manual_seed(V)
    rows = 24 if V <= 8192 else 6
    z = (torch.randn(rows, V, generator=g) * 3).to(dtype).to(DEV)
    u = torch.rand(rows, generator=g).to(DEV)
    for s in SETTINGS:
        check_draws(z, u, **s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 3, 255, 256, 260, 1000, 1024, 1025, 2047, 2500, 3001, 4095, 4096, 4097, 8003, 8192, 8193, 9000, 14336, 14849, 16384, 16385, 40001])
def test_draws_of_many_rows_equal_those_of_few(V, dtype):
    """Masses are whole numbers, so however a row's work is split its code and its logarithm are the same to the last bit; and the definition's."""
    from mqgan_amd import ops
    g = torch.Generator(device=DEV).manual_seed(V + 5)
    n = 4101
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    normal = torch.randn(n, V, generator=g, device=DEV) * 3
    z = normal.clone()
    z[::7] = (z[::7] * 2).round()                                # ties
    z[5::7] *= 0.01                                              # flat: top-p keeps most
    z[rand(n, V) < 0.1] = -INF
    z[3], z[40, V // 2], z[41] = -INF, INF, 2.5
    z[42, ::2], z[43], z[44] = torch.finfo(torch.float32).min, z[43] * 1e4, z[44].clamp(0, 0) * z[44].sign()      # zeros of both signs
    z, normal, u, padded = z.to(dtype), normal.to(dtype), rand(n), rand(n) < 0.1
    padded[40:45] = False
    by_row = {"temperature": rand(n) * 2 - 0.2, "top_p": rand(n), "top_k": torch.randint(-1, 200, (n,), generator=g, device=DEV, dtype=torch.int32)}
    for s in SETTINGS + [{"top_k": 90, "top_p": 0.95}, {"top_k": 120}, {"top_k": 200}, by_row, {"temperature": by_row["temperature"], "top_k": 30}]:
        s = dict(s, padded=padded)
        idx, logp = ops.sample_codes(z, u, return_logp=True, **s)
        for a, b in ((0, 50), (50, 350), (350, 1000), (1000, 3100), (3100, n)):
            part = {k: v[a:b] if torch.is_tensor(v) else v for k, v in s.items()}
            i, lp = ops.sample_codes(z[a:b], u[a:b], return_logp=True, **part)
            assert torch.equal(i, idx[a:b]) and torch.equal(lp, logp[a:b]), (s, a)
    for s in ({}, {"top_k": 20, "top_p": 0.9}, {"top_p": 0.7, "min_p": 0.01}):
        idx = ops.sample_codes(normal, u, **s)
        for r in range(0, n, 400):
            want, _, margin = ref_row(normal[r].float().cpu().numpy(), float(u[r]), **{{"top_k": "k", "top_p": "p", "min_p": "mp"}[k]: v for k, v in s.items()})
            assert 0 < margin < 1e-9 or int(idx[r]) == want, (s, r)


@pytest.mark.parametrize("kind", ["levels", "equal", "zeros of both signs", "masked", "one left", "lowest of the type", "steep", "falling", "rising"])
@pytest.mark.parametrize("V", [5, 257, 1000, 8003])
def test_draws_among_ties_masks_and_extremes(kind, V):
    g = torch.Generator().manual_seed(V + 1)
    z = torch.randn(16, V, generator=g)
    if kind == "levels":
        z = (z * 2).round()
    elif kind == "equal":
        z = torch.full_like(z, -3.25)
    elif kind == "zeros of both signs":
        z = torch.where(z > 0, 0.0, -0.0)
    elif kind == "masked":
        z[torch.rand(16, V, generator=g) < 0.9] = -INF
        z[3] = -INF
    elif kind == "one left":
        z = torch.full_like(z, -INF)
        z[torch.arange(16), torch.randint(0, V, (16,), generator=g)] = -5.0
    elif kind == "lowest of the type":
        z[:, ::3] = torch.finfo(torch.float32).min
        z[5] = torch.finfo(torch.float32).min
    elif kind == "steep":
        z = z * 1e4
    elif kind == "falling":
        z = -torch.arange(V).float().expand(16, V) * 0.01
    elif kind == "rising":
        z = torch.arange(V).float().expand(16, V) * 0.01
    z, u = z.contiguous().to(DEV), torch.rand(16, generator=g).to(DEV)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    for s in SETTINGS:
        check_draws(z, u, **s)


def test_draws_of_more_rows_than_one_launch_takes():
    from mqgan_amd import ops
    g = torch.Generator(device=DEV).manual_seed(8)
    n = (1 << 21) + 5
    z, u = torch.randn(n, 3, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
    idx, logp = ops.sample_codes(z, u, top_k=2, return_logp=True)
    half = 1 << 20
    for at in range(0, n, half):
        i, lp = ops.sample_codes(z[at:at + half], u[at:at + half], top_k=2, return_logp=True)
        assert torch.equal(i, idx[at:at + half]) and torch.equal(lp, logp[at:at + half])
    last = z.sort(dim=-1, descending=True, stable=True).indices[:, -1]      # of two equal lowest the one with the higher index
    assert int(idx.min()) >= 0 and not bool((idx == last).any())


def test_draws_with_a_top_k_past_32_bits():
    from mqgan_amd import ops
    z, u = torch.randn(4, 100, device=DEV), torch.rand(4, device=DEV)
    k = torch.tensor([2 ** 32 + 1, -2 ** 40, 2 ** 62, 1], device=DEV)
    assert torch.equal(ops.sample_codes(z, u, top_k=k), ops.sample_codes(z, u, top_k=torch.tensor([0, 0, 0, 1], dtype=torch.int32, device=DEV)))


def test_draws_with_infinite_and_undefined_scores():
    from mqgan_amd import ops
    z = torch.tensor([[0.0, INF, 1.0, INF], [float("nan"), 1.0, float("nan"), -INF], [float("nan")] * 4, [-INF] * 4, [1.0, 2.0, 3.0, 4.0]], device=DEV)
    u = torch.tensor([0.6, 0.99, 0.5, 0.5, 2.0], device=DEV)
    for s in SETTINGS[:3]:
        idx, logp = ops.sample_codes(z, u, return_logp=True, **s)
        assert idx.tolist() == [3, 1, -1, -1, 3]
        assert logp[:4].tolist() == pytest.approx([math.log(0.5), 0.0, 0.0, 0.0], abs=1e-7)
    assert ops.sample_codes(z, u, top_k=1).tolist() == [1, 1, -1, -1, 3]
    assert ops.sample_codes(z, u, temperature=0.0).tolist() == [1, 1, -1, -1, 3]
    assert ops.sample_codes(z[4:].expand(3, 4), torch.tensor([-1.0, float("nan"), INF], device=DEV)).tolist() == [0, 0, 3]
    assert ops.sample_codes(z[4:], u[4:], temperature=INF).tolist() == [3] and ops.sample_codes(z[4:], u[:1] * 0 + 0.3, temperature=INF).tolist() == [1]


@pytest.mark.parametrize("V", [1000, 8192])
def test_draws_with_settings_of_each_row(V):
    g = torch.Generator().manual_seed(V + 2)
    n = 40
    z, u = (torch.randn(n, V, generator=g) * 3).to(DEV), torch.rand(n, generator=g).to(DEV)
    t = (torch.rand(n, generator=g) * 2).to(DEV)
    t[:3] = torch.tensor([0.0, -1.0, 1e-6])
    k = torch.randint(0, 2 * V, (n,), generator=g, dtype=torch.int32).to(DEV)
    k[4:7] = torch.tensor([0, 1, -3], dtype=torch.int32)
    p, mp = torch.rand(n, generator=g).to(DEV), (torch.rand(n, generator=g) * 0.05).to(DEV)
    p[8:10] = torch.tensor([1.0, 0.0])
    mp[11:13] = torch.tensor([1.0, 0.0])
    check_draws(z, u, temperature=t, top_k=k, top_p=p, min_p=mp)


@pytest.mark.parametrize("settings", [{}, {"temperature": 0.8, "top_k": 20}, {"top_p": 0.7}, {"min_p": 0.2}], ids=str)
def test_evenly_spread_numbers_draw_each_code_its_share(settings):
    """n rows of the same scores with u = (j + 1/2) / n: a code with share q is drawn n q times, give or take one.  A code that no u falls on has
    a share under 1 / n, so the shares seen miss less than (codes not drawn) / n of 1."""
    from mqgan_amd import ops
    V, n = 150, 5000
    row = torch.randn(V, generator=torch.Generator().manual_seed(4)) * 1.5
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().to(DEV)
    idx, logp = ops.sample_codes(row.to(DEV).repeat(n, 1), u, return_logp=True, **settings)
    got = torch.bincount(idx, minlength=V).cpu().double()
    share = torch.zeros(V, dtype=torch.float64)
    share[idx.cpu()] = logp.cpu().double().exp()
    missed = 1 - float(share.sum())
    assert -1e-5 < missed < int((got == 0).sum()) / n + 1e-5 and float((got - n * share).abs().max()) <= 1.01


def test_draws_read_slices_in_place_and_skip_padded_rows():
    from mqgan_amd import ops
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(3, 7, 1003, generator=g).to(DEV)
    u = torch.rand(3, 7, generator=g).to(DEV)
    padded = torch.rand(3, 7, generator=g).to(DEV) < 0.4
    part = wide[..., 1:1001]
    want = ops.sample_codes(part.contiguous(), u, top_p=0.9)
    assert torch.equal(ops.sample_codes(part, u, top_p=0.9), want)
    assert torch.equal(ops.sample_codes(wide.transpose(0, 1)[..., 1:1001], u.t(), top_p=0.9), want.t())          # not one stride: copied
    dirty = part.clone()
    dirty[padded] = float("nan")
    got, logp = ops.sample_codes(dirty, u, top_p=0.9, padded=padded, return_logp=True)
    assert torch.equal(got, torch.where(padded, -1, want)) and bool((logp[padded] == 0).all())
    assert torch.equal(ops.sample_codes(dirty, u, top_p=0.9, padded=padded.to(torch.uint8)), got)
    assert ops.sample_codes(wide[:0], u[:0]).shape == (0, 7)
    one, lp = ops.sample_codes(wide[0, 0], u[0, 0], return_logp=True)
    assert one.shape == () and one == ops.sample_codes(wide[:1, 0], u[:1, 0])[0]


def test_draws_in_a_graph_and_on_another_stream():
    from mqgan_amd import ops
    g = torch.Generator().manual_seed(9)
    z, u = (torch.randn(50, 1000, generator=g) * 3).to(DEV), torch.rand(50, generator=g).to(DEV)
    ops.sample_codes(z, u, top_k=50, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_codes(z, u, top_k=50, top_p=0.9)
    for r in range(4):
        z.copy_(torch.randn(50, 1000, generator=g) * 3)
        u.copy_(torch.rand(50, generator=g))
        graph.replay()
        assert torch.equal(out, ops.sample_codes(z, u, top_k=50, top_p=0.9)), r
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops.sample_codes(z, u, top_k=50, top_p=0.9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, out)


def test_draw_refusals():
    from mqgan_amd import ops
    from mqgan_amd._lib import MqganHipError
    z, u = torch.zeros(4, 10, device=DEV), torch.zeros(4, device=DEV)
    for bad in (lambda: ops.sample_codes(z.double(), u), lambda: ops.sample_codes(z, u[:3]), lambda: ops.sample_codes(z, u.double()),
                lambda: ops.sample_codes(z, u, top_p=1.5), lambda: ops.sample_codes(z, u, min_p=-0.1), lambda: ops.sample_codes(z, u, top_k=-1),
                lambda: ops.sample_codes(z, u, temperature=-1.0), lambda: ops.sample_codes(z, u, temperature=float("nan")),
                lambda: ops.sample_codes(z, u, top_p=torch.ones(3, device=DEV)), lambda: ops.sample_codes(z[:, :0], u),
                lambda: ops.sample_codes(z, u, padded=torch.zeros(5, dtype=torch.uint8, device=DEV)), lambda: ops.sample_codes(z.cpu(), u),
                lambda: ops.sample_codes(z, u.cpu()), lambda: ops.sample_codes(torch.zeros(1, (1 << 20) + 1, device=DEV), u[:1])):
        with pytest.raises(MqganHipError):
            bad()


# ----------------------------------------------------------------------------- balance loss
def ref_balance(z, idx, padded):
    """(loss, counts, gradient, p, f, share per row) in f64."""
    z = z.double()
    N, E = z.shape
    keep = torch.nonzero(~padded).reshape(-1)
    nv = len(keep)
    p = torch.zeros_like(z)
    for n in keep.tolist():
        row = z[n]
        if bool((row == -INF).all()):
            continue
        w = torch.exp(row - row.max())
        p[n] = w / w.sum()
    chosen = idx[keep].reshape(-1).long()
    chosen = chosen[(chosen >= 0) & (chosen < E)]
    counts = torch.bincount(chosen, minlength=E)
    if nv == 0:
        return 0.0, counts, torch.zeros_like(z), p, counts.double(), torch.zeros(N, dtype=torch.float64)
    f = counts.double() / (nv * idx.shape[1])
    s = (p * f).sum(1)
    return float(E * s.sum() / nv), counts, E / nv * p * (f - s[:, None]) * (~padded)[:, None], p, f, s


def check_balance(z, idx, padded, gout=1.0):
    from mqgan_amd.losses import code_balance_loss
    E, dt = z.shape[-1], z.dtype
    z2, i2 = z.reshape(-1, E).cpu(), idx.reshape(z.numel() // E, -1).cpu()
    pad = torch.zeros(z2.shape[0], dtype=torch.bool) if padded is None else padded.reshape(-1).cpu() != 0
    loss, counts, grad, p, f, s = ref_balance(z2.float(), i2, pad)
    leaf = z.detach().requires_grad_(True)
    got, n = code_balance_loss(leaf, idx, padded)
    assert got.shape == () and got.dtype == torch.float32 and n.dtype == torch.int32 and not n.requires_grad
    assert torch.equal(n.cpu().long(), counts)
    # exp: its argument rounds by (|x - max| + 1) steps of its exponent, the function and the row sum add a few (sums of up to E / 64 terms a
    # lane, then a tree); both relative to p
    x = z2.double()
    top = torch.where(torch.isfinite(x), x, torch.full_like(x, -1e30)).amax(1, keepdim=True)
    depth = torch.where(p > 0, top - x, 0.0).clamp(min=0, max=200)
    dp = (depth + 12 + E / 64 + 16) * 2.0 ** -23
    dp = dp + (p * dp).sum(1, keepdim=True)
    assert abs(float(got.detach()) - loss) <= E / max(1, int((~pad).sum())) * float((p * dp * f).sum()) + 4 * 2.0 ** -24 * abs(loss)
    dz = torch.autograd.grad(got, leaf, torch.tensor(float(gout), device=DEV))[0]
    assert dz.dtype == dt and dz.shape == z.shape
    off = (dz.double().cpu().reshape(-1, E) - gout * grad).abs()
    nv = max(1, int((~pad).sum()))
    room = abs(gout) * E / nv * p * ((f - s[:, None]).abs() * dp + (f + s[:, None]) * (dp + 2.0 ** -20)) + HALF[dt] * abs(gout) * grad.abs()
    # the hardware's exp2 gives 0 for results under the smallest normal number, 2^-126: p is off by up to that much, and |f - s| <= 1
    room = room + (2.0 ** -25 if dt == torch.float16 else abs(gout) * E / nv * 2.0 ** -126)
    worst = float((off - room).max()) if off.numel() else 0.0
    assert worst <= 0, f"gradient off by {float(off.max()):.3e}, {worst:.3e} over the bound"
    assert bool((dz.reshape(-1, E)[pad.to(DEV)] == 0).all())
    return got, n, dz


ES = [1, 2, 5, 8, 16, 31, 64, 65, 100, 256, 257, 512, 1000, 1024, 1030, 2048, 2050, 4097, 8000, 8192, 12000, 16384, 16385, 33000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("E", ES)
def test_balance_loss_counts_and_gradient(E, dtype):
    g = torch.Generator().manual_seed(E)
    for N, K, share in ((1, 1, 0.0), (67, 1, 0.3), (515 if E < 5000 else 130, 2, 0.1)):
        z = (torch.randn(N, E, generator=g) * 2 + torch.randn(E, generator=g)).to(dtype).to(DEV)
        idx = torch.randint(0, E, (N, K), generator=g, dtype=torch.int32).to(DEV)
        padded = (torch.rand(N, generator=g) < share).to(DEV)
        check_balance(z, idx, padded, gout=1.0 if dtype != torch.float16 else 1024.0)


@pytest.mark.parametrize("E", [12, 1000, 8192])
def test_balance_of_masked_extreme_and_padded_rows(E):
    g = torch.Generator().manual_seed(E + 1)
    z = torch.randn(40, E, generator=g)
    z[1] = -INF
    z[2, : E // 2] = -INF
    z[3] = torch.finfo(torch.float32).min
    z[4, ::2] = torch.finfo(torch.float32).min
    z[5] = 3e38
    z[6] = z[6] * 100
    z[7] = 1e-40
    padded = torch.zeros(40, dtype=torch.uint8)
    padded[10:14] = 1
    z[10], z[11], z[12] = float("nan"), INF, -INF
    idx = torch.randint(0, E, (40, 3), generator=g)
    idx[8] = torch.tensor([-1, E, 2 ** 40])
    idx[11] = 2 ** 33
    check_balance(z.to(DEV), idx.to(DEV), padded.to(DEV))
    check_balance(z.to(DEV), idx.clamp(-5, E + 5).int().to(DEV), padded.to(DEV).bool(), gout=-3.0)
    loss, counts, dz = check_balance(z.to(DEV), idx.to(DEV), torch.ones(40, dtype=torch.uint8, device=DEV))
    assert float(loss) == 0.0 and int(counts.sum()) == 0 and not bool(dz.any())


def test_balance_ranges_from_one_to_the_number_of_codes():
    from mqgan_amd.losses import code_balance_loss
    E = 50
    even = torch.arange(E, device=DEV, dtype=torch.int32).repeat(4)
    flat = torch.zeros(4 * E, E, device=DEV)
    assert float(code_balance_loss(flat, even)[0]) == pytest.approx(1.0, abs=1e-6)
    one = torch.full((4 * E, E), -100.0, device=DEV)
    one[:, 7] = 100.0
    assert float(code_balance_loss(one, torch.full_like(even, 7))[0]) == pytest.approx(E, rel=1e-6)


def test_balance_gradient_against_differences():
    """Directional differences of the 64-bit loss (h = 1e-5: 1e-10 of truncation, 1e-11 of cancellation) against the kernel's gradient."""
    g = torch.Generator().manual_seed(6)
    z = torch.randn(30, 41, generator=g)
    idx = torch.randint(0, 41, (30, 2), generator=g)
    padded = torch.zeros(30, dtype=torch.bool)
    padded[4] = True
    _, _, dz = check_balance(z.to(DEV), idx.to(DEV), padded.to(DEV))
    for r in range(5):
        d = torch.randn(30, 41, generator=g).double()
        h = 1e-5
        up, down = (ref_balance(z.double() + s * h * d, idx, padded)[0] for s in (1, -1))
        want = (up - down) / (2 * h)
        got = float((dz.double().cpu() * d).sum())
        assert abs(got - want) <= 1e-5 * float((dz.double().cpu() * d).abs().sum()) + 1e-8


def test_balance_reads_slices_in_place_and_takes_batches():
    from mqgan_amd.losses import code_balance_loss
    g = torch.Generator().manual_seed(7)
    wide = torch.randn(3, 9, 261, generator=g).to(DEV).requires_grad_(True)
    idx = torch.randint(0, 256, (3, 9), generator=g).to(DEV)
    padded = (torch.rand(3, 9, generator=g) < 0.3).to(DEV)
    part = wide[..., 3:259]
    check_balance(part.detach(), idx, padded)
    loss, _ = code_balance_loss(part, idx, padded)
    loss.backward()
    own, _, dz = check_balance(part.detach().contiguous(), idx, padded)
    assert float(loss) == float(own) and torch.equal(wide.grad[..., 3:259], dz)
    assert not bool(wide.grad[..., :3].any()) and not bool(wide.grad[..., 259:].any())
    # a broadcast input gets the sum of its rows' gradients
    row = torch.randn(1, 64, generator=g).to(DEV).requires_grad_(True)
    many = row.expand(9, 64)
    i = torch.randint(0, 64, (9,), generator=g).to(DEV)
    (a,) = torch.autograd.grad(code_balance_loss(many, i)[0], row)
    _, _, b = check_balance(many.detach().contiguous(), i, None)
    assert torch.allclose(a[0], b.sum(0), rtol=1e-5, atol=1e-9)
    loss, counts = code_balance_loss(torch.zeros(0, 16, device=DEV, requires_grad=True), torch.zeros(0, dtype=torch.int32, device=DEV))
    assert float(loss) == 0.0 and counts.shape == (16,) and not bool(counts.any())
    (e,) = torch.autograd.grad(loss, [loss.grad_fn.next_functions[0][0].variable])
    assert e.shape == (0, 16)


class _Two:
    """Two ranks' communicator on one GPU: the first pass records a shard's sums, the second adds both up."""
    world, rank, active = 2, 0, True

    def __init__(self):
        self.seen, self.total = [], None

    def all_reduce_sum(self, t):
        if self.total is None:
            self.seen.append(t.clone())
        else:
            t.copy_(self.total)
        return t


def test_balance_of_shards_is_the_balance_of_the_batch():
    from mqgan_amd.losses import code_balance_loss
    g = torch.Generator().manual_seed(11)
    E, N = 300, 90
    z = torch.randn(N, E, generator=g).to(DEV)
    idx = torch.randint(0, E, (N, 2), generator=g).to(DEV)
    padded = (torch.rand(N, generator=g) < 0.3).to(DEV)
    whole, counts, dz = check_balance(z, idx, padded)
    comm, cuts = _Two(), (slice(0, 31), slice(31, N))
    for c in cuts:
        code_balance_loss(z[c], idx[c], padded[c], comm)
    comm.total = comm.seen[0] + comm.seen[1]
    for c in cuts:
        leaf = z[c].clone().requires_grad_(True)
        loss, n = code_balance_loss(leaf, idx[c], padded[c], comm)
        assert torch.equal(n, counts) and abs(float(loss) - float(whole)) <= 8 * 2.0 ** -24 * float(whole)
        (d,) = torch.autograd.grad(loss, leaf)
        # the two sums of a code's mass round apart: four half steps of f and s
        assert float((d - dz[c]).abs().max()) <= 8 * 2.0 ** -24 * float(dz.abs().max()) + 1e-12


def test_balance_is_the_same_on_every_run_and_in_a_graph():
    from mqgan_amd.losses import code_balance_loss
    g = torch.Generator().manual_seed(12)
    z = torch.randn(2000, 512, generator=g).to(DEV).requires_grad_(True)
    idx = torch.randint(0, 512, (2000,), generator=g).to(DEV)

    def once():
        loss, n = code_balance_loss(z, idx)
        return loss.detach().clone(), n, torch.autograd.grad(loss, z)[0]
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
    del first
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for r in range(4):
        with torch.no_grad():
            z.copy_(torch.randn(2000, 512, generator=g))
        idx.copy_(torch.randint(0, 512, (2000,), generator=g))
        graph.replay()
        want = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r


def test_balance_gradient_is_not_differentiated_again():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.losses import code_balance_loss
    z = torch.randn(4, 10, device=DEV, requires_grad=True)
    loss, _ = code_balance_loss(z, torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(MqganHipError, match="again"):
        torch.autograd.grad(loss, z, create_graph=True)


def test_balance_refusals():
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.losses import code_balance_loss
    z, i = torch.zeros(4, 10, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    for bad in (lambda: code_balance_loss(z.double(), i), lambda: code_balance_loss(z, i[:3]), lambda: code_balance_loss(z, i.float()),
                lambda: code_balance_loss(z, i, torch.zeros(4, device=DEV)), lambda: code_balance_loss(z, i, torch.zeros(3, dtype=torch.uint8, device=DEV)),
                lambda: code_balance_loss(z, i[:, None][:, :0]), lambda: code_balance_loss(z.cpu(), i), lambda: code_balance_loss(z, i.cpu()), lambda: code_balance_loss(z[:, :0], i)):
        with pytest.raises(MqganHipError):
            bad()
