"""Many rows: the balance loss where every team of lanes goes round several times (rows in flight, flags ahead, the exchange's two
buffers), and draws by every kernel for many rows, at the widths where one way of holding a row ends and the next begins."""
import pytest
import torch

import test_gpu_code_scores as few
from gpu_util import DEV

pytestmark = pytest.mark.gpu

# (codes, rows): five rows and more for every team of the gradient's 512 to 2048 blocks, each way of holding a row, whole quads and not
FORMS = [(8, 700_001, "f32"), (13, 660_007, "bf16"), (32, 330_011, "f16"), (100, 170_003, "f32"), (128, 90_001, "f32"), (256, 50_021, "bf16"),
         (250, 50_021, "f32"), (500, 45_011, "f16"), (1000, 44_003, "f32"), (1024, 42_001, "f32"), (2047, 41_003, "bf16"), (2048, 12_007, "f32"),
         (2049, 11_003, "f32"), (4096, 12_001, "bf16"), (4100, 6007, "f32"), (8192, 6001, "bf16"), (8192, 5501, "f32"), (8191, 5501, "f16"),
         (12_000, 2801, "f32"), (16_384, 2703, "f32"), (16_384, 5303, "bf16"), (16_500, 1203, "f32")]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("E,N,name", FORMS)
def test_balance_of_many_rows(E, N, name):
    from mqgan_amd.losses import code_balance_loss
    dt = TYPES[name]
    g = torch.Generator(device=DEV).manual_seed(E)
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    z = (torch.randn(N, E, generator=g, device=DEV) * 2).to(dt)
    idx = (rand(N) ** 2 * E).long().clamp(max=E - 1)
    padded = rand(N) < 0.2
    at = torch.arange(N, device=DEV)
    padded |= (at % 512) > 300 + (at // 512) % 212               # ragged ends of a batch of 512 frames
    padded[:3] = padded[-2:] = True
    padded[N // 2:N // 2 + N // 9] = True                        # nothing at all for many rounds of a team
    z[padded] = float("nan")                                     # not read
    leaf = z.requires_grad_(True)
    loss, counts = code_balance_loss(leaf, idx, padded)
    (dz,) = torch.autograd.grad(loss, leaf, torch.tensor(64.0, device=DEV))
    valid = torch.nonzero(~padded).reshape(-1)
    nv = len(valid)
    f = torch.bincount(idx[valid], minlength=E).double() / nv
    assert torch.equal(counts.long(), torch.bincount(idx[valid], minlength=E))
    # per entry as for few rows: exp's argument, the function and the row's sum, relative to p; column sums add a team's rows one by one
    want_loss, room_loss, worst = 0.0, 0.0, -1.0
    half = few.HALF[dt]
    for rows in valid.split(max(1, (1 << 24) // E)):
        x = z.detach()[rows].double()
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - top)
        p /= p.sum(1, keepdim=True)
        dp = ((top - x).clamp(max=200) + 28 + E / 64) * 2.0 ** -23
        dp = dp + (p * dp).sum(1, keepdim=True)
        s = (p * f).sum(1, keepdim=True)
        want_loss += float(s.sum()) * E / nv
        room_loss += float((p * (dp + 64 * 2.0 ** -24) * f).sum()) * E / nv
        want = 64.0 * E / nv * p * (f - s)
        room = 64.0 * E / nv * (p * ((f - s).abs() * dp + (f + s) * (dp + 2.0 ** -20)) + 2.0 ** -126) + half * want.abs()
        room = room + (2.0 ** -25 if dt == torch.float16 else 0.0)
        worst = max(worst, float(((dz[rows].double() - want).abs() - room).max()))
    assert abs(float(loss.detach()) - want_loss) <= room_loss + 4 * 2.0 ** -24 * want_loss
    assert worst <= 0, worst
    assert not bool(dz[padded].any())


@pytest.mark.parametrize("V,name", [(9896, "f32"), (9897, "f32"), (14848, "bf16"), (2047, "f16"), (2500, "f16"), (4096, "f16"), (5000, "f16"), (8192, "f16")])
def test_draws_of_many_rows_at_the_ends_of_each_form(V, name):
    few.test_draws_of_many_rows_equal_those_of_few(V, TYPES[name])


@pytest.mark.parametrize("V,name", [(9896, "f32"), (9897, "f32"), (14848, "f16"), (14849, "f16")])
def test_draws_at_the_ends_of_each_form_follow_the_definition(V, name):
    few.test_draws_follow_the_definition(V, TYPES[name])
