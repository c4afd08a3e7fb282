"""Draws from the widest rows of scores: the masses' unit against the steps of the uniform numbers."""
import pytest
import torch

from gpu_util import DEV
from test_gpu_code_scores import ref_row

pytestmark = pytest.mark.gpu
MOST = 1 << 19


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("V", [1000, 16385, MOST - 1, MOST])
def test_codes_that_weigh_nothing_are_not_drawn(V, dtype):
    """One code at 0, the others at -60 (e^-60 = 2^-86 each): only u = 0 may fall on one of them that stands before it."""
    from mqgan_amd import ops
    z = torch.full((2, V), -60.0, device=DEV, dtype=dtype)
    z[0, 0] = z[1, V - 1] = 0.0
    top = torch.tensor([1 - k * 2.0 ** -24 for k in range(1, 9)], device=DEV)
    low = torch.tensor([k * 2.0 ** -24 for k in range(1, 9)], device=DEV)
    for s in ({}, {"top_p": 1 - 2.0 ** -24}, {"top_k": V - 1}):
        assert ops.sample_codes(z[:1].expand(8, V), top, **s).tolist() == [0] * 8
        assert ops.sample_codes(z[1:].expand(8, V), low, **s).tolist() == [V - 1] * 8
    assert ops.sample_codes(z, torch.zeros(2, device=DEV)).tolist() == [0, 0]


@pytest.mark.parametrize("settings", [{}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.95}, {"min_p": 0.01, "temperature": 0.8}], ids=str)
def test_draws_of_the_widest_rows_follow_the_definition(settings):
    from mqgan_amd import ops
    g = torch.Generator().manual_seed(3)
    z = (torch.randn(5, MOST, generator=g) * 2).to(DEV)
    u = torch.rand(5, generator=g).to(DEV)
    idx, logp = ops.sample_codes(z, u, return_logp=True, **settings)
    name = {"temperature": "T", "top_k": "k", "top_p": "p", "min_p": "mp"}
    for n in range(5):
        i, lp, margin = ref_row(z[n].cpu().numpy(), float(u[n]), **{name[a]: v for a, v in settings.items()})
        if margin < 2.0 ** -24:                          # a border within all of the row's roundings
            continue
        assert int(idx[n]) == i
        assert abs(float(logp[n]) - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -24


def test_wider_rows_are_refused():
    from mqgan_amd import ops
    from mqgan_amd._lib import MqganHipError
    with pytest.raises(MqganHipError, match="2\\^19"):
        ops.sample_codes(torch.zeros(1, MOST + 1, device=DEV), torch.zeros(1, device=DEV))


def test_a_temperature_under_the_range_of_f32_is_not_zero():
    """Equal largest scores share the draw at every temperature above 0; at 0 the first of them has it."""
    from mqgan_amd import ops
    z = torch.zeros(4, 3, device=DEV)
    z[:, 0] = -1.0
    t = torch.tensor([1e-50, 1e-300, 0.0, -1e-50], dtype=torch.float64, device=DEV)
    u = torch.full((4,), 0.9, device=DEV)
    assert ops.sample_codes(z, u, temperature=t).tolist() == [2, 2, 1, 1]
    assert ops.sample_codes(z, u, temperature=1e-50).tolist() == [2] * 4
