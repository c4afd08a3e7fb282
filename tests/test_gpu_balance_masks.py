"""The balance loss over rows whose scores are large: masks by a large negative number in place of -inf, in whole rows, in one wave's
share of the columns and in a row's first codes, and scores on both sides of the size from which the softmax takes differences first."""
import pytest
import torch

from test_gpu_code_scores import check_balance

from gpu_util import DEV

pytestmark = pytest.mark.gpu

# every way a row is held: part of a wave, one wave, four, eight and sixteen waves (f32), and in memory
SIZES = [12, 1000, 2050, 8192, 16384, 16500]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("E", SIZES)
@pytest.mark.parametrize("mask", [-1e4, -1e6, -1e9, -1e10, -1e15, -1e20, -1e30, -9.9e36, 1e10, 1e12, 1e20, 9.9e36])
def test_balance_of_rows_masked_by_a_large_number(mask, E, dtype):
    g = torch.Generator().manual_seed(E)
    z = torch.randn(16, E, generator=g)
    z[0] = mask                                                  # nothing left: even, as the softmax says
    z[1, : E // 2] = mask
    z[2, E // 2:] = mask
    z[3, 0] = mask
    z[4, : min(E - 1, 300)] = mask                               # the first codes of every thread
    z[5, 1:] = mask
    z[6, ::2] = mask
    for r, at in ((7, 256), (8, 512), (9, 1024), (10, 4096)):    # a wave's share of a row that several waves hold
        if at < E:
            z[r, at:at + 256] = mask
    z[11, : E - 1] = mask
    z[12] = mask
    z[12, E // 3] = 1.0
    idx = torch.randint(0, E, (16, 2), generator=g)
    padded = torch.zeros(16, dtype=torch.bool)
    padded[14] = True
    check_balance(z.to(dtype).to(DEV), idx.to(DEV), padded.to(DEV))


@pytest.mark.parametrize("E", SIZES)
@pytest.mark.parametrize("level", [1e3, -1e4, 1e5, 2.0 ** 20, -2.0 ** 20, 2.0 ** 21, -2.0 ** 21, 3e6])
def test_balance_of_scores_around_a_large_level(level, E):
    """Scores a quarter apart around the level: a wave's maximum falls on either side of it, and no share of a row may be off by its rounding."""
    g = torch.Generator().manual_seed(E + 1)
    z = (level + torch.randint(-24, 25, (20, E), generator=g) * 0.25).float()
    z[1] = level
    z[2, : E // 2] = level - 1.0
    idx = torch.randint(0, E, (20,), generator=g)
    check_balance(z.to(DEV), idx.to(DEV), None)
