"""Uniform numbers, settings and padded flags belong to rows in their order: of the scores' leading shape, up to dimensions of 1, or flat."""
import pytest
import torch

from gpu_util import DEV

pytestmark = pytest.mark.gpu


def test_values_of_another_order_are_refused():
    from mqgan_amd import ops
    from mqgan_amd._lib import MqganHipError
    from mqgan_amd.losses import code_balance_loss
    z, u = torch.randn(3, 5, 20, device=DEV), torch.rand(3, 5, device=DEV)
    idx, padded = torch.zeros(3, 5, dtype=torch.int32, device=DEV), torch.zeros(3, 5, dtype=torch.bool, device=DEV)
    one = torch.ones(3, 5, device=DEV)
    for bad in (lambda: ops.sample_codes(z, u.t()), lambda: ops.sample_codes(z, u, padded=padded.t()), lambda: ops.sample_codes(z, u, temperature=one.t()),
                lambda: ops.sample_codes(z, u, top_p=one.t()), lambda: ops.sample_codes(z, u, top_k=one.t().int()), lambda: ops.sample_codes(z, u, min_p=one.t()),
                lambda: ops.sample_codes(z, u.t()[None]), lambda: code_balance_loss(z, idx, padded.t()), lambda: code_balance_loss(z, idx, padded.t()[:, None])):
        with pytest.raises(MqganHipError):
            bad()


def test_flat_values_and_dimensions_of_one_are_taken():
    from mqgan_amd import ops
    from mqgan_amd.losses import code_balance_loss
    g = torch.Generator().manual_seed(1)
    z, u = torch.randn(3, 5, 20, generator=g).to(DEV), torch.rand(3, 5, generator=g).to(DEV)
    padded = torch.zeros(3, 5, dtype=torch.bool, device=DEV)
    padded[1, 3:] = True
    t = torch.rand(3, 5, generator=g).to(DEV) + 0.5
    want = ops.sample_codes(z, u, temperature=t, padded=padded)
    for form in (lambda x: x.reshape(-1), lambda x: x[:, None], lambda x: x[..., None], lambda x: x[None]):
        assert torch.equal(ops.sample_codes(z, form(u), temperature=form(t), padded=form(padded)), want)
    assert torch.equal(ops.sample_codes(z[:1], u[:1].reshape(5)), ops.sample_codes(z[:1], u[:1]))
    loss = code_balance_loss(z, want.clamp(min=0), padded)[0]
    assert float(code_balance_loss(z, want.clamp(min=0), padded[:, None])[0]) == float(loss) == float(code_balance_loss(z, want.clamp(min=0), padded.reshape(-1))[0])
