"""AdamW's 8-bit moments under gradients of two bytes, bit for bit against the format, and the norm of such gradients."""
import math

import numpy as np
import pytest
import torch

import test_gpu_adamw as base
from gpu_util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("unaligned", [False, True], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_eight_bit_steps_of_two_byte_gradients(dtype, unaligned):
    from mqgan_amd.optim import AdamW
    f, sizes = np.float32, base.SIZES + [8192 + 4096, 40_000]
    ps = [x[1] for x in base._leaves(sizes, 2, unaligned)]
    opt = AdamW(ps, lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=77)
    total = opt.positions[-1]
    rows = total // 256
    mc, mb, vc, vb = np.zeros(total, np.uint8), np.zeros(rows, np.uint8), np.zeros(total, np.uint8), np.zeros(rows, np.uint8)
    for t in range(1, 5):
        gs = base._grads(sizes, 100 + t, dtype, scale=10.0 ** (t - 3))
        if unaligned:
            gs = [torch.cat([g.new_zeros(1), g])[1:] for g in gs]
        opt.step(grads=gs)
        g = np.zeros(total, f)
        for a, x in zip(opt.positions, gs):
            g[a:a + x.numel()] = x.float().cpu().numpy()
        m, v = base.np_decode(mc, mb, 4), base.np_decode(vc, vb, 5)
        m = m + (g - m) * f(1 - 0.9)
        v = v * f(0.999) + f(1 - 0.999) * g * g
        w = base.np_words(total, 77, t)
        mc, mb = base.np_encode(m, 4, w >> np.uint32(16))
        vc, vb = base.np_encode(v, 5, w & np.uint32(0xFFFF))
        for got, want, what in ((opt.exp_avg, mc, "m"), (opt._bases[0], mb, "m base"), (opt.exp_avg_sq, vc, "v"), (opt._bases[1], vb, "v base")):
            d = got.cpu().numpy() != want
            assert not d.any(), f"step {t}: {int(d.sum())} of {d.size} {what} differ, first at {int(d.argmax())}"
    opt.step(max_norm=0.01, grads=gs)
    norm = math.sqrt(sum(float(x.double().square().sum()) for x in gs))
    assert abs(float(opt.grad_norm()) / norm - 1) <= 4 * base.H32


@pytest.mark.parametrize("bits", [32, 8])
def test_two_byte_gradients_step_as_the_same_values_in_f32(bits):
    from mqgan_amd.optim import AdamW
    sizes = base.SIZES + [50_000]
    gs = base._grads(sizes, 3, torch.bfloat16)
    runs = []
    for grads in (gs, [g.float() for g in gs]):
        ps = [x[1] for x in base._leaves(sizes, 4)]
        opt = AdamW(ps, lr=1e-2, state_bits=bits, seed=5)
        for _ in range(3):
            opt.step(max_norm=0.5, grads=grads)
        runs.append(ps + list(opt.moments()))
    for a, b in zip(*runs):
        assert float((a - b).abs().max()) == 0.0
