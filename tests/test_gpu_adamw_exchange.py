"""AdamW behind the gradient exchange with one rank and every collective forced: over RCCL through torch.distributed and through the C ABI,
against the same steps without collectives, bit for bit (the set of tensors with a gradient then comes from the device)."""
import numpy as np
import pytest
import torch

from conftest import load_golden
from test_gpu_exchange import _batch, _trainer

pytestmark = pytest.mark.gpu


def _rank(port, kind, abi, q):
    import torch.distributed as dist
    try:
        torch.cuda.set_device(0)
        if not abi:
            dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1, device_id=torch.device("cuda", 0))
        from mqgan_amd import ddp
        from mqgan_amd.comm import RcclAbiComm
        from mqgan_amd.train import WarmupLR
        g = load_golden("g7_trainstep.npz")
        batches = [_batch(T, 700 + 10 * i) for i, T in enumerate((40, 24, 48))]

        def run(force):
            c = RcclAbiComm(force=True) if abi and force else None
            tr = _trainer(g, comm=c, force_collectives=force) if abi else _trainer(g, force_collectives=force)
            tr.config["training"] = {**tr.config["training"], "optimizer": kind, "weight_decay": 0.1}
            tr.optimizer_g, tr.optimizer_d = tr._init_optimizers()
            tr.scheduler_g = WarmupLR(tr.optimizer_g, tr.config["training"]["warmup_steps"])
            if force:
                for r in (tr.reducer_g, tr.reducer_d):
                    r.remove()
                more = {"comm": c} if abi else {}
                tr.reducer_g = ddp.GradReducer(tr.arena_g, bucket_bytes=64 << 10, force=True, **more)
                tr.reducer_d = ddp.GradReducer(tr.arena_d, bucket_bytes=64 << 10, force=True, **more)
                assert tr.reducer_g.enabled and len(tr.reducer_g.buckets) >= 2
            for x, lens in batches:              # no host synchronisation between the steps
                tr.train_step(x, lens)
                assert (tr.arena_g.present is not None) == (tr.arena_d.present is not None) == force
            torch.cuda.synchronize()
            out = [tr.arena_g.flat_param.cpu().numpy(), tr.arena_d.flat_param.cpu().numpy()]
            out += [m.float().cpu().numpy() for o in (tr.optimizer_g, tr.optimizer_d) for m in o.moments()]
            out += [np.array(o._steps()[0]) for o in (tr.optimizer_g, tr.optimizer_d)]
            if c is not None:
                c.close()
            return out
        q.put(("ok", run(False), run(True)))
    except BaseException as e:                   # noqa: BLE001 - reported by the parent
        import traceback
        q.put(("error", repr(e), traceback.format_exc()))
    finally:
        if dist.is_initialized():
            dist.destroy_process_group()


@pytest.mark.parametrize("abi", [False, True], ids=["torch.distributed", "C ABI"])
@pytest.mark.parametrize("kind", ["adamw", "adamw8bit"])
def test_forced_collectives_change_no_bit(kind, abi):
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    p = ctx.Process(target=_rank, args=(port, kind, abi, q))
    p.start()
    msg = q.get(timeout=100)
    p.join(timeout=60)
    assert msg[0] == "ok", msg[1:]
    assert p.exitcode == 0
    for i, (a, b) in enumerate(zip(msg[1], msg[2])):
        assert np.array_equal(a, b, equal_nan=True), i
    assert 0 in msg[1][-2] and 3 in msg[1][-2]   # some tensor of the generator never has a gradient
