"""Which tensors AdamW steps under data parallelism: a gradient that one rank alone has reaches every rank through the reducer, so every rank
has to step its tensor; one that no rank has is left out everywhere.  Host logic under two gloo ranks (no GPU needed)."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_ddp_gloo import AsyncBucketDouble, Net, _free_port


def _optimiser(arena):
    """An AdamW's host side over a CPU arena (its kernels need a GPU)."""
    from mqgan_amd.optim import AdamW
    opt = AdamW.__new__(AdamW)
    opt.arena, opt.params = arena, arena.params
    arena.track_presence = True
    return opt


def _worker(rank, world, port, out_q, abi):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from mqgan_amd.ddp import FlatArena, GradReducer
        torch.manual_seed(5)
        net = Net()
        arena = FlatArena([net], gather=True)
        opt = _optimiser(arena)
        red = GradReducer(arena, comm=AsyncBucketDouble() if abi else None)
        assert red.enabled and len(red.buckets) == 1
        out = []
        for step in range(3):
            arena.zero_grad()
            assert arena.present is None
            red.start()
            x = torch.randn(6, 13, generator=torch.Generator().manual_seed(10 * step + rank))
            h = torch.relu(net.a(x))
            # step 0: both ranks use every layer but `unused`; steps 1 and 2: rank 1 stops after the first layer
            y = h.pow(2).sum() if rank and step else (net.c(torch.tanh(net.b(h))) * net.scale).pow(2).sum()
            y.backward()
            red.finish()
            grads = opt._gradients(None)
            out.append(([g is not None for g in grads], arena.present.clone(), arena.flat_grad.clone(), [p.grad is not None for p in arena.params]))
        out_q.put((rank, out))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("abi", [False, True], ids=["torch.distributed", "async-bucket communicator"])
def test_ranks_step_the_same_tensors(abi):
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q, abi)) for r in range(2)]
    for p in procs:
        p.start()
    (_, a), (_, b) = sorted([q.get(timeout=60) for _ in range(2)], key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    net = Net()
    never = {id(p) for p in net.unused.parameters()}
    used = torch.tensor([id(p) not in never for p in net.parameters()])
    assert int(used.sum()) == 7
    for step, ((given0, present0, flat0, own0), (given1, present1, flat1, own1)) in enumerate(zip(a, b)):
        assert torch.equal(flat0, flat1) and given0 == given1 == [True] * len(given0)
        assert torch.equal(present0, present1) and torch.equal(present0 > 0, used), step
        assert (own0 != own1) == (step > 0)                  # the case is what it says


def test_without_a_reducer_a_tensor_is_stepped_where_it_has_a_gradient():
    from mqgan_amd.ddp import FlatArena, GradReducer
    net = Net()
    arena = FlatArena([net], gather=True)
    opt = _optimiser(arena)
    red = GradReducer(arena)
    assert not red.enabled
    red.start()
    net(torch.randn(6, 13)).sum().backward()
    red.finish()
    assert arena.present is None
    grads = opt._gradients(None)
    never = {id(p) for p in net.unused.parameters()}
    for p, g, o in zip(arena.params, grads, arena.offsets):
        assert (g is None) == (id(p) in never)
        assert g is None or g.data_ptr() == arena.flat_grad.data_ptr() + 4 * o


def test_a_present_set_is_needed_by_its_entry_point():
    import ctypes as C

    import __graft_entry__ as g
    g.build()
    from mqgan_amd import _lib
    lib = _lib.load()
    sizes = (C.c_int64 * 1)(300)
    d = _lib.AdamwDesc(n_tensors=1, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0, grad_scale=1.0, seed=0)
    at = C.c_void_p(4096)
    call = lambda present, n=8: lib.mq_adamw_step_present(C.byref(d), sizes, at, (C.c_void_p * 1)(4096), None, present, at, at, n, None)  # noqa: E731
    for present in (None, C.c_void_p(4098)):
        assert call(present) != 0 and b"present" in lib.mq_last_error()
    assert call(at, n=0) != 0 and b"workspace" in lib.mq_last_error()
