"""Data-parallel ranks that hold the same averaged gradients clip them alike: two
processes on one GPU, each with gradients of its own, averaged by GradBucket over
gloo on the host, clipped on the device, stepped."""
import os
import socket

import pytest
import torch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZES = [(7 * 7 * 32, 32), (32,), (25, 32, 5, 5), (1,), (9001,), (3, 0)]
MAX = 0.75


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _params(rank):
    """The same parameters on every rank, a rank's own gradients; one without."""
    g = torch.Generator().manual_seed(11)
    params = [torch.nn.Parameter(torch.randn(s, generator=g)) for s in SIZES]
    g = torch.Generator().manual_seed(100 + rank)
    for p in params[:-1]:
        p.grad = torch.randn(p.shape, generator=g)
    return params


def _clip_and_step(params):
    """(norm, parameters after the step) of host parameters, on the device."""
    from ptamd import clip
    dev = [torch.nn.Parameter(p.detach().cuda()) for p in params]
    for d, p in zip(dev, params):
        d.grad = None if p.grad is None else p.grad.cuda()
    opt = torch.optim.Adam(dev, lr=0.1, fused=True)
    norm = clip.clip_grad_norm_(dev, MAX)
    grads = [d.grad.cpu().numpy().copy() for d in dev if d.grad is not None]
    opt.step()
    return float(norm), grads, [d.detach().cpu().numpy().copy() for d in dev]


def _worker(rank, port, out_q):
    import sys
    sys.path[:0] = [REPO, os.path.join(REPO, "pathtracker-models_amd")]
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist
    from ptamd.dist import GradBucket
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=2)
    params = _params(rank)
    GradBucket(params, "cpu").allreduce_mean()
    out_q.put((rank, _clip_and_step(params)))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_two_ranks_clip_by_the_same_factor():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm device")
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = dict(q.get(timeout=200) for _ in range(2))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    (n0, g0, p0), (n1, g1, p1) = res[0], res[1]
    assert n0 == n1 > MAX
    assert all((a == b).all() for a, b in zip(g0 + p0, g1 + p1))
    # the gradients' mean, clipped: as one process that holds both has it
    shards = [_params(r) for r in range(2)]
    for a, b in zip(*shards):
        if a.grad is not None:
            a.grad = (a.grad + b.grad) / 2
    norm, grads, params = _clip_and_step(shards[0])
    assert norm == n0 and all((a == b).all() for a, b in zip(grads + params, g0 + p0))
