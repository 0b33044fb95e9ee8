"""Clipping under data parallelism: two processes (both on cuda:0, gloo for the exchange) train on their halves of a batch with
Adam(clipnorm=...).  The norm is that of the mean gradient over the ranks, not of a rank's own: both see the norm of one process on the
whole batch, and stay in lock step.

Bars: the mean gradient equals the whole batch's up to the order of sums, 1e-4 of the norm in the first step (64-bit norm, fp32 sums of
2,000 positions a weight); weights as in test_gpu_dist_train.py, where the same steps are compared without clipping."""
import os
import sys

import numpy as np
import pytest

from test_gpu_dist_train import ROOT, _batch, _clips, _free_port

pytestmark = pytest.mark.gpu

BOUND = 5e-3


def _train(rank, world, n):
    """Losses are not looked at: the norms of three steps and the weights behind them, of ranks [rank, rank + n) of the batch."""
    from layers import Adam, GeneratorCore, GeneratorModel
    from oracle import ref_numpy as rn
    core = GeneratorCore((16, 16, 3), dtype="fp32", device=0)
    core.set_tensors(list(rn.make_weights(seed=7).items()))
    m = GeneratorModel(core, "FRVSR")
    m.compile(loss=["mean_squared_error"] * 2, loss_weights=[1., 1.], optimizer=Adam(lr=1e-4, clipnorm=BOUND))
    a, b, c, hr = _batch(2 * world, 16, 16)
    sl = slice(2 * rank, 2 * (rank + n))
    norms = []
    for _ in range(2):
        m.train_on_batch([a[sl], b[sl], c[sl]], [hr[sl], a[sl]])
        norms.append(core.ctx(1).grad_norm())
    m.train_on_clips(_clips(world)[rank:rank + n])
    norms.append(core.ctx(1).grad_norm())
    return norms, [x.copy() for x in m.get_weights()]


def _worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK="0",
                      SR_DIST_BACKEND="gloo")
    for p in (ROOT, os.path.join(ROOT, "super-resolution_amd")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import torch.distributed as dist
    out.put((rank, *_train(rank, world, 1)))
    dist.barrier()
    dist.destroy_process_group()


def test_two_ranks_clip_by_the_norm_of_their_mean_gradient():
    import torch.multiprocessing as mp
    world = 2
    spawn = mp.get_context("spawn")
    q, port = spawn.Queue(), _free_port()
    procs = [spawn.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = sorted([q.get(timeout=240) for _ in range(world)], key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    norms, weights = _train(0, world, world)
    own, _ = _train(0, world, 1)
    assert min(norms) > 2 * BOUND                                                # every step clips
    assert abs(own[0] - norms[0]) > 1e-3 * norms[0]                              # a rank's own norm is another
    for _, n, w in got:
        assert abs(n[0] - norms[0]) <= 1e-4 * norms[0] and np.allclose(n, norms, rtol=1e-2), (n, norms)
        d = np.concatenate([np.abs(x - y).ravel() for x, y in zip(w, weights)])
        assert d.mean() <= 0.01 * 3e-4 and np.quantile(d, 0.999) <= 0.5 * 3e-4, (d.mean(), d.max())
    assert got[0][1] == got[1][1]
    for x, y in zip(got[0][2], got[1][2]):
        np.testing.assert_array_equal(x, y)
