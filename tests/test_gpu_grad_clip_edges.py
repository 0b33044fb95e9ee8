"""clip_grads and clipped optimizer steps at the ends of fp32's range, against float64.  Tolerances as in test_gpu_grad_clip.py: the
factor is 64 bits rounded to fp32, or with its scale two roundings more, then a product and the rounding to the tensor's type."""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_gpu_grad_clip import BF16, F32, TINY, U, check_clipped, norm64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def uniform(seed, n, lo, hi):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(n, device="cuda").uniform_(lo, hi, generator=g)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("size,n,max_norm,scale", [
    (1e38, 1_000_003, 1.0, 1.0),          # the factor is 1e-41: 13 bits of an fp32 subnormal
    (3e38, 70_001, 1e-4, 1.0),            # 1e-45: the last one
    (3e38, 70_001, 1e-9, 0.125),          # below them all
    (1e12, 9_001, 1.0, 1e35),             # the factor alone is below fp32, with its scale it is 1e-14
    (1e12, 9_001, 1e30, 1e35),            # the norm is above fp32
    (1.0, 9_001, 1e-36, 1.0), (1e-30, 9_001, 1e-37, 1e-5), (1e30, 300, 1e-30, 1e-20),
    (1e38, 5_001, 1e38, 1e-39), (2.0, 5_001, 1e38, 1e-39)])                # a subnormal scale, clipped and not
def test_factors_beyond_fp32(sh, dt, size, n, max_norm, scale):
    scale, max_norm = ctypes.c_float(scale).value, ctypes.c_float(max_norm).value
    t = (uniform(1, n, -1.0, 1.0) * size).to(dt)
    want = norm64([t]) * scale
    for upload in (True, False):
        out = torch.full_like(t, 9.0)
        norm = float(sh.clip_grads(sh.TensorList([t], upload=upload), max_norm, scale=scale, out=[out]))
        assert abs(norm - want) <= want * (U + 1e-12) + TINY[F32] / 2 if want < 3.4e38 else math.isinf(norm)
        check_clipped(out, t, want, max_norm, scale)
        mine = t.clone()
        sh.clip_grads([mine], max_norm, scale=scale)
        assert torch.equal(mine, out)


def test_subnormal_gradients_pass_as_they_are(sh):
    t = torch.arange(1, 3000, device="cuda", dtype=torch.int32).view(F32)            # 2^-149 and up
    out = torch.empty_like(t)
    sh.clip_grads([t], 1.0, out=[out])
    assert torch.equal(out, t)
    sh.clip_grads([t], 1.0, scale=0.5, out=[out])
    assert torch.equal(out, t * 0.5)


@pytest.mark.parametrize("size,max_norm,scale", [(1e37, 1.0, 1.0), (1e37, 1e-6, 0.25), (1e12, 1.0, 1e35), (1e-3, 1e-4, 1.0 / 3)])
def test_clipped_step_is_the_step_of_clipped_gradients(sh, weights7, size, max_norm, scale):
    """Bit for bit, as both take the same partial sums and the same factor."""
    got = []
    for clipped in (True, False):
        c = sh.Context(16, 24, max_batch=1, dtype="fp32")
        c.load_weights(weights7)
        c.train_grads(*[np.zeros((1, k * 16, k * 24, 3), np.float32) for k in (1, 1, 4, 4)])        # a step wants to have been prepared
        for step in range(2):
            g = uniform(step, c.param_count(), -1.0, 1.0) * size
            c.set_clipnorm(max_norm if clipped else 0)
            if not clipped:
                sh.clip_grads([g], max_norm, scale=scale)
            torch.cuda.synchronize()
            c.train_apply(d_grads=g.data_ptr(), grad_scale=scale if clipped else 1.0)
        got.append(c.get_weights())
        c.close()
    moved = 0
    for (n, x), (_, y) in zip(*got):
        assert (x == y).all(), n
        moved += int((x != weights7[n]).sum())
    assert moved > 0


@pytest.mark.parametrize("n", [900, 901, 2000])
def test_norm_of_each_of_many_tensors_without_records(sh, n):
    """Lists made for one call and captured ones: the tensors' partial sums travel in the kernel arguments, 900 tensors a launch."""
    ts = [uniform(i, 1 + i * 7 % 50, -1.0, 1.0) for i in range(n)]
    norm, each = sh.grad_norm(sh.TensorList(ts), per_tensor=True)
    got = sh.grad_norm(ts, per_tensor=True)
    assert torch.equal(got[0], norm) and torch.equal(got[1], each)
    want = torch.stack([(t.double() ** 2).sum().sqrt() for t in ts])
    assert float(((each.double() - want).abs() - want * (U + 1e-12)).max()) <= 0
    lst = sh.TensorList(ts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sh.grad_norm(lst, per_tensor=True)
    for i in range(3):
        for t in ts:
            t.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = sh.grad_norm(ts, per_tensor=True)
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1]) and torch.equal(eager[1], each * 0.5 ** (i + 1))
