"""Two residual blocks with norms, gate and scale, their gradients and the clipping of all of them, as a training step runs them:
residual_norm and residual_norm_bwd around the framework's own conv3x3 and conv3x3_bwd, then clip_grads, against torch autograd in
float64.  Bar: 1e-3 of each tensor's largest gradient -- four passes through a convolution at 2e-4 each (tests/test_gpu_train.py); the
norms' own error (tests/test_gpu_residual_norm.py) is far below it."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

B, H, W, C = 2, 8, 12, 64


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def layer(v, gain):
    return F.layer_norm(v, (C,), eps=1e-6) * gain


@pytest.mark.parametrize("share", [0.25, 10.0])
def test_step(sh, share):
    rng = np.random.default_rng(5)
    new = lambda *s, m=0.0, d=1.0: rng.standard_normal(s).astype(np.float32) * d + np.float32(m)
    p = {"x": new(B, H, W, C), "g0": new(C, m=1, d=.2), "w0": new(3, 3, C, C, d=.05), "b0": new(C, d=.1), "gate": new(B, C),
         "p1": new(C, m=1, d=.2), "g1": new(C, m=1, d=.2), "w1": new(3, 3, C, C, d=.05), "b1": new(C, d=.1), "p2": new(C, m=1, d=.2)}
    R = new(B, H, W, C)
    # the step on the GPU
    t = {k: torch.from_numpy(v).cuda() for k, v in p.items()}
    dev = lambda a: torch.from_numpy(a).cuda()
    num = lambda a: a.cpu().numpy()
    kw = dict(kind="layer", scale=0.5)
    _, n0 = sh.residual_norm(t["x"], pre_gain=t["g0"], norms="pre", kind="layer")
    y0 = dev(sh.conv3x3(num(n0), p["w0"], p["b0"]))
    h1, n1 = sh.residual_norm(t["x"], y0, gate=t["gate"], post_gain=t["p1"], pre_gain=t["g1"], gate_act="sigmoid", **kw)
    y1 = dev(sh.conv3x3(num(n1), p["w1"], p["b1"]))
    h2, _ = sh.residual_norm(h1, y1, post_gain=t["p2"], norms="post", **kw)
    d2 = sh.residual_norm_bwd(h2, y1, dev(R), post_gain=t["p2"], norms="post", **kw)
    dn1, dw1, db1 = sh.conv3x3_bwd(num(n1), p["w1"], num(d2.dy))
    d1 = sh.residual_norm_bwd(h1, y0, d2.dx, dev(dn1), gate=t["gate"], post_gain=t["p1"], pre_gain=t["g1"], gate_act="sigmoid", **kw)
    dn0, dw0, db0 = sh.conv3x3_bwd(num(n0), p["w0"], num(d1.dy))
    d0 = sh.residual_norm_bwd(t["x"], None, d1.dx, dev(dn0), pre_gain=t["g0"], norms="pre", kind="layer")
    grads = {"x": d0.dx, "g0": d0.pre_gain, "w0": dev(dw0), "b0": dev(db0), "gate": d1.dgate, "p1": d1.post_gain, "g1": d1.pre_gain,
             "w1": dev(dw1), "b1": dev(db1), "p2": d2.post_gain}
    # the same in float64
    q = {k: torch.from_numpy(v).double().requires_grad_(True) for k, v in p.items()}
    conv = lambda v, w, b: F.conv2d(v.permute(0, 3, 1, 2), w.permute(3, 2, 0, 1), b, padding=1).permute(0, 2, 3, 1)
    a0 = conv(layer(q["x"], q["g0"]), q["w0"], q["b0"])
    a1 = q["x"] + 0.5 * torch.sigmoid(q["gate"])[:, None, None] * layer(a0, q["p1"])
    a2 = a1 + 0.5 * layer(conv(layer(a1, q["g1"]), q["w1"], q["b1"]), q["p2"])
    (a2 * torch.from_numpy(R).double()).sum().backward()
    assert float((h2.cpu().double() - a2.detach()).abs().max()) <= 1e-3 * float(a2.detach().abs().max())
    want = {k: v.grad for k, v in q.items()}
    for k, g in grads.items():
        assert float((g.cpu().double() - want[k]).abs().max()) <= 1e-3 * float(want[k].abs().max()), k
    # and clipped by their global norm
    total = float(sum((v ** 2).sum() for v in want.values())) ** 0.5
    norm = sh.clip_grads(list(grads.values()), share * total)
    assert abs(float(norm) - total) <= 1e-3 * total
    for k, g in grads.items():
        ref = want[k] * min(1.0, share)
        assert float((g.cpu().double() - ref).abs().max()) <= 2e-3 * float(ref.abs().max()), k
