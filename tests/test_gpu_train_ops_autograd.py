"""residual_norm, residual_norm_bwd, grad_norm and clip_grads beside torch's autograd: nothing that it needs to know is lost in silence."""
import pytest
import torch

from test_gpu_residual_norm import BF16, F32, case, expect_bwd, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def test_tensors_that_require_grad_are_refused_while_gradients_are_recorded(sh):
    C = 48
    c = case(1, (9,), C, F32, BF16, "element")
    fwd = ["x", "y", "gate", "post_gain", "post_bias", "pre_gain", "pre_bias"]
    bwd = ["x", "y", "dh", "dn", "gate", "post_gain", "post_bias", "pre_gain"]
    call = {"forward": lambda v: sh.residual_norm(*[v[k] for k in fwd]), "backward": lambda v: sh.residual_norm_bwd(*[v[k] for k in bwd])}
    for which, names in (("forward", fwd), ("backward", bwd)):
        call[which](c)
        for k in names:
            v = dict(c, **{k: c[k].clone().requires_grad_(True)})
            with pytest.raises(ValueError, match="requires grad"):
                call[which](v)
            with pytest.raises(ValueError, match="requires grad"):
                call[which](dict(c, **{k: v[k] * 1}))                # not a leaf
            with torch.no_grad():
                got = call[which](v)
            assert all(a is None or not a.requires_grad for a in got)
            with torch.inference_mode():
                call[which](v)
    for out in ("h", "n"):
        t = torch.zeros(9, C, device="cuda", dtype=F32 if out == "h" else BF16).requires_grad_(True)
        with pytest.raises(ValueError, match="requires grad"):
            sh.residual_norm(c["x"], c["y"], **{out: t})


def test_as_a_function_of_autograd(sh):
    """The way the message names: forward and backward in a torch.autograd.Function."""
    class Block(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y, gate, post_gain, pre_gain):
            h, n = sh.residual_norm(x, y, gate=gate, post_gain=post_gain, pre_gain=pre_gain, gate_act="sigmoid", scale=0.7, eps=1e-5)
            ctx.save_for_backward(h, y, gate, post_gain, pre_gain)
            return h, n

        @staticmethod
        def backward(ctx, dh, dn):
            h, y, gate, post_gain, pre_gain = ctx.saved_tensors
            g = sh.residual_norm_bwd(h, y, dh, dn, gate=gate, post_gain=post_gain, pre_gain=pre_gain, gate_act="sigmoid", scale=0.7, eps=1e-5)
            return g.dx, g.dy, g.dgate, g.post_gain, g.pre_gain

    C, lead = 72, (3, 50)
    c = case(2, lead, C, F32, F32, 3, bias=False)
    leaf = {k: c[k].clone().requires_grad_(True) for k in ("x", "y", "gate", "post_gain", "pre_gain")}
    h, n = Block.apply(*leaf.values())
    ((h * c["dh"]).sum() + (n * c["dn"]).sum()).backward()
    want = expect_bwd(dict(c, x=h.detach()), "both", "rms", "sigmoid", 0.7, 1e-5)
    for k, name in (("x", "dx"), ("y", "dy"), ("gate", "dgate"), ("post_gain", "post_gain"), ("pre_gain", "pre_gain")):
        ref, mag = want[name]
        within(leaf[k].grad.reshape(ref.shape), ref, mag, 320, name)
