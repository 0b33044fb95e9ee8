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


def test_what_a_call_writes_counts_as_changed(sh):
    """A backward pass that wanted the old contents is refused, as after any in-place operation, and not computed from the new ones."""
    C = 48
    c = case(3, (9,), C, F32, F32)
    w = torch.ones(9, C, device="cuda", requires_grad=True)
    mine = lambda k: c[k].clone()
    calls = {
        "h": lambda t: sh.residual_norm(t, mine("y"), h=t), "n": lambda t: sh.residual_norm(mine("x"), t, n=t),
        "dx": lambda t: sh.residual_norm_bwd(mine("x"), mine("y"), t, mine("dn"), dx=t), "dy": lambda t: sh.residual_norm_bwd(mine("x"), mine("y"), mine("dh"), t, dy=t),
        "a view": lambda t: sh.residual_norm(t[2:5], mine("y")[2:5], h=t[2:5]),
        "clipped": lambda t: sh.clip_grads([t], 1e-3), "a clipped view": lambda t: sh.clip_grads([t[2:5]], 1e-3),
        "a list's": lambda t: sh.clip_grads(sh.TensorList([mine("y"), t]), 1e-3), "a list's view": lambda t: sh.clip_grads(sh.TensorList([t[0], t[4]]), 1e-3),
        "out": lambda t: sh.clip_grads([mine("x")], 1e-3, out=[t]), "a list's out": lambda t: sh.clip_grads([mine("x")], 1e-3, out=sh.TensorList([t])),
    }
    for name, call in calls.items():
        t = mine("x")
        lost = (w * t).sum()
        with torch.no_grad():
            call(t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            lost.backward()
            print(name)
    for call in (lambda t: sh.residual_norm(t, mine("y")), lambda t: sh.residual_norm(mine("x"), t), lambda t: sh.grad_norm([t]),
                 lambda t: sh.clip_grads([t], 1e-3, out=[mine("x")]), lambda t: sh.residual_norm_bwd(mine("x"), mine("y"), t, mine("dn"))):
        t = mine("x")                            # only read: the backward pass goes ahead
        kept = (w * t).sum()
        call(t)
        kept.backward()
        assert torch.equal(w.grad, t)
        w.grad = None
    with torch.inference_mode():                 # tensors without a count
        t = torch.ones(9, C, device="cuda")
    sh.residual_norm(t, mine("y"), h=t)
    sh.clip_grads([t], 1e-3)
    with torch.inference_mode():
        sh.clip_grads(sh.TensorList([t, t[:0]]), 1e-3)
