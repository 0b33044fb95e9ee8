"""residual_norm and residual_norm_bwd where inputs are at an edge, and without the gradients of biases.

Formulas, magnitudes and tolerances are those of test_gpu_residual_norm.py: eps_T / 2 of the value, plus K * 2^-24 of the formula with
every term replaced by its magnitude.  K = 256 for what a row's own values give; a sum over rows adds its chain, which for the
shapes here is at most 25 rows of a team, 8 slices and 18 levels of joining: 51 roundings more, K = 320."""
import pytest
import torch

import test_gpu_residual_norm as base
from test_gpu_residual_norm import BF16, F16, F32, TYPES, case, expect_bwd, randn, within

pytestmark = pytest.mark.gpu

K = 320


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("lead,gate", [((2, 0), (2,)), ((2, 0), (2, 1)), ((0, 5), (3,)), ((0,), (1,)), ((3, 0, 4), (3, 1, 1)), ((0, 5), (0,))])
def test_gate_gradient_of_no_rows_is_zero(sh, dt, lead, gate):
    """The sum over no positions, where the gate has rows and the stream has none."""
    C = 64
    x = torch.empty(*lead, C, dtype=dt, device="cuda")
    g = randn(1, *gate, C).to(dt)
    torch.cuda.synchronize()
    for i in range(2):
        dirty = [torch.full((*gate, C), 7.0, dtype=dt, device="cuda") for _ in range(6)]      # what the allocator hands out next
        del dirty
        got = sh.residual_norm_bwd(x, x, x, x, gate=g, bias_grads=True)
        assert got.dgate.shape == g.shape and got.dgate.dtype == dt and not got.dgate.any()
        assert got.dx.shape == got.dy.shape == x.shape and not any(bool(v.any()) for v in got[3:])


def check_gains_only(sh, c, norms, act="sigmoid", scale=0.7, eps=1e-5):
    """An rms norm without the gradients of biases: kernels of their own."""
    want = {k: v for k, v in expect_bwd(c, norms, "rms", act, scale, eps).items() if not k.endswith("bias")}
    got = sh.residual_norm_bwd(c["x"], c["y"], c["dh"], c["dn"] if norms != "post" else None, gate=c["gate"], post_gain=c["post_gain"],
                               post_bias=c["post_bias"], pre_gain=c["pre_gain"], norms=norms, kind="rms", gate_act=act, scale=scale, eps=eps)
    for name, v in got._asdict().items():
        assert (v is None) == (name not in want), name
        if v is not None:
            ref, mag = want[name]
            within(v.reshape(ref.shape), ref, mag, K, name)


@pytest.mark.parametrize("C", [1, 3, 8, 33, 64, 65, 250, 256, 511, 512, 513, 520, 771, 1000, 1541, 2048, 4095, 4097, 5000, 8191, 8192])
@pytest.mark.parametrize("types", range(5))
def test_gains_only(sh, C, types):
    """Few rows (one workgroup) and more, no gate, a gate for each element, one gate row, a gate row for half of the rows."""
    ts, tb = TYPES[types]
    for i, (rows, gate) in enumerate([(2, None), (2, "element"), (700, None), (700, "element"), (700, 1), (700, 2)]):
        j = i + C + types
        check_gains_only(sh, case(j, (rows,), C, ts, tb, gate, ["both", "post", "pre"][j % 3], bias=j % 2 == 0, gains=j % 5 != 0), ["both", "post", "pre"][j % 3],
                         ["linear", "sigmoid"][j // 2 % 2])


@pytest.mark.parametrize("C", [1, 7, 16, 65, 130, 257, 511])
@pytest.mark.parametrize("lead,gate", [((6001,), None), ((6002,), "element"), ((3000, 2), 3000), ((2001, 3), 2001), ((350, 17), 350), ((2, 3001), 2)])
def test_gains_only_rows_within_a_wave(sh, C, lead, gate):
    """Gate rows of a team, of a workgroup, of several workgroups."""
    for ts, tb in ((F32, F32), (BF16, BF16), (F32, F16)):
        check_gains_only(sh, case(C, lead, C, ts, tb, gate), "both")


@pytest.mark.parametrize("C", [2048, 2056, 2060, 2304, 2600, 3060, 3080, 3300])
def test_gains_only_fp32_rows_of_eight_to_thirteen_waves(sh, C):
    """Without a gate a lane has 8 elements of these rows, or 4."""
    for tb in (F32, BF16):
        check_gains_only(sh, case(C, (600,), C, F32, tb, None), "both")


@pytest.mark.parametrize("lead,C,gate", [((1500, 3), 520, 1500), ((600, 2), 4100, 600), ((500, 8), 1001, 500), ((60, 40), 4096, 60), ((2, 1300), 1030, 2)])
def test_gains_only_long_rows_that_share_a_gate(sh, lead, C, gate):
    """Several gate rows to a workgroup, a gate row to one or to several."""
    for ts, tb in ((F32, F32), (BF16, BF16)):
        check_gains_only(sh, case(3, lead, C, ts, tb, gate), "both")


def far_gates(c, rows, C, act):
    """gate_of of test_gpu_residual_norm.py without the cancellation of 1 - sigmoid(g)."""
    g = c["gate"].double().reshape(-1, C)
    g = g.repeat_interleave(rows // g.shape[0], 0)
    return torch.sigmoid(g), torch.sigmoid(g) * torch.sigmoid(-g)


@pytest.mark.parametrize("C", [24, 65, 600, 4100])
@pytest.mark.parametrize("lead,gate", [((5,), "element"), ((900,), "element"), ((4, 2), 4), ((1500, 2), 1500), ((3000, 2), 3000), ((90, 40), 90), ((2, 700), 2)])
def test_gradient_of_far_gates(sh, monkeypatch, C, lead, gate):
    """The slope of a sigmoid far out is exp(-|g|), however close to 1 the sigmoid itself is: the gradient keeps its precision there.
    The slope is made of an exponential (2 ulp), a reciprocal (1 ulp), a sum and two products, well inside of K."""
    monkeypatch.setattr(base, "gate_of", far_gates)
    for ts, tb in ((F32, F32), (F32, BF16)):
        c = case(7, lead, C, ts, tb, gate)
        steps = torch.tensor([0.0, 2.0, 5.0, 8.0, 12.0, 16.0, 16.625, 17.0, 20.0, 40.0, 80.0], device="cuda")
        g = steps.repeat_interleave(2) * torch.tensor([1.0, -1.0], device="cuda").repeat(len(steps))
        c["gate"] = g.repeat(c["gate"].numel() // len(g) + 1)[:c["gate"].numel()].reshape(c["gate"].shape).to(tb)
        for kind, bias in (("rms", False), ("layer", True)):
            want = expect_bwd(c, "both", kind, "sigmoid", 0.7, 1e-5)
            got = sh.residual_norm_bwd(c["x"], c["y"], c["dh"], c["dn"], gate=c["gate"], post_gain=c["post_gain"], post_bias=c["post_bias"],
                                       pre_gain=c["pre_gain"], kind=kind, gate_act="sigmoid", scale=0.7, eps=1e-5, bias_grads=bias)
            for name, v in got._asdict().items():
                if v is not None:
                    ref, mag = want[name]
                    within(v.reshape(ref.shape), ref, mag, K, name)


@pytest.mark.parametrize("strided", [False, True])
def test_shapes_of_outputs(sh, strided):
    """Tensors that hold the stream's rows in other leading dimensions: h and n come in the stream's shape, dy in y's."""
    C = 40
    c = case(5, (12,), C, F32, BF16)
    wide = {k: torch.zeros(12, 3 * C, device="cuda", dtype=c[k].dtype) for k in ("x", "y", "dh", "dn")}
    v = {}
    for k, w in wide.items():
        w[:, :C].copy_(c[k])
        v[k] = (w[:, :C] if strided else c[k]).unflatten(0, (12,) if k in ("y", "dn") else (3, 4))
    h, n = sh.residual_norm(v["x"], v["y"])
    flat = sh.residual_norm(c["x"], c["y"])
    assert h.shape == n.shape == (3, 4, C) and torch.equal(h.view(12, C), flat[0]) and torch.equal(n.view(12, C), flat[1])
    g = sh.residual_norm_bwd(h, v["y"], v["dh"], v["dn"])
    assert g.dx.shape == (3, 4, C) and g.dy.shape == (12, C)
    g = sh.residual_norm_bwd(h, None, v["dh"], v["dn"], norms="pre", branch=True)
    assert g.dx.shape == g.dy.shape == (3, 4, C) and g.dy.dtype == BF16
