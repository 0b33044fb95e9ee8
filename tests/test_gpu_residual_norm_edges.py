"""residual_norm and residual_norm_bwd where inputs are at an edge."""
import pytest
import torch

from test_gpu_residual_norm import BF16, F16, F32, randn

pytestmark = pytest.mark.gpu


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
