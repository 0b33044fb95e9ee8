"""What the Python side of the gradient operators refuses before it looks for a GPU."""
import numpy as np
import pytest
import torch

import sr_hip


@pytest.mark.parametrize("bad", [None, 1.0, np.zeros(4, np.float32), [torch.zeros(4)]], ids=["None", "number", "array", "list"])
def test_lists_hold_tensors_only(bad):
    """zip(params, grads) with a parameter that had no part in the loss: its gradient is None."""
    for call in (sr_hip.TensorList, sr_hip.grad_norm, lambda t: sr_hip.clip_grads(t, 1.0)):
        for ts in ([bad], [bad, torch.zeros(4)]):
            with pytest.raises(ValueError, match="tensor 0 is not a tensor"):
                call(ts)
    if bad is None:
        with pytest.raises(ValueError, match="leave out what has no gradient"):
            sr_hip.grad_norm([None])


def test_a_bound_below_float32_is_not_taken_for_no_bound():
    from layers import Adam
    with pytest.raises(ValueError, match="clipnorm"):
        Adam(clipnorm=1e-46)
    assert Adam(clipnorm=1e-45).clipnorm == 1e-45 and Adam(clipnorm=0.0).clipnorm == 0.0
    for cls in (sr_hip.Context, sr_hip.Discriminator):
        c = object.__new__(cls)
        c._h = None
        with pytest.raises(ValueError, match="below float32"):
            c.set_clipnorm(1e-46)
