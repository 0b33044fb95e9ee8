"""What the entry points on device tensors refuse before they touch a GPU (include/sr_hip.h sr_op_residual_norm*, sr_tensors_*,
sr_op_grad_norm, sr_op_clip_grads), through the C ABI: a call that passes every check fails with "no HIP device" on a machine
without one.  The addresses are never read here."""
import ctypes as C

import pytest

import sr_hip

P = 1 << 20                    # addresses: 1 MiB apart


class Desc(C.Structure):
    _fields_ = ([("rows", C.c_int64), ("rows_per_gate", C.c_int64)]
                + [(n, C.c_int64) for n in ("ldx", "ldy", "ldg", "ldh", "ldn", "lddh", "lddn", "lddx", "lddy", "lddg")]
                + [(n, C.c_int32) for n in ("channels", "stream_type", "branch_type", "kind", "norms", "gate_act")]
                + [("scale", C.c_float), ("eps", C.c_float)])


def desc(**kw):
    d = dict(rows=4, rows_per_gate=1, channels=16, stream_type=0, branch_type=0, kind=0, norms=3, gate_act=0, scale=1.0, eps=1e-6)
    d.update({n: 16 for n in ("ldx", "ldy", "ldg", "ldh", "ldn", "lddh", "lddn", "lddx", "lddy", "lddg")})
    d.update(kw)
    return Desc(**d)


def forward(d, x=P, y=2 * P, gate=None, pw=None, pb=None, qw=None, qb=None, h=3 * P, n=4 * P):
    rc = sr_hip.lib().sr_op_residual_norm(0, C.byref(d) if d is not None else None, x, y, gate, pw, pb, qw, qb, h, n, None)
    return rc, sr_hip._err(None)


def backward(d, h=P, y=2 * P, gate=None, dh=3 * P, dn=4 * P, dx=5 * P, dy=6 * P, dgate=None, vec=(7 * P, None, 8 * P, None), ws=16 * P, size=1 << 20,
             gains=(None, None, None)):
    rc = sr_hip.lib().sr_op_residual_norm_bwd(0, C.byref(d) if d is not None else None, h, y, gate, *gains, dh, dn, dx, dy, dgate, *vec, ws, size, None)
    return rc, sr_hip._err(None)


@pytest.fixture(autouse=True)
def no_gpu():
    if sr_hip.device_count() > 0:
        pytest.skip("made-up addresses: only where no GPU can read them")


def test_complete_calls_get_as_far_as_the_device():
    for got in (forward(desc()), forward(desc(), gate=5 * P), forward(desc(), h=P, n=2 * P), backward(desc()),
                backward(desc(), gate=9 * P, dgate=10 * P), forward(desc(norms=2), y=None, h=None)):
        assert got[0] == -4 and "no HIP device" in got[1], got


BAD_DESC = [dict(rows=-1), dict(rows=2_000_000_001), dict(channels=0), dict(channels=8193), dict(stream_type=3), dict(branch_type=-1),
            dict(stream_type=1), dict(stream_type=1, branch_type=2), dict(kind=2), dict(norms=0), dict(norms=4), dict(gate_act=2),
            dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("kw", BAD_DESC, ids=str)
def test_bad_descriptors(kw):
    need = C.c_size_t()
    assert forward(desc(**kw))[0] == -1
    assert backward(desc(**kw))[0] == -1
    assert sr_hip.lib().sr_op_residual_norm_bwd_workspace(C.byref(desc(**kw)), 0, C.byref(need)) == -1


def test_bad_calls_forward():
    assert forward(None)[0] == -1
    for kw in (dict(x=None), dict(h=None), dict(n=None), dict(y=None), dict(x=P + 2), dict(pw=P + 2)):
        assert forward(desc(), **kw)[0] == -1, kw
    for kw in (dict(ldx=15), dict(ldh=-16), dict(ldn=0), dict(ldx=1 << 41)):
        assert forward(desc(**kw))[0] == -1, kw
    for rpg in (0, -1, 3, 5):
        assert forward(desc(rows_per_gate=rpg), gate=5 * P)[0] == -1
    assert forward(desc(rows_per_gate=3))[0] == -4                       # not looked at without a gate
    for kw in (dict(h=P + 64), dict(h=2 * P - 4), dict(n=3 * P), dict(n=3 * P + 64), dict(h=P, n=P), dict(pw=3 * P + 128), dict(qb=4 * P - 60)):
        rc, msg = forward(desc(), **kw)
        assert rc == -1 and "overlaps" in msg, kw
    assert forward(desc(ldx=40, ldh=40), x=P, h=P + 64)[0] == -4          # column blocks of one matrix
    assert forward(desc(ldx=40, ldh=40), x=P, h=P + 60)[0] == -1
    assert forward(desc(ldx=40, ldh=40), x=P, h=P + 100)[0] == -1         # wraps into the next row
    assert forward(desc(ldx=40, ldh=44), x=P, h=P + 64)[0] == -1
    assert forward(desc(rows_per_gate=2), gate=3 * P)[0] == -1            # a shared gate under h
    assert forward(desc(rows_per_gate=1), gate=3 * P)[0] == -4


def test_bad_calls_backward():
    assert backward(None)[0] == -1
    for kw in (dict(h=None), dict(dn=None), dict(dx=None), dict(y=None), dict(dy=None), dict(dgate=9 * P)):
        assert backward(desc(), **kw)[0] == -1, kw
    many = desc(rows=4000)
    assert backward(many)[0] == -4
    for kw in (dict(ws=None), dict(ws=16 * P + 8), dict(size=16), dict(ws=5 * P), dict(ws=7 * P), dict(gains=(None, None, 16 * P))):
        assert backward(many, **kw)[0] == -1, kw
    assert backward(desc(), ws=None, size=0)[0] == -4                    # a few rows: no workspace
    assert backward(desc(), dh=None)[0] == -4
    assert backward(desc(norms=1), dh=None, vec=(None,) * 4)[0] == -1
    assert backward(desc(norms=1), vec=(7 * P, None, 8 * P, None))[0] == -1      # no pre norm, so no gradient of its gain
    assert backward(desc(norms=2), vec=(None, 7 * P, None, None))[0] == -1
    for kw in (dict(dx=P + 4), dict(dy=5 * P), dict(dx=7 * P - 4), dict(vec=(7 * P, 7 * P + 32, None, None)),
               dict(gains=(5 * P, None, None)), dict(gains=(None, None, 8 * P))):
        rc, msg = backward(desc(), **kw)
        assert rc == -1 and "overlaps" in msg, kw
    assert backward(desc(), dx=P, dy=2 * P)[0] == -4
    assert backward(desc(), dx=3 * P, dy=4 * P)[0] == -4
    need = C.c_size_t()
    assert sr_hip.lib().sr_op_residual_norm_bwd_workspace(C.byref(desc(rows=0)), 0, C.byref(need)) == 0 and need.value == 0
    assert backward(desc(rows=0), ws=None, size=0)[0] == -4


def tensors(*t):
    arr = (sr_hip._TensorDesc * max(len(t), 1))(*[sr_hip._TensorDesc(data=a, count=n, type=k) for a, n, k in t])
    h = C.c_void_p()
    rc = sr_hip.lib().sr_tensors_create(C.byref(h), 0, len(t), arr)
    return rc, h


def test_tensor_lists():
    l = sr_hip.lib()
    for bad in ((None, 5, 0), (P + 2, 5, 0), (P + 1, 5, 1), (P, -1, 0), (P, 5, 3), (P, (1 << 40) + 1, 1)):
        rc, h = tensors((P, 4, 0), bad)
        assert rc == -1 and not h.value, bad
    assert l.sr_tensors_create(None, 0, 0, None) == -1
    h = C.c_void_p()
    assert l.sr_tensors_create(C.byref(h), 0, -1, None) == -1 and l.sr_tensors_create(C.byref(h), 0, 2, None) == -1
    assert l.sr_tensors_create(C.byref(h), -1, 0, None) == -1
    assert l.sr_tensors_destroy(None) == 0 and l.sr_tensors_upload(None) == -1
    rc, h = tensors((None, 0, 0), (P, 100_000, 1), (2 * P, 3, 2))
    assert rc == 0
    need = C.c_size_t()
    assert l.sr_tensors_workspace(h, C.byref(need)) == 0 and 8 * 14 <= need.value <= 8 * (4096 + 3)
    W, N = 8 * P, 9 * P
    assert l.sr_op_grad_norm(h, 1.0, N, None, W, need.value, None) == -4              # as far as the device
    for args in ((None, 1.0, N, None, W, need.value, None), (h, 0.0, N, None, W, need.value, None), (h, 1.0, None, None, W, need.value, None),
                 (h, 1.0, N, None, None, need.value, None), (h, 1.0, N, None, W + 4, need.value, None), (h, 1.0, N, None, W, need.value - 8, None),
                 (h, 1.0, N, N, W, need.value, None), (h, 1.0, W + 8, None, W, need.value, None), (h, 1.0, P + 8, None, W, need.value, None),
                 (h, 1.0, N, W, W, need.value, None), (h, 1.0, N, None, P, need.value, None), (h, 1.0, N, 2 * P, W, need.value, None)):
        assert l.sr_op_grad_norm(*args) == -1, args
    assert l.sr_op_clip_grads(h, None, 1.0, 1.0, N, W, need.value, None) == -4 and l.sr_tensors_upload(h) == -4
    for m, s in ((0.0, 1.0), (-1.0, 1.0), (float("nan"), 1.0), (1.0, -1.0), (1.0, float("nan"))):
        assert l.sr_op_clip_grads(h, None, m, s, N, W, need.value, None) == -1
    for other in (((P, 100_000, 1), (2 * P, 3, 2)), ((None, 0, 0), (P, 99_999, 1), (2 * P, 3, 2)), ((None, 0, 0), (P, 100_000, 2), (2 * P, 3, 2)),
                  ((None, 0, 0), (2 * P, 100_000, 1), (P, 3, 2)), ((None, 0, 0), (P + 2, 100_000, 1), (4 * P, 3, 2)),
                  ((None, 0, 0), (4 * P, 100_000, 1), (4 * P + 10, 3, 2)), ((None, 0, 0), (W, 100_000, 1), (4 * P, 3, 2))):
        rc, o = tensors(*other)
        assert rc == 0 and l.sr_op_clip_grads(h, o, 1.0, 1.0, N, W, need.value, None) == -1, other
        l.sr_tensors_destroy(o)
    rc, o = tensors((None, 0, 0), (P, 100_000, 1), (4 * P, 3, 2))                     # one in place, one not
    assert l.sr_op_clip_grads(h, o, 1.0, 1.0, N, W, need.value, None) == -4
    l.sr_tensors_destroy(o)
    l.sr_tensors_destroy(h)


def test_python_side_needs_a_gpu():
    import torch
    with pytest.raises(ValueError, match="no CPU fallback"):
        sr_hip.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(ValueError, match="no CPU fallback"):
        sr_hip.TensorList([torch.zeros(4)])


def test_adam_clipnorm_argument():
    from layers import Adam
    assert Adam().clipnorm == 0.0 and Adam(clipnorm=None).clipnorm == 0.0 and Adam(clipnorm=2).clipnorm == 2.0
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            Adam(clipnorm=bad)
    l = sr_hip.lib()
    v = C.c_float()
    assert l.sr_train_set_clipnorm(None, 1.0) == -1 and l.sr_disc_set_clipnorm(None, 1.0) == -1
    assert l.sr_train_grad_norm(None, C.byref(v)) == -1 and l.sr_disc_grad_norm(None, C.byref(v)) == -1
