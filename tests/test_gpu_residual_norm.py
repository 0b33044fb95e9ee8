"""residual_norm and residual_norm_bwd (include/sr_hip.h sr_op_residual_norm*) against their formulas in float64.

Tolerances, element by element.  With u = 2^-24 and eps_T = torch.finfo(T).eps, an output differs from the 64-bit value of the
same inputs by at most
    eps_T / 2 * |value| + tiny_T / 2            the one rounding to its type (tiny: the smallest subnormal)
  + K * u * A                                   fp32 arithmetic
where A is the formula with every term replaced by its magnitude (no cancellation) and K counts the roundings that reach an
element: a row sum adds at most 8 values a lane, 6 lane exchanges and 4 between waves (18 roundings); the chain mean, centred value,
variance, reciprocal root (1 ulp), gain, gate (expf 2 ulp, reciprocal 1 ulp), scale, sum has two such row sums and about 20 more
roundings for each norm.  Two norms in a row: K = 2 * (2 * 18 + 20) = 112 < 128 forward; the backward pass goes through both norms
and both of their gradients: K = 256.  Sums over rows add at most R / 1024 + 8 rows in a chain before they are joined in a tree of
at most 16 + 10 levels, which K = 256 covers for the sizes here."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def within(got, want, mag, k, what):
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + TINY[got.dtype] / 2 + k * U * mag
    bad = (got.double() - want).abs() - tol
    assert got.shape == want.shape, what
    assert not got.isnan().any(), what
    if got.numel():
        assert float(bad.max()) <= 0, f"{what}: off by {float((got.double() - want).abs().max()):.3e}, over the bound by {float(bad.max()):.3e}"


def randn(seed, *shape, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale + shift


def case(seed, lead, C, ts, tb, gate=None, norms="both", bias=True, gains=True):
    """Inputs of a call: lead = leading dimensions, gate None, 'element' or a number of gate rows."""
    c = {"x": randn(seed, *lead, C, scale=2.0, shift=0.3).to(ts), "y": randn(seed + 1, *lead, C, scale=0.7, shift=-0.1).to(tb),
         "gate": None}
    if gate is not None:
        c["gate"] = randn(seed + 2, *(lead if gate == "element" else (gate,)), C).to(tb)
    for i, w in enumerate(("post", "pre")):
        on = norms in (w, "both")
        c[w + "_gain"] = randn(seed + 3 + i, C, scale=0.2, shift=1.0) if on and gains else None
        c[w + "_bias"] = randn(seed + 5 + i, C, scale=0.1) if on and bias else None
    c["dh"], c["dn"] = randn(seed + 7, *lead, C).to(ts), randn(seed + 8, *lead, C).to(tb)
    return c


def one_norm(v, gain, bias, layer, eps, mag):
    """hat(v) and gain hat + bias in 64 bits, with their magnitudes; mag >= |v|: the magnitude that v's own error scales with."""
    d = v - v.mean(-1, keepdim=True) if layer else v
    rs = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    hat = d * rs
    m = rs * (mag + mag.mean(-1, keepdim=True))                       # error of the centred value
    m = m + hat.abs() * (1 + rs * torch.sqrt((mag * mag).mean(-1, keepdim=True)))   # ... and of the reciprocal root
    g = torch.ones(v.shape[-1], dtype=torch.float64, device="cuda") if gain is None else gain.double()
    b = 0.0 if bias is None else bias.double()
    return hat, rs, hat * g + b, m * g.abs() + (0.0 if bias is None else b.abs()), m, g


def gate_of(c, rows, C, act):
    if c["gate"] is None:
        one = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        return one, 0 * one
    g = c["gate"].double().reshape(-1, C)
    g = g.repeat_interleave(rows // g.shape[0], 0) if rows else g.reshape(0, C)
    if act == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s)
    return g, torch.ones_like(g)


def expect(c, norms, kind, act, scale, eps):
    C = c["x"].shape[-1]
    x, y = c["x"].double().reshape(-1, C), c["y"].double().reshape(-1, C)
    layer = kind == "layer"
    p, mp = y, y.abs()
    if norms != "pre":
        _, _, p, mp, _, _ = one_norm(y, c["post_gain"], c["post_bias"], layer, eps, y.abs())
    a, _ = gate_of(c, len(x), C, act)
    h = x + scale * a * p
    mh = x.abs() + abs(scale) * a.abs() * mp
    if norms == "post":
        return h, mh, None, None
    _, _, n, mn, _, _ = one_norm(h, c["pre_gain"], c["pre_bias"], layer, eps, mh)
    return h, mh, n, mn


def check_fwd(sh, c, norms, kind, act, scale=0.7, eps=1e-5, **kw):
    h, mh, n, mn = expect(c, norms, kind, act, scale, eps)
    got_h, got_n = sh.residual_norm(c["x"], c["y"], gate=c["gate"], post_gain=c["post_gain"], post_bias=c["post_bias"],
                                    pre_gain=c["pre_gain"], pre_bias=c["pre_bias"], norms=norms, kind=kind, gate_act=act, scale=scale,
                                    eps=eps, **kw)
    C = c["x"].shape[-1]
    within(got_h.reshape(-1, C), h, mh, 128, "h")
    assert (got_n is None) == (norms == "post")
    if n is not None:
        within(got_n.reshape(-1, C), n, mn, 128, "n")
    return got_h, got_n


def hat_bwd(q, mq, hat, mhat, rs, layer):
    out = q - hat * (q * hat).mean(-1, keepdim=True) - (q.mean(-1, keepdim=True) if layer else 0.0)
    mag = mq + mhat * (mq * mhat).mean(-1, keepdim=True) + mq.mean(-1, keepdim=True)
    return rs * out, rs * mag


def expect_bwd(c, norms, kind, act, scale, eps):
    """From h = c['x'] as given: the gradients and their magnitudes."""
    C = c["x"].shape[-1]
    h, y, layer = c["x"].double().reshape(-1, C), c["y"].double().reshape(-1, C), kind == "layer"
    rows = len(h)
    T = c["dh"].double().reshape(-1, C) if c["dh"] is not None else torch.zeros_like(h)
    mT = T.abs()
    out = {}
    if norms != "post":
        dn = c["dn"].double().reshape(-1, C)
        hat, rs, _, _, mhat, g = one_norm(h, c["pre_gain"], None, layer, eps, h.abs())
        out["pre_gain"] = ((dn * hat).sum(0), (dn.abs() * mhat).sum(0))
        out["pre_bias"] = (dn.sum(0), dn.abs().sum(0))
        t, mt = hat_bwd(dn * g, (dn * g).abs(), hat, mhat, rs, layer)
        T, mT = T + t, mT + mt
    out["dx"] = (T, mT)
    p, mp = y, y.abs()
    if norms != "pre":
        hat, rs, p, mp, mhat, g = one_norm(y, c["post_gain"], c["post_bias"], layer, eps, y.abs())
    a, slope = gate_of(c, rows, C, act)
    if c["gate"] is not None:
        dg, mg = scale * slope * p * T, abs(scale) * slope.abs() * mp * mT
        G = c["gate"].numel() // C
        out["dgate"] = (dg.reshape(G, -1, C).sum(1), mg.reshape(G, -1, C).sum(1)) if rows else (dg, mg)
    dp, mdp = scale * a * T, abs(scale) * a.abs() * mT
    if norms != "pre":
        out["post_gain"] = ((dp * hat).sum(0), (mdp * mhat).sum(0))
        out["post_bias"] = (dp.sum(0), mdp.sum(0))
        dp, mdp = hat_bwd(dp * g, mdp * g.abs(), hat, mhat, rs, layer)
    out["dy"] = (dp, mdp)
    return out


def check_bwd(sh, c, norms, kind, act, scale=0.7, eps=1e-5, k=256, **kw):
    want = expect_bwd(c, norms, kind, act, scale, eps)
    got = sh.residual_norm_bwd(c["x"], c["y"], c["dh"], c["dn"] if norms != "post" else None, gate=c["gate"], post_gain=c["post_gain"],
                               post_bias=c["post_bias"], pre_gain=c["pre_gain"], norms=norms, kind=kind, gate_act=act, scale=scale, eps=eps,
                               bias_grads=True, **kw)
    for name, v in got._asdict().items():
        assert (v is None) == (name not in want), name
        if v is not None:
            ref, mag = want[name]
            within(v.reshape(ref.shape), ref, mag, k, name)
    return got


# channels around every border: one lane, a lane's vector, a team, the wave's 512, a workgroup's 8192; odd ones start rows at any address
CHANNELS = [1, 3, 7, 8, 9, 48, 64, 65, 128, 250, 256, 257, 511, 512, 513, 515, 1000, 2048, 4097, 8191, 8192]


@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("types", range(5))
def test_forward(sh, C, types):
    ts, tb = TYPES[types]
    i = CHANNELS.index(C) + types
    lead = [(3, 11), (1,), (2, 4, 5), (70,)][i % 4]
    rows = math.prod(lead)
    gate = [None, "element", lead[0], 1][(i // 2) % 4]
    norms = ["both", "both", "post", "pre"][(i // 3) % 4]
    c = case(C + types, lead, C, ts, tb, gate, norms, bias=i % 3 != 0, gains=i % 5 != 0)
    for kind in ("rms", "layer"):
        check_fwd(sh, c, norms, kind, ["linear", "sigmoid"][i % 2], eps=[1e-5, 1e-3][rows % 2])


@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("types", range(5))
def test_backward(sh, C, types):
    ts, tb = TYPES[types]
    i = CHANNELS.index(C) + 2 * types
    lead = [(3, 41), (1,), (2, 4, 5), (150,)][i % 4]
    gate = [None, "element", lead[0], 1][(i // 2) % 4]
    norms = ["both", "both", "post", "pre"][(i // 3) % 4]
    c = case(C + types, lead, C, ts, tb, gate, norms, bias=i % 3 != 0, gains=i % 5 != 0)
    for kind in ("rms", "layer"):
        check_bwd(sh, c, norms, kind, ["linear", "sigmoid"][i % 2])


@pytest.mark.parametrize("lead,C,gate", [((40, 640), 64, 40), ((7, 1000), 48, 7), ((1500, 3), 64, 1500), ((3000,), 520, 1), ((2, 1300), 1030, 2), ((2100, 2), 521, 2100),
                                         ((600, 2), 4100, 600), ((2, 4, 300), 250, 2), ((500, 8), 1001, 500), ((60, 40), 4096, 60),
                                         ((9, 3000), 20, 9)])
def test_backward_many_rows(sh, lead, C, gate):
    """Several workgroups to a gate row, several gate rows to a workgroup (which then adds to its partial sums), gate rows that are
    whole in one."""
    check_bwd(sh, case(5, lead, C, F32, F32, gate), "both", "layer", "sigmoid")
    check_bwd(sh, case(6, lead, C, BF16, BF16, "element"), "both", "rms", "linear")


@pytest.mark.parametrize("C", [1, 3, 7, 9, 13, 16, 33, 64, 65, 130, 257, 511])
@pytest.mark.parametrize("lead,gate", [((6001,), None), ((6002,), "element"), ((3000, 2), 3000), ((2401, 3), 2401), ((450, 17), 450), ((70, 90), 70),
                                       ((2, 3001), 2)])
def test_backward_rows_within_a_wave(sh, C, lead, gate):
    """More rows than one workgroup takes, of few channels, and gate rows for two rows and for thousands: a team's own, a workgroup's,
    several workgroups'."""
    i = C + lead[-1]
    ts, tb = TYPES[i % 5]
    check_bwd(sh, case(i, lead, C, ts, tb, gate), "both", ["rms", "layer"][i // 2 % 2], "sigmoid")
    check_bwd(sh, case(i, lead, C, F32, F32, gate, bias=False), ["both", "post", "pre"][i % 3], "rms", "linear")


@pytest.mark.parametrize("C,teams", [(5, 256), (16, 256), (64, 64), (250, 16), (500, 8), (700, 1), (4100, 1)])
@pytest.mark.parametrize("gate", [None, "element", 1, 2])
def test_backward_around_one_workgroup(sh, C, teams, gate):
    """Rows up to what one workgroup takes, which leaves the gradients itself, and one more."""
    for rows in (1, 2, teams, teams + 1, 2 * teams, 2 * teams + 2, 3 * teams, 3 * teams + 1):
        if gate == 2 and rows % 2:
            continue
        c = case(rows, (rows,), C, BF16, BF16, gate)
        a = check_bwd(sh, c, "both", "layer", "sigmoid")
        b = check_bwd(sh, c, "both", "layer", "sigmoid")
        for p, q in zip(a, b):
            assert (p is None and q is None) or torch.equal(p, q)


@pytest.mark.parametrize("ts,tb", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_rows_of_a_wider_matrix(sh, ts, tb):
    """Pitches, odd starts, outputs beside inputs in one buffer; what lies between the rows stays as it was."""
    for C in (5, 64, 515, 900):
        c = case(C, (33,), C, ts, tb)
        wide = torch.full((33, 4 * C + 7), -5.0, dtype=ts, device="cuda")
        thin = torch.full((33, 3 * C + 5), -5.0, dtype=tb, device="cuda")
        x, h = wide[:, 1:1 + C], wide[:, 2 * C + 3:3 * C + 3]
        y, n = thin[:, 1:1 + C], thin[:, C + 3:2 * C + 3]
        x.copy_(c["x"])
        y.copy_(c["y"])
        before = wide.clone(), thin.clone()
        plain = check_fwd(sh, c, "both", "layer", "linear")
        got = check_fwd(sh, dict(c, x=x, y=y), "both", "layer", "linear", h=h, n=n)
        assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
        h.fill_(-5.0)
        n.fill_(-5.0)
        assert torch.equal(wide, before[0]) and torch.equal(thin, before[1])
        dx, dy = wide[:, 2 * C + 3:3 * C + 3], thin[:, C + 3:2 * C + 3]
        a, b = check_bwd(sh, dict(c, x=x, y=y), "both", "rms", "linear", dx=dx, dy=dy), check_bwd(sh, c, "both", "rms", "linear")
        for p, q in zip(a, b):
            assert (p is None and q is None) or torch.equal(p, q)


def test_in_place(sh):
    for ts, tb, C in ((F32, F32, 64), (BF16, BF16, 1027), (F32, BF16, 130)):
        c = case(9, (5, 13), C, ts, tb, "element")
        kw = dict(post_gain=c["post_gain"], pre_gain=c["pre_gain"], kind="layer", gate_act="sigmoid")
        h, n = sh.residual_norm(c["x"], c["y"], gate=c["gate"], **kw)
        x, y = c["x"].clone(), c["y"].clone()
        h2, n2 = sh.residual_norm(x, y, gate=c["gate"], h=x, n=y, **kw)
        assert h2 is x and n2 is y and torch.equal(h, x) and torch.equal(n, y)
        g = sh.residual_norm_bwd(h, c["y"], c["dh"], c["dn"], gate=c["gate"], **kw)
        dh, dn = c["dh"].clone(), c["dn"].clone()
        g2 = sh.residual_norm_bwd(h, c["y"], dh, dn, gate=c["gate"], dx=dh, dy=dn, **kw)
        assert torch.equal(g.dx, dh) and torch.equal(g.dy, dn) and torch.equal(g.dgate, g2.dgate) and torch.equal(g.post_gain, g2.post_gain)


def test_without_a_branch(sh):
    for ts, tb in TYPES:
        c = case(3, (4, 9), 72, ts, tb)
        h, n = sh.residual_norm(c["x"], pre_gain=c["pre_gain"], pre_bias=c["pre_bias"], norms="pre", kind="layer", eps=1e-5, branch_dtype=tb)
        assert h is c["x"] and n.dtype == tb
        zero = dict(c, y=torch.zeros_like(c["y"]))
        want = expect(zero, "pre", "layer", "linear", 1.0, 1e-5)
        within(n.reshape(-1, 72), want[2], want[3], 128, "n")
        g = sh.residual_norm_bwd(c["x"], None, c["dh"], c["dn"], pre_gain=c["pre_gain"], norms="pre", kind="layer", eps=1e-5, bias_grads=True)
        ref = expect_bwd(zero, "pre", "layer", "linear", 1.0, 1e-5)
        assert g.dy is None and g.dgate is None and g.post_gain is None
        for name in ("dx", "pre_gain", "pre_bias"):
            within(getattr(g, name).reshape(ref[name][0].shape), *ref[name], 256, name)


def test_no_gradient_through_the_stream(sh):
    c = dict(case(3, (4, 9), 72, F32, BF16), dh=None)
    check_bwd(sh, c, "both", "rms", "linear")


def test_no_rows(sh):
    c = case(3, (0, 5), 64, F32, F32, "element")
    h, n = sh.residual_norm(c["x"], c["y"], gate=c["gate"], post_gain=c["post_gain"], pre_gain=c["pre_gain"])
    assert h.shape == n.shape == (0, 5, 64)
    g = sh.residual_norm_bwd(h, c["y"], c["dh"], c["dn"], gate=c["gate"], bias_grads=True)
    assert g.dx.shape == (0, 5, 64) and all(not v.any() for v in (g.post_gain, g.post_bias, g.pre_gain, g.pre_bias))


def test_rows_of_one_value_and_of_zeros(sh):
    """A layer norm of a constant row divides by sqrt(eps): the output is the bias; an rms norm of zeros likewise."""
    for C in (64, 700):
        y = torch.full((6, C), 3.25, device="cuda")
        x = torch.zeros(6, C, device="cuda")
        b, w = randn(1, C), randn(2, C)
        h, n = sh.residual_norm(x, y, post_gain=w, post_bias=b, pre_gain=w, kind="layer")
        # the mean comes out as 3.25 to two roundings, and what is left is divided by sqrt(eps) = 1e-3
        assert bool(((h - b).abs() <= 2 * U * 3.25 * 1e3 * w.abs() + 4 * U * b.abs()).all())
        h, n = sh.residual_norm(x, torch.zeros_like(y), post_gain=w, pre_gain=w, pre_bias=b, kind="rms")
        assert not h.any() and torch.equal(n, b.expand(6, C))


def test_infinities_and_nan_stay_in_their_row(sh):
    for C in (24, 64, 600):
        c = case(4, (40,), C, F32, BF16, "element")
        kw = dict(post_gain=c["post_gain"], pre_gain=c["pre_gain"], kind="layer")
        clean = sh.residual_norm(c["x"], c["y"], gate=c["gate"], **kw)
        grads = sh.residual_norm_bwd(clean[0], c["y"], c["dh"], c["dn"], gate=c["gate"], **kw)
        y, x, g = c["y"].clone(), c["x"].clone(), c["gate"].clone()
        y[3, 2], x[9, C - 1], g[17, 0] = float("inf"), float("nan"), float("-inf")
        h, n = sh.residual_norm(x, y, gate=g, **kw)
        bad = torch.zeros(40, dtype=torch.bool, device="cuda")
        bad[[3, 9, 17]] = True
        assert n[bad].isnan().any(-1).all()
        assert torch.equal(h[~bad], clean[0][~bad]) and torch.equal(n[~bad], clean[1][~bad])
        hb = clean[0].clone()
        hb[9, 0] = float("nan")
        got = sh.residual_norm_bwd(hb, y, c["dh"], c["dn"], gate=g, **kw)
        assert torch.equal(got.dx[~bad], grads.dx[~bad]) and torch.equal(got.dy[~bad], grads.dy[~bad])
        assert got.pre_gain.isnan().any()


def test_nan_stays_in_its_gate_row(sh):
    """Gate rows of 2, 50 and 2000 positions: a team's own, a workgroup's, several workgroups'."""
    for rows, G, C in ((6000, 3000, 24), (6000, 120, 40), (6000, 3, 64), (4000, 2000, 600)):
        c = case(14, (rows,), C, F32, BF16, G)
        kw = dict(gate=c["gate"], post_gain=c["post_gain"], pre_gain=c["pre_gain"], kind="layer")
        want = sh.residual_norm_bwd(c["x"], c["y"], c["dh"], c["dn"], **kw)
        dn = c["dn"].clone()
        dn[rows // G] = float("nan")             # the first position of gate row 1
        got = sh.residual_norm_bwd(c["x"], c["y"], c["dh"], dn, **kw)
        keep = torch.arange(G, device="cuda") != 1
        assert torch.equal(got.dgate[keep], want.dgate[keep]) and got.dgate[1].isnan().all()
        keep = torch.arange(rows, device="cuda") != rows // G
        assert torch.equal(got.dx[keep], want.dx[keep]) and torch.equal(got.dy[keep], want.dy[keep])
        assert got.dx[~keep].isnan().all() and got.pre_gain.isnan().all()


def test_against_differences(sh):
    """d/dt of <h, dh> + <n, dn> along a direction in all inputs, by central differences D of the forward kernel, extrapolated:
    (4 D(t / 2) - D(t)) / 3 is off by t^4 / 480 of the fifth derivative (t = 2^-6: 1e-10) and by rounding: 5760 terms of about 2,
    each off by u, over t: 2 u sqrt(5760) 2^7 = 1e-3, beside a derivative whose terms have a 2-norm of 100 or so.  1e-3 of that
    2-norm is 100 times the error expected."""
    C, lead = 48, (4, 15)
    for kind in ("rms", "layer"):
        c = {k: v.float() if v is not None else None for k, v in case(31, lead, C, F32, F32, 4).items()}
        names = ["x", "y", "gate", "post_gain", "post_bias", "pre_gain", "pre_bias"]
        step = {n: randn(50 + i, *c[n].shape) for i, n in enumerate(names)}

        def value(t):
            h, n = sh.residual_norm(*[c[k] + t * step[k] for k in names], kind=kind, gate_act="sigmoid", scale=0.8, eps=1e-3)
            return float((h.double() * c["dh"].double()).sum() + (n.double() * c["dn"].double()).sum())

        t = 2.0 ** -6
        slope = lambda t: (value(t) - value(-t)) / (2 * t)
        numeric = (4 * slope(t / 2) - slope(t)) / 3
        h, _ = sh.residual_norm(*[c[k] for k in names], kind=kind, gate_act="sigmoid", scale=0.8, eps=1e-3)
        g = sh.residual_norm_bwd(h, c["y"], c["dh"], c["dn"], gate=c["gate"], post_gain=c["post_gain"], post_bias=c["post_bias"],
                                 pre_gain=c["pre_gain"], kind=kind, gate_act="sigmoid", scale=0.8, eps=1e-3, bias_grads=True)
        terms = [(v.double() * step[n].double()) for v, n in zip(g, names)]
        exact = sum(float(v.sum()) for v in terms)
        size = math.sqrt(sum(float((v * v).sum()) for v in terms))
        assert abs(numeric - exact) <= 1e-3 * max(abs(exact), size), (kind, numeric, exact)


def test_same_bits_every_time_and_on_another_stream(sh):
    c = case(8, (16, 300), 64, F32, BF16, 16)
    kw = dict(gate=c["gate"], post_gain=c["post_gain"], pre_gain=c["pre_gain"], kind="layer")
    h, n = sh.residual_norm(c["x"], c["y"], **kw)
    g = sh.residual_norm_bwd(h, c["y"], c["dh"], c["dn"], **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h2, n2 = sh.residual_norm(c["x"], c["y"], **kw)
        g2 = sh.residual_norm_bwd(h2, c["y"], c["dh"], c["dn"], **kw)
    other = sh.residual_norm(c["x"], c["y"], stream=side.cuda_stream, **kw)      # the default stream waits for none of it
    torch.cuda.synchronize()
    assert torch.equal(h, h2) and torch.equal(n, n2) and torch.equal(h, other[0])
    for a, b in zip(g, g2):
        assert (a is None and b is None) or torch.equal(a, b)


def test_captured_and_replayed(sh):
    c = case(12, (6, 50), 96, BF16, BF16, 6)
    kw = dict(gate=c["gate"], post_gain=c["post_gain"], pre_gain=c["pre_gain"], kind="layer", gate_act="sigmoid")

    def step():
        h, n = sh.residual_norm(c["x"], c["y"], **kw)
        return [h, n] + [v for v in sh.residual_norm_bwd(h, c["y"], c["dh"], c["dn"], **kw) if v is not None]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        c["x"].copy_(randn(100 + i, 6, 50, 96))
        c["dn"].copy_(randn(200 + i, 6, 50, 96))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,G,C", [(5, 1, 48), (6000, 3000, 24), (2000, 250, 1000)])
def test_captured_twice_with_other_work_between(sh, rows, G, C):
    """Two graphs of the same call, replayed in turn with eager calls: each has a workspace of its own, or none."""
    c = case(13, (rows,), C, F32, F32, G)
    kw = dict(gate=c["gate"], post_gain=c["post_gain"], pre_gain=c["pre_gain"], gate_act="sigmoid")
    call = lambda dn: [v for v in sh.residual_norm_bwd(c["x"], c["y"], c["dh"], dn, **kw) if v is not None]
    other = 2 * c["dn"]
    want = call(c["dn"]), call(other)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, dn in zip(graphs, (c["dn"], other)):
        with torch.cuda.graph(g):
            outs.append(call(dn))
    for i in range(3):
        for o in outs[0] + outs[1]:
            o.fill_(7.0)
        graphs[i % 2].replay()
        graphs[1 - i % 2].replay()
        call(other)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_positions_behind_2_31_elements(sh):
    rows, C = 266_000, 8192                        # 2.18e9 elements
    x = torch.zeros(rows, C, dtype=BF16, device="cuda")
    y = torch.zeros(rows, C, dtype=BF16, device="cuda")
    c = case(2, (4,), C, BF16, BF16)
    x[-4:].copy_(c["x"])
    y[-4:].copy_(c["y"])
    kw = dict(post_gain=c["post_gain"], pre_gain=c["pre_gain"])
    small = sh.residual_norm(c["x"], c["y"], **kw)
    h, n = sh.residual_norm(x, y, h=x, n=y, **kw)
    assert torch.equal(h[-4:], small[0]) and torch.equal(n[-4:], small[1]) and not h[:-4].any()
    y[-4:].copy_(c["y"])
    dn = torch.zeros_like(y)
    dn[-4:].copy_(c["dn"])
    few = sh.residual_norm_bwd(small[0], c["y"], None, c["dn"], **kw)
    g = sh.residual_norm_bwd(h, y, None, dn, dx=h, dy=dn, **kw)
    assert torch.equal(g.dx[-4:], few.dx) and torch.equal(g.dy[-4:], few.dy) and not g.dx[:-4].any()
    assert torch.allclose(g.pre_gain, few.pre_gain, rtol=1e-5, atol=1e-5)      # the other rows add zeros, in another order


def test_refusals(sh):
    x, y = torch.zeros(6, 16, device="cuda"), torch.zeros(6, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    ok = dict(post_gain=w, pre_gain=w)
    sh.residual_norm(x, y, **ok)
    for bad in (dict(gate=torch.zeros(4, 16, device="cuda")), dict(gate=torch.zeros(6, 8, device="cuda")), dict(post_gain=torch.ones(8, device="cuda")),
                dict(pre_gain=w.bfloat16()), dict(pre_bias=torch.zeros(16)), dict(eps=0.0), dict(eps=float("nan")), dict(scale=float("inf")),
                dict(norms="none"), dict(kind="batch"), dict(gate_act="relu"), dict(h=y.t().contiguous().t()), dict(h=torch.zeros(6, 16, device="cuda", dtype=BF16)),
                dict(h=y[:3]), dict(n=x[:, ::2]), dict(scale=1e300), dict(gate=torch.zeros(2, 1, 16, device="cuda"))):
        with pytest.raises(ValueError):
            sh.residual_norm(x, y, **{**ok, **bad})
    x4 = torch.zeros(2, 3, 3, 16, device="cuda")
    for g in ((2, 16), (2, 1, 1, 16), (2, 3, 1, 16), (2, 3, 3, 16), (1, 16), (6, 16), (1, 1, 1, 16)):
        sh.residual_norm(x4, x4, gate=torch.zeros(*g, device="cuda"), **ok)
    for g in ((3, 16), (4, 16), (1, 3, 3, 16), (2, 1, 3, 16), (3, 3, 16), (1, 1, 16), (2, 3, 16), (9, 1, 1, 16)):
        if g == (3, 16):
            sh.residual_norm(x4, x4, gate=torch.zeros(*g, device="cuda"), **ok)      # (G, C): any number of rows that divides 18
            continue
        with pytest.raises(ValueError, match="gate"):
            sh.residual_norm(x4, x4, gate=torch.zeros(*g, device="cuda"), **ok)
    flat = torch.zeros(400, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):      # one element further on
        sh.residual_norm(flat[:96].view(6, 16), y, h=flat[1:97].view(6, 16), **ok)
    with pytest.raises(ValueError, match="overlaps"):
        sh.residual_norm(x, y, h=flat[:96].view(6, 16), n=flat[48:144].view(6, 16), **ok)
    with pytest.raises(ValueError, match="overlaps"):
        sh.residual_norm(x, y, h=flat[:96].view(6, 16), post_gain=flat[16:32], pre_gain=w)
    with pytest.raises(ValueError, match="overlaps"):      # a shared gate is read by other rows
        sh.residual_norm(x, y, gate=flat[:16].view(1, 16), h=flat[:96].view(6, 16), **ok)
    with pytest.raises(ValueError):
        sh.residual_norm(x.bfloat16(), y, **ok)            # an fp32 branch beside a 16-bit stream
    with pytest.raises(ValueError):
        sh.residual_norm(x.double(), y.double(), **ok)
    with pytest.raises(ValueError):
        sh.residual_norm(x, y.cpu(), **ok)
    with pytest.raises(ValueError):
        sh.residual_norm(torch.zeros(2, 8193, device="cuda"), torch.zeros(2, 8193, device="cuda"))
    with pytest.raises(ValueError):
        sh.residual_norm(x, pre_gain=w)                    # norms='both' without y
    with pytest.raises(ValueError):
        sh.residual_norm_bwd(x, y, None, None, norms="both")
    with pytest.raises(ValueError, match="overlaps"):
        sh.residual_norm_bwd(x, y, x, y, dx=flat[:96].view(6, 16), dy=flat[8:104].view(6, 16))
