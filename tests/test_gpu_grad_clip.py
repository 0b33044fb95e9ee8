"""grad_norm, clip_grads (include/sr_hip.h sr_tensors_*, sr_op_grad_norm, sr_op_clip_grads) against float64.

Tolerances: squares are added in 64 bits, so a norm is the 64-bit norm to 1e-12 and then rounded once to fp32 (2^-24 relative).  A
clipped element is g * f with f = fp32(fp32(max_norm) / norm) * scale: three roundings of the factor and one of the product
(4 * 2^-24), then one to its type (eps / 2 relative, or half a smallest subnormal)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def randn(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check_norm(got, want):
    assert abs(float(got) - want) <= want * (U + 1e-12) + TINY[F32] / 2, (float(got), want)


def check_clipped(got, src, norm, max_norm, scale):
    f = scale * (max_norm / norm if norm > max_norm else 1.0)
    want = src.double() * f
    tol = torch.finfo(src.dtype).eps / 2 * want.abs() * (1 + 4 * U) + TINY[src.dtype] / 2 + 4 * U * want.abs()
    assert got.dtype == src.dtype and got.shape == src.shape
    if src.numel():
        assert float(((got.double() - want).abs() - tol).max()) <= 0


LISTS = {
    "one element": ([1], F32), "one tensor": ([100_003], BF16), "small": ([1, 2, 3, 0, 5, 7, 8, 9, 15, 16, 17, 255, 256, 257], F16),
    "chunk borders": ([8191, 8192, 8193, 16384, 24577], F32), "many": ([(i * 37) % 1000 for i in range(1500)], F32),
    "long": ([20_000_001, 3, 9_999_999], BF16), "empty ones": ([0, 0, 5, 0], F32),
}


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("layout", ["apart", "views", "mixed"])
def test_norm_and_clip(sh, name, layout):
    sizes, dt = LISTS[name]
    if layout == "views":            # consecutive views, most of them at odd addresses
        flat = randn(1, sum(sizes) + 1, scale=0.1).to(dt)[1:]
        ts = list(torch.split(flat, sizes))
    else:
        ts = [randn(i, n, scale=0.1).to(dt if layout == "apart" else (F32, BF16, F16)[i % 3]) for i, n in enumerate(sizes)]
    lst = sh.TensorList(ts)
    for scale in (1.0, 0.125):
        want = norm64(ts) * scale
        norm, each = sh.grad_norm(lst, scale=scale, per_tensor=True)
        check_norm(norm, want)
        check_norm(sh.grad_norm(ts, scale=scale), want)
        assert each.shape == (len(ts),)
        for i, t in list(enumerate(ts))[:: max(1, len(ts) // 200)]:
            check_norm(each[i], norm64([t]) * scale)
        for share in (0.3, 3.0):
            out = [torch.full_like(t, 9.0) for t in ts]
            got = sh.clip_grads(lst, share * want + 1e-9, scale=scale, out=out)
            assert torch.equal(got, norm)
            for o, t in zip(out, ts):
                check_clipped(o, t, want, share * want + 1e-9, scale)
            mine = [t.clone() for t in ts]
            assert torch.equal(sh.clip_grads(mine, share * want + 1e-9, scale=scale), norm)
            for o, m in zip(out, mine):
                assert torch.equal(o, m)


def test_no_tensors(sh):
    assert float(sh.grad_norm([])) == 0.0
    norm, each = sh.grad_norm([torch.empty(0, device="cuda")], per_tensor=True)
    assert float(norm) == 0.0 and float(each[0]) == 0.0
    assert float(sh.clip_grads([torch.empty(0, device="cuda")], 1.0)) == 0.0
    assert float(sh.clip_grads([torch.zeros(70, device="cuda")], 1.0)) == 0.0


def test_views_into_a_buffer_leave_the_rest(sh):
    """Outputs at every misalignment of a 16-byte vector against their sources; the elements around them stay."""
    for dt in (F32, BF16, F16):
        for a in range(8):
            for n in (1, 6, 8, 100, 9000):
                src = randn(a, n + 16).to(dt)
                dst = torch.full((n + 16,), -3.0, dtype=dt, device="cuda")
                g, o = src[a:a + n], dst[7 - a:7 - a + n]
                w = norm64([g])
                sh.clip_grads([g], w / 2, out=[o])
                check_clipped(o, g, w, w / 2, 1.0)
                o.fill_(-3.0)
                assert bool((dst == -3.0).all())


@pytest.mark.parametrize("dt", [F32, F16])
@pytest.mark.parametrize("upload", [True, False])
def test_thousands_of_tensors(sh, dt, upload):
    """A partial sum a tensor: these are joined before the clipping launch."""
    sizes = [1 + i * 7 % 900 for i in range(9000)]
    flat = randn(2, sum(sizes), scale=0.1).to(dt)
    ts, dst = list(torch.split(flat, sizes)), torch.full_like(flat, 9.0)
    lst, out = sh.TensorList(ts, upload=upload), sh.TensorList(list(torch.split(dst, sizes)), upload=upload)
    want = norm64([flat])
    for share in (0.3, 3.0):
        norm = sh.clip_grads(lst, share * want, out=out)
        check_norm(norm, want)
        check_clipped(dst, flat, want, share * want, 1.0)
    keep = flat.clone()
    check_norm(sh.clip_grads(lst, want / 8, scale=0.5), want / 2)
    check_clipped(flat, keep, want / 2, want / 8, 0.5)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_large_lists_stored_past_the_caches(sh, dt):
    """More than 128 MB: in place, and into views at odd addresses, whose surroundings stay."""
    sizes = [1, 30_000_001, 4099, 45_000_007]
    ts = [randn(i, n, scale=0.1).to(dt) for i, n in enumerate(sizes)]
    whole = torch.full((sum(sizes) + 3,), -3.0, dtype=dt, device="cuda")
    out = list(torch.split(whole[1:-2], sizes))
    want = norm64(ts)
    norm = sh.clip_grads(sh.TensorList(ts), want / 3, out=sh.TensorList(out))
    check_norm(norm, want)
    for o, t in zip(out, ts):
        check_clipped(o, t, want, want / 3, 1.0)
    assert float(whole[0]) == -3.0 and bool((whole[-2:] == -3.0).all())
    assert torch.equal(sh.clip_grads(ts, want / 3), norm)
    for o, t in zip(out, ts):
        assert torch.equal(o, t)


def test_any_dense_order_of_dimensions(sh):
    t = randn(3, 5, 4, 6, 7)
    p = t.permute(0, 3, 1, 2)
    check_norm(sh.grad_norm([p, t.transpose(0, 1)]), norm64([t, t]))
    want = norm64([t])
    q = t.clone().permute(2, 0, 3, 1)
    sh.clip_grads([q], want / 4)
    check_clipped(q, t.permute(2, 0, 3, 1), want, want / 4, 1.0)
    with pytest.raises(ValueError, match="gaps"):
        sh.TensorList([t[:, ::2]])
    with pytest.raises(ValueError, match="gaps"):
        sh.TensorList([torch.zeros(1, device="cuda").expand(8)])


def test_squares_beyond_fp32(sh):
    big, tiny = torch.full((5000,), 1e30, device="cuda"), torch.full((5000,), 1e-30, device="cuda")
    check_norm(sh.grad_norm([big]), float(big[0].double()) * math.sqrt(5000))
    check_norm(sh.grad_norm([tiny]), float(tiny[0].double()) * math.sqrt(5000))
    sh.clip_grads([big], 1.0)
    assert abs(norm64([big]) - 1.0) <= 4 * U
    sub = torch.full((3000,), 2.0 ** -149, device="cuda")
    assert abs(float(sh.grad_norm([sub])) - 2.0 ** -149 * math.sqrt(3000)) <= 2.0 ** -150


def test_infinity_and_nan(sh):
    t = randn(1, 9000)
    a = [t.clone(), t.clone()]
    a[1][77] = float("inf")
    norm, each = sh.grad_norm(a, per_tensor=True)
    assert math.isinf(float(norm)) and math.isinf(float(each[1])) and math.isfinite(float(each[0]))
    assert math.isinf(float(sh.clip_grads(a, 1.0)))
    assert not a[0].any() and bool(a[1][77].isnan()) and not a[1][:77].any() and not a[1][78:].any()
    b = [t.clone(), t.clone()]
    b[0][5] = float("nan")
    assert math.isnan(float(sh.clip_grads(b, 1e-3)))
    assert torch.equal(b[1], t) and torch.equal(b[0][6:], t[6:]) and bool(b[0][5].isnan())


def test_borders_of_the_bound(sh):
    t = torch.zeros(300, device="cuda")
    t[0], t[299] = 3.0, 4.0
    u = t.clone()
    assert float(sh.clip_grads([u], 5.0)) == 5.0 and torch.equal(u, t)            # norm == max_norm: as it was
    sh.clip_grads([u], float("inf"))
    assert torch.equal(u, t)
    sh.clip_grads([u], 2.5)
    assert torch.equal(u, t * 0.5)
    u = t.clone()
    assert float(sh.clip_grads([u], 100.0, scale=0.25)) == 1.25 and torch.equal(u, t * 0.25)


def test_same_bits_streams_and_lists_at_once(sh):
    ts = [randn(i, 50_001, scale=0.1) for i in range(20)]
    a, b = sh.TensorList(ts), sh.TensorList(ts[:10])
    first = sh.grad_norm(a)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for q in s:
        q.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):                          # two streams, one list: each call has its own workspace
        for q, lst in zip(s, (a, b)):
            with torch.cuda.stream(q):
                got.append((lst is a, sh.grad_norm(lst)))
    torch.cuda.synchronize()
    half = sh.grad_norm(b)
    for whole, v in got:
        assert torch.equal(v, first if whole else half)


def test_captured_and_replayed(sh):
    ts = [randn(i, n) for i, n in enumerate((70_000, 3, 8192, 999))]
    lst = sh.TensorList(ts)
    out = [torch.empty_like(t) for t in ts]
    outs = sh.TensorList(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, each = sh.grad_norm(lst, per_tensor=True)
        clipped = sh.clip_grads(lst, 2.0, out=outs)
    for i in range(4):
        for t in ts:
            t.copy_(randn(40 + i, t.numel(), scale=10.0 ** -i))
        graph.replay()
        torch.cuda.synchronize()
        want = norm64(ts)
        check_norm(norm, want)
        assert torch.equal(norm, clipped)
        for o, t in zip(out, ts):
            check_clipped(o, t, want, 2.0, 1.0)
        assert torch.equal(sh.grad_norm(ts), norm)


def test_long_list_captured_replayed_and_gone(sh):
    """A graph does not read what the list has on the GPU: it is replayed after the list is gone and others took its place, one of
    them while a capture is under way."""
    ts = [randn(i, 1 + i * 13) for i in range(400)]
    lst, out = sh.TensorList(ts), [torch.empty_like(t) for t in ts]
    outs, old = sh.TensorList(out), sh.TensorList(ts[:200])
    eager = sh.clip_grads(lst, 1.0, out=outs)
    first = [o.clone() for o in out]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = sh.clip_grads(lst, 1.0, out=outs)
        again = sh.grad_norm(ts)                 # a list made inside the capture
        old.close()
    del lst, outs
    for i in range(3):
        more = [sh.TensorList(ts[i:300 + i]) for i in range(4)]
        for o in out:
            o.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager) and torch.equal(again, eager)
        for o, f in zip(out, first):
            assert torch.equal(o, f)
        del more


def test_tensor_behind_2_31_elements(sh):
    t = torch.zeros((1 << 31) + 11, dtype=BF16, device="cuda")
    t[-1], t[1 << 30], t[0], t[(1 << 31)] = 2.0, 4.0, 4.0, 8.0
    norm, each = sh.grad_norm([t], per_tensor=True)
    assert float(norm) == 10.0 and float(each[0]) == 10.0
    sh.clip_grads([t], 5.0)
    assert float(t[-1]) == 1.0 and float(t[1 << 31]) == 4.0 and float(t[1 << 30]) == 2.0 and float(t[0]) == 2.0


def test_refusals(sh):
    a, b = torch.ones(40, device="cuda"), torch.ones(40, device="cuda")
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            sh.clip_grads([a], bad)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            sh.grad_norm([a], scale=bad)
    with pytest.raises(ValueError, match="share memory"):
        sh.clip_grads([a, a], 1.0)               # the same tensor twice cannot be written
    assert abs(float(sh.grad_norm([a, a])) - math.sqrt(80)) < 1e-6        # ... but read
    with pytest.raises(ValueError, match="share memory"):
        sh.clip_grads([a[:30], a[20:]], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        sh.clip_grads([a, b], 1.0, out=[torch.empty(40, device="cuda")] * 2)
    with pytest.raises(ValueError, match="another gradient"):
        sh.clip_grads([a, b], 1.0, out=[b, a])
    with pytest.raises(ValueError, match="another gradient"):
        sh.clip_grads([a, b], 1.0, out=[b, torch.empty(40, device="cuda")])
    c = torch.ones(80, device="cuda")
    with pytest.raises(ValueError, match="another gradient"):
        sh.clip_grads([c[:40]], 1.0, out=[c[20:60]])
    with pytest.raises(ValueError, match="another gradient"):
        sh.clip_grads([a, a], 1.0, out=[a, b])
    sh.clip_grads([a, b], 1.0, out=[a, torch.empty(40, device="cuda")])     # one in place, one not
    with pytest.raises(ValueError, match="differ"):
        sh.clip_grads([a, b], 1.0, out=[torch.empty(40, device="cuda")])
    with pytest.raises(ValueError, match="differs"):
        sh.clip_grads([a], 1.0, out=[torch.empty(41, device="cuda")])
    with pytest.raises(ValueError, match="differs"):
        sh.clip_grads([a], 1.0, out=[torch.empty(40, device="cuda", dtype=BF16)])
    with pytest.raises(ValueError):
        sh.TensorList([a, b.cpu()])
    with pytest.raises(ValueError):
        sh.TensorList([a.cpu()])
    with pytest.raises(ValueError):
        sh.TensorList([a.double()])
    lst = sh.TensorList([a])
    lst.close()
    with pytest.raises(ValueError, match="closed"):
        sh.grad_norm(lst)
