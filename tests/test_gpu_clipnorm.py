"""Clipped optimizer steps: sr_train_set_clipnorm, sr_disc_set_clipnorm, Adam(clipnorm=...), train.clipnorm (include/sr_hip.h; Keras
2.2.4 optimizers.py get_gradients).  A clipped step must be the unclipped step of gradients that were clipped before, bit for bit: both
take the same partial sums in the same order and multiply a gradient by the same factor once.  Norms against float64: 2^-24."""
import os

import numpy as np
import pytest

from oracle import ref_disc as rd
from oracle import ref_numpy as rn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def sh():
    import sr_hip
    assert sr_hip.device_count() >= 1, "no HIP device: the product path has no CPU fallback"
    return sr_hip


def batch(seed, B=2, h=16, w=24):
    rng = np.random.default_rng(seed)
    lr = rng.random((2, B, h, w, 3), dtype=np.float32)
    hr = rng.random((2, B, 4 * h, 4 * w, 3), dtype=np.float32)
    return lr[0], lr[1], hr[0], hr[1]


def context(sh, weights, model="frvsr", h=16, w=24):
    c = sh.Context(h, w, max_batch=2, dtype="fp32", model=model)
    c.load_weights(weights)
    return c


def same_weights(a, b):
    for (n, x), (_, y) in zip(a.get_weights(), b.get_weights()):
        assert np.array_equal(x, y), n


def norm64(*flat):
    return float(np.sqrt(sum((np.asarray(f, np.float64) ** 2).sum() for f in flat)))


@pytest.mark.parametrize("grad_scale", [1.0, 0.25])
def test_generator_step(sh, weights7, grad_scale):
    import torch
    data = batch(1)
    clipped, plain, loose = context(sh, weights7), context(sh, weights7), context(sh, weights7)
    loose.set_clipnorm(1e6)
    with pytest.raises(RuntimeError, match="no step with clipping"):
        clipped.grad_norm()
    for step in range(2):                       # the second step has moments
        flats = [c.train_grads(*data, read=True)[1] for c in (clipped, plain)]
        assert np.array_equal(*flats)
        want = norm64(flats[0]) * grad_scale
        bound = want * (0.3, 0.9)[step]
        clipped.set_clipnorm(bound)
        clipped.train_apply(grad_scale=grad_scale)
        assert abs(clipped.grad_norm() - want) <= 2 * U * want
        g = torch.from_numpy(flats[1]).cuda()
        out = torch.empty_like(g)
        norm = sh.clip_grads([g], bound, scale=grad_scale, out=[out])
        assert float(norm) == clipped.grad_norm()
        torch.cuda.synchronize()
        plain.train_apply(d_grads=out.data_ptr())
        same_weights(clipped, plain)
        assert np.array_equal(clipped.train_read_grads(), flats[0])          # the gradient itself is as it was
    # a bound that is not reached changes nothing, and 0 is off
    off = context(sh, weights7)
    for c in (loose, off):
        c.train_grads(*data)
        c.train_apply(grad_scale=grad_scale)
    same_weights(loose, off)
    assert abs(loose.grad_norm() - norm64(off.train_read_grads()) * grad_scale) <= 2 * U * loose.grad_norm()
    off.set_clipnorm(1e-3)
    off.set_clipnorm(0)
    for c in (loose, off):
        c.train_on_batch(*data)
    same_weights(loose, off)
    for c in (clipped, plain, loose, off):
        c.close()


def test_train_on_batch_and_on_clips_clip_too(sh, weights7):
    data = batch(2)
    a, b = context(sh, weights7), context(sh, weights7)
    for c in (a, b):
        c.set_clipnorm(1e-2)
    a.train_on_batch(*data)
    b.train_grads(*data)
    b.train_apply()
    same_weights(a, b)
    assert a.grad_norm() > 1e-2
    hr = rn.synth_clip(5, 2, 64, 96, scale=4)[None]
    a.train_on_clips(hr)
    b.train_clips_grads(hr)
    b.train_apply()
    same_weights(a, b)
    a.close()
    b.close()


def test_discriminator_step(sh):
    import torch
    w = rd.make_disc_weights(4, 32, 48)
    rng = np.random.default_rng(0)
    imgs = [rng.random((2, 32, 48, 3), dtype=np.float32) for _ in range(9)]
    clipped, plain = [sh.Discriminator(32, 48, max_batch=2) for _ in range(2)]
    for d in (clipped, plain):
        d.load_weights(w)
    with pytest.raises(RuntimeError, match="no step with clipping"):
        clipped.grad_norm()
    for t in (1, 2):
        flats = [d.train_grads(imgs, [1.0, 0.0], read=True)[1] for d in (clipped, plain)]
        want = norm64(flats[0])
        clipped.set_clipnorm(want / 4)
        clipped.apply(t)
        assert abs(clipped.grad_norm() - want) <= 2 * U * want
        g = torch.from_numpy(flats[1]).cuda()
        sh.clip_grads([g], want / 4)
        torch.cuda.synchronize()
        plain.apply(t, d_grads=g.data_ptr())
        same_weights(clipped, plain)
    clipped.close()
    plain.close()


@pytest.mark.parametrize("train_disc", [True, False])
def test_combined_step_clips_both_models_by_one_norm(sh, weights7, train_disc):
    import torch
    B, h, w = 2, 16, 16
    rng = np.random.default_rng(3)
    lr = [rng.random((B, h, w, 3), dtype=np.float32) for _ in range(2)]
    hr = [rng.random((B, 4 * h, 4 * w, 3), dtype=np.float32) for _ in range(7)]
    feats = [rng.standard_normal((B, 64 >> (k + 1), 64 >> (k + 1), c)).astype(np.float32) for k, c in enumerate((64, 64, 128, 256))]
    pairs = []
    for _ in range(2):
        ctx, d = context(sh, weights7, "tecogan", h, w), sh.Discriminator(4 * h, 4 * w, max_batch=B)
        d.load_weights(rd.make_disc_weights(6, 4 * h, 4 * w))
        pairs.append((ctx, d))
    (ctx, d), (ctx2, d2) = pairs
    d.set_clipnorm(1e-9)                        # the discriminator's own bound is not the combined step's
    for t in (3, 4):
        for c, q in pairs:
            sh.tecogan_grads(c, q, lr[0], lr[1], *hr, feats, hr[6][::-1].copy(), rd.LOSS_WEIGHTS)
        g, gd = (torch.from_numpy(f).cuda() for f in (ctx2.train_read_grads(), d2.read_grads()))
        want = norm64(*[f.cpu().numpy() for f in ((g, gd) if train_disc else (g,))])
        ctx.set_clipnorm(want / 3)
        sh.tecogan_apply(ctx, d, t, train_disc=train_disc)
        assert abs(ctx.grad_norm() - want) <= 2 * U * want
        sh.clip_grads([g, gd] if train_disc else [g], want / 3)
        torch.cuda.synchronize()
        sh.tecogan_apply(ctx2, d2, t, d_gen_grads=g.data_ptr(), d_disc_grads=gd.data_ptr(), train_disc=train_disc)
        same_weights(ctx, ctx2)
        same_weights(d, d2)
    for c, q in pairs:
        c.close()
        q.close()


def test_generator_step_right_behind_a_combined_one(sh, weights7):
    """The discriminator's part of a combined step runs on its own stream and reads the ctx's partial sums; the ctx's next step, which
    writes them anew, comes behind it."""
    import torch
    B, h, w = 1, 16, 16
    rng = np.random.default_rng(4)
    pairs = []
    for _ in range(2):
        ctx, d = context(sh, weights7, "tecogan", h, w), sh.Discriminator(4 * h, 4 * w, max_batch=B)
        d.load_weights(rd.make_disc_weights(6, 4 * h, 4 * w))
        pairs.append((ctx, d))
    (ctx, d), (ctx2, d2) = pairs
    lr = [rng.random((B, h, w, 3), dtype=np.float32) for _ in range(2)]
    hr = [rng.random((B, 4 * h, 4 * w, 3), dtype=np.float32) for _ in range(7)]
    feats = [rng.standard_normal((B, 64 >> (k + 1), 64 >> (k + 1), c)).astype(np.float32) for k, c in enumerate((64, 64, 128, 256))]
    for c, q in pairs:
        sh.tecogan_grads(c, q, lr[0], lr[1], *hr, feats, hr[6][::-1].copy(), rd.LOSS_WEIGHTS)
        c.set_clipnorm(1e-2)
    g, gd = (torch.from_numpy(f).cuda() for f in (ctx.train_read_grads(), d.read_grads()))
    other = 50 * g                              # another norm for the generator's own steps
    torch.cuda.synchronize()
    for t in range(1, 9):
        for c, q in pairs:
            sh.tecogan_apply(c, q, t, d_gen_grads=g.data_ptr(), d_disc_grads=gd.data_ptr())
            if c is ctx2:
                torch.cuda.synchronize()
            c.train_apply(d_grads=other.data_ptr())
            if c is ctx2:
                torch.cuda.synchronize()
    assert ctx.grad_norm() == ctx2.grad_norm() > 1e-2
    same_weights(ctx, ctx2)
    same_weights(d, d2)
    for c, q in pairs:
        c.close()
        q.close()


def test_refusals(sh, weights7):
    c = context(sh, weights7)
    d = sh.Discriminator(16, 16)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            c.set_clipnorm(bad)
        with pytest.raises(ValueError):
            d.set_clipnorm(bad)
    c.close()
    d.close()


def build(kind, tmp_path, weights, train):
    import weights_io
    from FRVSR import FrameRecurrentVideoSR
    from TecoGAN import TecoGAN
    weights_io.write_tensors(str(tmp_path / 'w.h5'), list(weights.items()))
    cfg = {'root_dir': str(tmp_path), 'dtype': 'fp32', 'data': {'videos': str(tmp_path / 'clips'), 'rows': 1, 'cols': 1, 'high_res': 64},
           'cnn': {'model': kind, 'pretrained_model': 'w.h5'}, 'train': train}
    m = {'frvsr': FrameRecurrentVideoSR, 'tecogan': TecoGAN}[kind]((16, 16, 3), (64, 64, 3), str(tmp_path), cfg)
    m.build()
    m._load_pretrained()
    return m


def test_train_stage_with_clipnorm(sh, tmp_path, weights7):
    os.makedirs(tmp_path / 'clips')
    np.save(tmp_path / 'clips' / '0.npy', (rn.synth_clip(20, 8, 96, 96, scale=4) * 255).astype(np.uint8))
    train = {'iterations': 1, 'batch_size': 2, 'c_frames': 3, 'sample_freq': 10, 'checkpoint_freq': 10, 'info_freq': 10, 'seed': 1}
    got = {}
    for bound in (None, 0, 1e9, 1e-3):
        m = build('frvsr', tmp_path, weights7, dict(train, clipnorm=bound))
        assert m.opt.clipnorm == (bound or 0)
        m.train()
        got[bound] = m.frvsr.get_weights()
        if bound:
            assert m.core._ctx.grad_norm() > 1e-3
    for x, y, z, c in zip(got[None], got[0], got[1e9], got[1e-3]):
        assert np.array_equal(x, y) and np.array_equal(x, z)
    assert any(not np.array_equal(x, c) for x, c in zip(got[None], got[1e-3]))


def test_adversarial_iteration_with_clipnorm(sh, tmp_path, weights7):
    """The fused native pass and the step-by-step one clip alike: the same weights, bit for bit, and not those without clipping."""
    hr = rn.synth_clip(41, 4, 64, 64, scale=4)[None]
    dw = list(rd.make_disc_weights(9, 64, 64).values())
    got = []
    for bound, steps in ((2e-3, True), (2e-3, False), (None, False)):
        t = build('tecogan', tmp_path, weights7, {'clipnorm': bound})
        t.discriminator.set_weights(dw)
        t.step_by_step = steps
        t.gan_iteration(hr)
        if bound:
            assert t.core._ctx.grad_norm() > bound and t.discriminator._native.grad_norm() > 0
        got.append(t.generator.get_weights() + t.discriminator.get_weights())
    for x, y in zip(got[0], got[1]):
        assert np.array_equal(x, y)
    assert any(not np.array_equal(x, z) for x, z in zip(got[0], got[2]))
