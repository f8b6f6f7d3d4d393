"""Dropout and the gated residual norm on the CPU path: the mask's definition,
the formulas, the gradients against differences, and the refusals."""
import math

import pytest
import torch

from paddlebox_amd.ops.dropout import dropout, keep_mask
from paddlebox_amd.ops.residual import residual_norm

from .block_oracle import Residual, keep, near, philox_words


def test_philox_known_answers():
    """The test vectors published with the generator (key and counter all zero, all ones)."""
    ones = (1 << 64) - 1
    assert philox_words(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox_words(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("n,p,seed,offset", [(1, 0.5, 0, 0), (8, 0.5, 1, 2), (203, 0.1, 12345678901234, 3),
                                             (64, 0.9, -5, -1), (17, 1.0, 3, 1 << 40), (9, 0.0, 3, 0)])
def test_mask_definition(n, p, seed, offset):
    got = keep_mask((n,), round(p * 65536), None, seed, offset, torch.device("cpu"))
    assert torch.equal(got, keep(n, p, seed & (1 << 64) - 1, offset & (1 << 64) - 1))
    t = keep_mask((n,), round(p * 65536), torch.tensor([seed, offset]), 0, 0, torch.device("cpu"))
    assert torch.equal(got, t)


@pytest.mark.parametrize("mode", ["upscale_in_train", "downgrade_in_infer"])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
def test_dropout_cpu(p, mode):
    x = torch.randn(5, 7, generator=torch.Generator().manual_seed(1)).requires_grad_()
    y = dropout(x, p, 7, 1, mode=mode)
    k = keep(35, p, 7, 1).reshape(5, 7)
    up = (1 / (1 - p) if p < 1 else 0.0) if mode == "upscale_in_train" else 1.0
    assert torch.equal(y, torch.where(k, x * up, torch.zeros(())))
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(g, k.float() * up)
    z = dropout(x, p, training=False, mode=mode)
    assert torch.equal(z, x if mode == "upscale_in_train" else x * (1 - p))


def test_dropout_drops_infinities():
    x = torch.full((64,), math.inf)
    y = dropout(x, 0.5, 3)
    k = keep(64, 0.5, 3, 0)
    assert torch.isinf(y[k]).all() and (y[~k] == 0).all()


@pytest.mark.parametrize("kw,err", [
    (dict(p=-0.1, seed=1), ValueError), (dict(p=1.1, seed=1), ValueError), (dict(p=float("nan"), seed=1), ValueError),
    (dict(p=True, seed=1), ValueError), (dict(p=0.5), ValueError), (dict(p=0.5, seed=1.5), TypeError),
    (dict(p=0.5, seed=1, offset=0.5), TypeError), (dict(p=0.5, seed=1, mode="other"), ValueError),
    (dict(p=0.5, seed=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(p=0.5, seed=torch.zeros(2)), ValueError),
    (dict(p=0.5, seed=torch.zeros(2, dtype=torch.int64), offset=1), ValueError)])
def test_dropout_refusals(kw, err):
    with pytest.raises(err):
        dropout(torch.zeros(4), **kw)
    with pytest.raises(TypeError):
        dropout(torch.zeros(4, dtype=torch.float64), 0.5, 1)


def case(M, D, dt, st, post, pre, gate, seed=0, grad=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = {}
    for n, k in (("post", post), ("pre", pre)):
        w[n + "_weight"] = 1 + 0.2 * r(D) if k != "none" else None
        w[n + "_bias"] = 0.2 * r(D) if k == "layer" else None
    gt = {None: None, "channel": r(D), "row": r(M, 1), "full": r(M, D).to(dt)}[gate]
    t = dict(x=r(M, D).to(st), y=(2 * r(M, D) + 0.5).to(dt), gate=gt, **w)
    for v in t.values():
        if v is not None and grad:
            v.requires_grad_()
    return t, r(M, D).to(st), r(M, D).to(dt)


@pytest.mark.parametrize("dt,st", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float32)])
@pytest.mark.parametrize("post,pre,gate,act,p", [
    ("none", "none", None, "none", 0.0), ("rms", "layer", "channel", "sigmoid", 0.3), ("layer", "rms", "row", "none", 0.0),
    ("layer", "layer", "full", "sigmoid", 0.5), ("none", "rms", "row", "sigmoid", 0.1), ("rms", "none", "full", "none", 0.0)])
@pytest.mark.parametrize("M,D", [(3, 40), (1, 1), (0, 5), (4, 129)])
def test_residual_cpu(M, D, post, pre, gate, act, p, dt, st):
    t, dr, dh = case(M, D, dt, st, post, pre, gate)
    r, h = residual_norm(**t, x_scale=0.9, y_scale=0.5, gate_act=act, post=post, pre=pre, eps=1e-5, p=p, seed=11, offset=2)
    k = keep(M * D, p, 11, 2) if p else None
    o = Residual(t["x"], t["y"], x_scale=0.9, y_scale=0.5, gate=t["gate"], gate_kind=gate, sigmoid=act == "sigmoid",
                 post=post, pre=pre, w=t, eps=1e-5, keep=k, up=65536 / (65536 - round(p * 65536)))
    near(r, o.r, o.r_mag)
    assert (h is None) == (pre == "none")
    if h is not None:
        near(h, o.h, o.h_mag)


def test_residual_oracle_gradients_are_differences():
    """The oracle's gradient formulas against central differences of its own forward, in 64 bits."""
    for seed, (post, pre, gate, act, p) in enumerate([("rms", "layer", "channel", True, 0.3), ("layer", "rms", "row", True, 0.0),
                                                      ("layer", "layer", "full", False, 0.4), ("none", "rms", None, False, 0.2)]):
        M, D = 3, 11
        t, dr, dh = case(M, D, torch.float32, torch.float32, post, pre, gate, seed, grad=False)
        t = {n: v.double() if v is not None else None for n, v in t.items()}
        k = keep(M * D, p, 1, 0) if p else None

        def make(t):
            return Residual(t["x"], t["y"], x_scale=0.9, y_scale=0.5, gate=t["gate"], gate_kind=gate, sigmoid=act,
                            post=post, pre=pre, w=t, eps=1e-5, keep=k, up=1 / (1 - p))

        o = make(t)
        loss = lambda o: float((o.r * dr.double()).sum() + (o.h * dh.double()).sum())  # noqa: E731
        for name, (grad, _) in o.backward(dr, dh).items():
            gen = torch.Generator().manual_seed(5)
            v = torch.randn(t[name].shape, generator=gen, dtype=torch.float64)
            e = 1e-5
            num = (loss(make({**t, name: t[name] + e * v})) - loss(make({**t, name: t[name] - e * v}))) / (2 * e)
            # truncation e^2 times a third derivative, 2^-53 / e of the loss's terms: both under 1e-8 here
            assert abs(num - float((grad * v).sum())) < 1e-7 * (1 + abs(num)), (name, post, pre)


def test_residual_cpu_gradients():
    t, dr, dh = case(6, 24, torch.float32, torch.float32, "layer", "rms", "channel", 3)
    r, h = residual_norm(**t, y_scale=0.5, gate_act="sigmoid", post="layer", pre="rms", p=0.25, seed=4)
    names = [n for n, v in t.items() if v is not None]
    grads = torch.autograd.grad((r, h), [t[n] for n in names], (dr, dh))
    o = Residual(t["x"], t["y"], x_scale=1.0, y_scale=0.5, gate=t["gate"], gate_kind="channel", sigmoid=True, post="layer",
                 pre="rms", w=t, eps=1e-6, keep=keep(144, 0.25, 4, 0), up=4 / 3)
    want = o.backward(dr, dh)
    for n, g in zip(names, grads):
        near(g, *want[n], roundings=4 * Residual.ROUNDINGS)  # torch's autograd takes more steps than the formulas


W = torch.ones(8)


@pytest.mark.parametrize("kw,err", [
    (dict(pre="rms"), ValueError), (dict(pre="layer", pre_weight=W), ValueError), (dict(pre="none", pre_weight=W), ValueError),
    (dict(pre="max", pre_weight=W), ValueError), (dict(pre="rms", pre_weight=W.double()), ValueError),
    (dict(pre="rms", pre_weight=torch.ones(7)), ValueError), (dict(pre="rms", pre_weight=W, post="rms"), ValueError),
    (dict(pre="rms", pre_weight=W, gate=torch.ones(7)), ValueError), (dict(pre="rms", pre_weight=W, gate=torch.ones(4)), ValueError),
    (dict(pre="rms", pre_weight=W, gate=W.half()), ValueError), (dict(pre="rms", pre_weight=W, gate=W, gate_act="tanh"), ValueError),
    (dict(pre="rms", pre_weight=W, gate_act="sigmoid"), ValueError), (dict(pre="rms", pre_weight=W, eps=-1.0), ValueError),
    (dict(pre="rms", pre_weight=W, p=0.5), ValueError), (dict(pre="rms", pre_weight=W, p=2.0, seed=1), ValueError),
    (dict(pre="rms", pre_weight=W, y=torch.zeros(4, 7)), ValueError),
    (dict(pre="rms", pre_weight=W, y=torch.zeros(4, 8, dtype=torch.float64)), TypeError),
    (dict(pre="rms", pre_weight=W, x=torch.zeros(4, 8).half()), TypeError)])
def test_residual_refusals(kw, err):
    a = dict(x=torch.zeros(4, 8), y=torch.zeros(4, 8))
    a.update(kw)
    with pytest.raises(err):
        residual_norm(**a)


def test_residual_width_limit():
    D = 16385
    with pytest.raises(ValueError, match="columns"):
        residual_norm(torch.zeros(1, D), torch.zeros(1, D), pre="none")
    with pytest.raises(ValueError, match="columns"):
        residual_norm(torch.zeros(3, 0), torch.zeros(3, 0), pre="none")
