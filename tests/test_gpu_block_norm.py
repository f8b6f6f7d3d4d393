"""Dropout and the gated residual norm on the GPU (csrc/hip/block_norm.hip)
against 64-bit oracles; bounds are counted in tests/block_oracle.py."""
import pytest
import torch

from paddlebox_amd.ops.dropout import dropout, keep_mask
from paddlebox_amd.ops.residual import residual_norm

from .block_oracle import HALF, Residual, keep, near
from .test_block_norm import case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def cpu_keep(shape, p, seed, offset):
    return keep_mask(shape, round(p * 65536), None, seed, offset, torch.device("cpu"))


def check_drop(y, x, k, p):
    """Kept values are x / (1 - p) with one fp32 rounding of the scale, one of the product and one to x's type."""
    up = 65536 / (65536 - round(p * 65536)) if p < 1 else 0.0
    want = torch.where(k, x.double().cpu() * up, torch.zeros((), dtype=torch.float64))
    near(y, want, want.abs(), roundings=2 * 2.0 ** -24)
    assert (y.cpu()[~k] == 0).all()


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (3, 5, 129), (2, 4096), (257, 400), (0, 4)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(shape, p, dt):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(3)).to(dt).to(DEV).requires_grad_()
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
    y = dropout(x, p, -77, 5)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert y.dtype == dt and y.shape == x.shape and dx.shape == x.shape
    k = cpu_keep(shape, p, -77, 5)
    check_drop(y, x.detach(), k, p)
    check_drop(dx, dy, k, p)


def test_dropout_mask_is_the_definition():
    y = dropout(torch.ones(2001, device=DEV), 0.25, 123456789012345, 1 << 33)
    assert torch.equal(y.cpu() != 0, keep(2001, 0.25, 123456789012345, 1 << 33))


def test_dropout_drops_nan_and_infinity():
    x = torch.full((4096,), float("nan"), device=DEV)
    x[::2] = float("inf")
    k = cpu_keep((4096,), 0.5, 9, 0)
    y = dropout(x, 0.5, 9).cpu()
    assert (y[~k] == 0).all() and not torch.isfinite(y[k]).any()


@pytest.mark.parametrize("mode", ["upscale_in_train", "downgrade_in_infer"])
def test_dropout_modes(mode):
    x = torch.randn(100, device=DEV)
    y = dropout(x, 0.25, 9, mode=mode)
    k = cpu_keep((100,), 0.25, 9, 0).to(DEV)
    near(y, torch.where(k, x, 0.0).double().cpu() * (4 / 3 if mode == "upscale_in_train" else 1.0), x.double().cpu().abs(),
         roundings=2 * 2.0 ** -24)
    z = dropout(x, 0.25, training=False, mode=mode)
    assert torch.equal(z, x if mode == "upscale_in_train" else x * 0.75)


def test_dropout_strides_and_offset_pointers():
    base = torch.randn(70, 33, device=DEV, dtype=BF16)
    for x in (base.t(), base[1:, 3:], base[::2], base[:, :1].expand(70, 9), base.reshape(-1)[1:2000]):
        k = cpu_keep(tuple(x.shape), 0.3, 5, 6)
        check_drop(dropout(x, 0.3, 5, 6), x, k, 0.3)
    x = torch.randn(6, 5, device=DEV).requires_grad_()
    (g,) = torch.autograd.grad(dropout(x, 0.3, 5, 6).sum(), x)  # an expanded gradient
    check_drop(g, torch.ones(6, 5), cpu_keep((6, 5), 0.3, 5, 6), 0.3)


def test_dropout_seed_tensor_is_read_and_kept_for_the_backward():
    x = torch.randn(1000, device=DEV).requires_grad_()
    s = torch.tensor([42, 7], device=DEV)
    y = dropout(x, 0.5, s)
    assert torch.equal(y, dropout(x, 0.5, 42, 7))
    s[1] += 1  # the program moves on before the backward
    (g,) = torch.autograd.grad(y, x, torch.ones_like(x))
    check_drop(g, torch.ones(1000), cpu_keep((1000,), 0.5, 42, 7), 0.5)
    assert not torch.equal(dropout(x, 0.5, s), y)


def test_dropout_device_refusal():
    with pytest.raises(ValueError, match="seed tensor"):
        dropout(torch.zeros(8, device=DEV), 0.5, torch.zeros(2, dtype=torch.int64))


def test_dropout_first_order_only():
    x = torch.randn(8, device=DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(dropout(x, 0.5, 1).sum(), x, create_graph=True)


def test_dropout_long():
    """Over 2^31 elements: the element index passes 32 bits."""
    n = (1 << 31) + 1000
    y = dropout(torch.ones(n, device=DEV, dtype=BF16), 0.5, 3, 4)
    b0 = (n - 1000) // 8
    from .block_oracle import philox_words

    tail = [h >= 32768 for b in range(b0, b0 + 100) for w in philox_words(b, 4, 3) for h in (w & 0xFFFF, w >> 16)]
    assert (y[b0 * 8: b0 * 8 + 800].cpu() != 0).tolist() == tail


# ------------------------------------------------------------------ residual norm
KINDS = [("none", "none", None, "none", 0.0), ("rms", "layer", "channel", "sigmoid", 0.3),
         ("layer", "rms", "row", "none", 0.0), ("layer", "layer", "full", "sigmoid", 0.5),
         ("none", "rms", "row", "sigmoid", 0.1), ("rms", "none", "full", "none", 0.0),
         ("none", "layer", "channel", "none", 0.0), ("rms", "rms", None, "none", 0.25)]


def run(M, D, dt, st, post, pre, gate, act, p, seed=0, seeds=(11, 2), use=("r", "h"), wrt=None, lead=None):
    t, dr, dh = case(M, D, dt, st, post, pre, gate, seed, grad=False)
    t = {n: v.to(DEV).requires_grad_(wrt is None or n in wrt) if v is not None else None for n, v in t.items()}
    a = dict(t)
    if lead:  # the same rows under more leading dimensions
        for n in ("x", "y"):
            a[n] = t[n].reshape(*lead, D)
        if gate == "row":
            a["gate"] = t["gate"].reshape(*lead, 1)
        elif gate == "full":
            a["gate"] = t["gate"].reshape(*lead, D)
    r, h = residual_norm(**a, x_scale=0.9, y_scale=0.5, gate_act=act, post=post, pre=pre, eps=1e-5, p=p, seed=seeds[0],
                         offset=seeds[1])
    k = cpu_keep((M, D), p, *seeds) if p else None
    o = Residual(t["x"], t["y"], x_scale=0.9, y_scale=0.5, gate=t["gate"], gate_kind=gate, sigmoid=act == "sigmoid",
                 post=post, pre=pre, w=t, eps=1e-5, keep=k, up=65536 / (65536 - round(p * 65536)))
    assert r.dtype == st and r.shape == a["x"].shape and (h is None) == (pre == "none")
    near(r.reshape(M, D), o.r, o.r_mag)
    if h is not None:
        assert h.dtype == dt
        near(h.reshape(M, D), o.h, o.h_mag)
    outs, gos = [], []
    if "r" in use or h is None:
        outs.append(r), gos.append(dr.to(DEV).reshape(r.shape))
    else:
        dr = None
    if "h" in use and h is not None:
        outs.append(h), gos.append(dh.to(DEV).reshape(h.shape))
    else:
        dh = None
    names = [n for n, v in t.items() if v is not None and v.requires_grad]
    grads = torch.autograd.grad(outs, [t[n] for n in names], gos, allow_unused=True)
    want = o.backward(dr, dh)
    for n, g in zip(names, grads):
        key = n.replace("_weight", "_weight")
        if g is None:
            continue
        v, mag = want[key]
        assert g.dtype == t[n].dtype and g.shape == t[n].shape
        # column sums add up to M rows: one more rounding a level of at most M additions of what mag already counts
        extra = (M + 64) * 2.0 ** -24 if v.dim() == 1 else 0.0
        near(g, v, mag, roundings=Residual.ROUNDINGS + extra)
    return t, r, h, dict(zip(names, grads))


@pytest.mark.parametrize("dt,st", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("kinds", KINDS, ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("M,D", [(5, 40), (33, 400), (3, 1537)])
def test_residual_kinds(M, D, kinds, dt, st):
    run(M, D, dt, st, *kinds)


@pytest.mark.parametrize("M,D", [(1, 1), (7, 1), (1, 8), (1, 4096), (300, 7), (17, 127), (16, 128), (5, 129), (9, 511),
                                 (4, 512), (6, 513), (3, 2047), (2, 2048), (2, 2049), (3, 4097), (2, 8191), (1, 8200),
                                 (2, 16384), (1, 16383), (2100, 64), (1030, 2056)])
@pytest.mark.parametrize("dt,st", [(F32, F32), (BF16, F32)])
def test_residual_sizes(M, D, dt, st):
    run(M, D, dt, st, "layer", "rms", "channel", "sigmoid", 0.2)


@pytest.mark.parametrize("kinds", KINDS, ids=lambda k: "-".join(map(str, k)))
def test_residual_no_rows(kinds):
    post, pre, gate, act, p = kinds
    t, _, _ = case(0, 24, F32, F32, post, pre, gate, grad=False)
    t = {n: v.to(DEV).requires_grad_() if v is not None else None for n, v in t.items()}
    r, h = residual_norm(**t, gate_act=act, post=post, pre=pre, p=p, seed=1)
    assert r.shape == (0, 24)
    names = [n for n, v in t.items() if v is not None]
    outs = [o for o in (r, h) if o is not None]
    for n, g in zip(names, torch.autograd.grad(outs, [t[n] for n in names], [torch.zeros_like(o) for o in outs])):
        assert g.shape == t[n].shape and (g == 0).all()


@pytest.mark.parametrize("use", [("r",), ("h",)])
@pytest.mark.parametrize("kinds", [KINDS[1], KINDS[3]], ids=["channel", "full"])
def test_residual_one_output_used(use, kinds):
    run(9, 72, F32, F32, *kinds, use=use)


@pytest.mark.parametrize("wrt", [("x",), ("y",), ("gate",), ("pre_weight",), ("post_bias", "x"), ("post_weight", "pre_bias")])
def test_residual_some_gradients(wrt):
    for gate in ("channel", "row", "full"):
        run(9, 72, F32, F32, "layer", "layer", gate, "sigmoid", 0.2, wrt=wrt)


@pytest.mark.parametrize("gate", ["channel", "row", "full"])
def test_residual_leading_dimensions(gate):
    run(24, 40, BF16, BF16, "rms", "rms", gate, "none", 0.1, lead=(2, 3, 4))


def test_residual_strides():
    """Rows of a wider buffer, a transposed stream, a broadcast branch and strided gradients give the bits of their copies."""
    w = torch.rand(48, device=DEV) + 0.5
    big = torch.randn(20, 100, device=DEV)
    for x, y in ((big[:, 3:51], big[:, 50:98]), (torch.randn(48, 20, device=DEV).t(), big[:, 1:49]),
                 (big[:, :48], big[:1, :48].expand(20, 48)), (big[::2, :48], big[1::2, 52:])):
        a = residual_norm(x, y, pre="rms", pre_weight=w, post="rms", post_weight=w)
        b = residual_norm(x.contiguous(), y.contiguous(), pre="rms", pre_weight=w, post="rms", post_weight=w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x, y = (torch.randn(20, 48, device=DEV).requires_grad_() for _ in range(2))
    r, h = residual_norm(x, y, pre="rms", pre_weight=w)
    for gr, gh in ((big[:, 5:53], big.t()[:48, :20].t()[:, :48]), (torch.ones(1, 1, device=DEV).expand(20, 48),) * 2):
        u = torch.autograd.grad((r, h), (x, y), (gr, gh), retain_graph=True)
        v = torch.autograd.grad((r, h), (x, y), (gr.contiguous(), gh.contiguous()), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(u, v))


def test_residual_unaligned_rows():
    """Every byte offset of a 16-bit row start."""
    base = torch.randn(3 * 40 + 9, device=DEV).to(BF16)
    w = torch.ones(40, device=DEV)
    for off in range(9):
        x = base[off:off + 120].view(3, 40)
        a = residual_norm(x, x, pre="rms", pre_weight=w)
        b = residual_norm(x.clone(), x.clone(), pre="rms", pre_weight=w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_residual_same_bits_every_time():
    out = [run(700, 400, BF16, F32, "layer", "layer", "channel", "sigmoid", 0.2) for _ in range(2)]
    assert torch.equal(out[0][1], out[1][1]) and torch.equal(out[0][2], out[1][2])
    for n in out[0][3]:
        assert torch.equal(out[0][3][n], out[1][3][n]), n


def test_residual_gradients_are_differences():
    """Directional derivatives of the kernel's own forward (fp32) by the four-point quotient
    (8 (L(e) - L(-e)) - (L(2e) - L(-2e))) / 12e: off the gradient by the truncation, taken from the 64-bit forward at the
    same points, and by the forward's roundings of the loss's terms times 18 / 12e."""
    M, D, e = 6, 48, 2.0 ** -4
    t, dr, dh = case(M, D, F32, F32, "layer", "rms", "channel", 1, grad=False)
    k = keep(M * D, 0.25, 11, 2)

    def oracle(t):
        return Residual(t["x"], t["y"], x_scale=0.9, y_scale=0.5, gate=t["gate"], gate_kind="channel", sigmoid=True,
                        post="layer", pre="rms", w=t, eps=1e-5, keep=k, up=4 / 3)

    def kernel(t, grad=False):
        d = {n: v.float().to(DEV).requires_grad_(grad) if v is not None else None for n, v in t.items()}
        r, h = residual_norm(**d, x_scale=0.9, y_scale=0.5, gate_act="sigmoid", post="layer", pre="rms", eps=1e-5, p=0.25,
                             seed=11, offset=2)
        return d, r, h

    def loss(r, h):
        return float((r.double().cpu() * dr.double()).sum() + (h.double().cpu() * dh.double()).sum())

    d, r, h = kernel(t, True)
    names = [n for n, v in t.items() if v is not None]
    grads = dict(zip(names, torch.autograd.grad((r, h), [d[n] for n in names], (dr.to(DEV), dh.to(DEV)))))
    o = oracle(t)
    want = o.backward(dr, dh)
    size = float((o.r_mag * dr.abs()).sum() + (o.h_mag * dh.abs()).sum())
    for n in names:
        v = torch.randint(-1, 2, t[n].shape, generator=torch.Generator().manual_seed(2)).float()
        num = num64 = 0.0
        for c, m in ((8, 1), (-8, -1), (-1, 2), (1, -2)):
            at = {**t, n: t[n].double() + m * e * v}
            num += c * loss(*kernel(at)[1:]) / (12 * e)
            num64 += c * loss(oracle(at).r, oracle(at).h) / (12 * e)
        exact = float((want[n][0] * v.double()).sum())
        got = float((grads[n].double().cpu() * v.double()).sum())
        lim = abs(num64 - exact) * (1 + 1e-3) + 1.5 * Residual.ROUNDINGS * size / e
        assert abs(num - got) <= lim, (n, num, got, lim)
        assert lim < 0.05 * max(1.0, abs(exact)) + 0.5, (n, lim)  # the bound says something


def test_residual_zero_and_extreme_rows():
    w = torch.ones(32, device=DEV)
    x = torch.zeros(4, 32, device=DEV)
    r, h = residual_norm(x, x, post="rms", post_weight=w, pre="layer", pre_weight=w, pre_bias=w)
    assert (r == 0).all() and torch.equal(h, torch.ones_like(h))
    y = torch.randn(4, 32, device=DEV)
    y[1, 3] = float("inf")
    y[2, 5] = float("nan")
    r, h = residual_norm(x, y, pre="rms", pre_weight=w)
    assert torch.isfinite(h[[0, 3]]).all() and torch.isnan(h[2]).all()  # rows do not touch one another
    assert torch.isinf(r[1, 3]) and torch.isnan(r[2, 5])


def test_residual_refuses_devices_and_second_order():
    w = torch.ones(8, device=DEV)
    x = torch.zeros(4, 8, device=DEV).requires_grad_()
    with pytest.raises(ValueError):
        residual_norm(x, torch.zeros(4, 8), pre="rms", pre_weight=w)
    with pytest.raises(ValueError):
        residual_norm(x, x, pre="rms", pre_weight=w.cpu())
    with pytest.raises(ValueError):
        residual_norm(x, x, pre="rms", pre_weight=w, gate=torch.ones(8))
    with pytest.raises(ValueError):
        residual_norm(x, x, pre="rms", pre_weight=w, p=0.5, seed=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(residual_norm(x, x, pre="rms", pre_weight=w)[1].sum(), x, create_graph=True)


def test_residual_in_place_change_is_seen():
    """An input that the backward needs and that changed in place raises instead of giving wrong gradients."""
    w = torch.ones(8, device=DEV).requires_grad_()
    y = torch.randn(4, 8, device=DEV)
    _, h = residual_norm(torch.zeros(4, 8, device=DEV), y, post="rms", post_weight=w, pre="rms", pre_weight=w)
    y += 1
    with pytest.raises(RuntimeError, match="inplace"):
        h.sum().backward()


def test_residual_other_stream_and_two_calls_at_once():
    torch.cuda.synchronize()
    w = torch.rand(400, device=DEV) + 0.5
    x, y = torch.randn(3000, 400, device=DEV), torch.randn(3000, 400, device=DEV)
    want = residual_norm(x, y, pre="rms", pre_weight=w, post="rms", post_weight=w, p=0.5, seed=3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(residual_norm(x, y, pre="rms", pre_weight=w, post="rms", post_weight=w, p=0.5, seed=3))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])


def test_captured_step_replays():
    """Forward and backward of both operators in one graph; the seed tensor moves between replays, and eager work of
    the same leaves runs before and between them."""
    w = (torch.rand(72, device=DEV) + 0.5).requires_grad_()
    x, y = (torch.randn(50, 72, device=DEV).requires_grad_() for _ in range(2))
    seed = torch.tensor([5, 0], device=DEV)
    go = torch.randn(50, 72, device=DEV)

    def step():
        r, h = residual_norm(x, dropout(y, 0.3, seed), post="rms", post_weight=w, pre="rms", pre_weight=w, p=0.2, seed=seed)
        return (r, h) + torch.autograd.grad((r, h), (x, y, w), (go, go))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        seed[1] = i
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i


def test_low_bits_of_types():
    assert HALF[BF16] == 2.0 ** -8 and HALF[F16] == 2.0 ** -11 and HALF[F32] == 2.0 ** -24


def test_more_rows_than_a_launch_dimension():
    """2^24 + 37 rows of 3: past 2^20 workgroups of 16 rows, forward and backward, against the same rows in a short call."""
    m, part = (1 << 24) + 37, 1 << 16
    y = torch.randn(part, 3, device=DEV, dtype=BF16).repeat(m // part + 1, 1)[:m].requires_grad_()
    x = torch.zeros_like(y).detach()
    w = torch.ones(3, device=DEV)
    r, h = residual_norm(x, y, post="rms", post_weight=w, pre="rms", pre_weight=w)
    (dy,) = torch.autograd.grad(h, y, y.detach().clone())
    ys = y.detach()[:part].clone().requires_grad_()
    r1, h1 = residual_norm(x[:part], ys, post="rms", post_weight=w, pre="rms", pre_weight=w)
    (dy1,) = torch.autograd.grad(h1, ys, ys.detach().clone())
    for at in range(0, m, part):
        n = min(part, m - at)
        for a, b in ((r, r1), (h, h1), (dy, dy1)):
            assert torch.equal(a[at : at + n], b[:n])
