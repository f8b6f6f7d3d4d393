"""8-bit blocks and the fc on them, CPU path: the format's definition, the
formulas and their gradients, and the refusals."""
import pytest
import torch

from paddlebox_amd.ops.fp8 import Fp8Blocks, fp8_matmul, fp8_quantize, scaled_fp8fc

from .block_oracle import held, near, product_near

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def values(m, k, dt=F32, seed=0):
    """Columns of very different scale, exact ties, zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(2 * torch.randn(k, generator=g))
    x[:, ::7] = torch.randint(-40, 41, x[:, ::7].shape, generator=g) / 16
    if m > 1:
        x[m // 2] = 0
    return x.to(dt)


def special(dt=F32):
    """A block of each kind that a scale can go wrong on."""
    x = torch.zeros(12, 128)
    x[0, 3] = float("inf")
    x[1, 5], x[1, 6] = float("nan"), 3.0
    x[2], x[2, 0] = 448.0, -448.0
    x[3, 0] = 448.5
    x[4, 0] = 449.0
    x[5] = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    x[6], x[6, 1] = torch.finfo(dt).max, -1.0
    x[7] = 2.0 ** -20
    x[8, :64], x[8, 64:] = 1.0, 2.0 ** -12
    x[9] = -0.0
    x[10] = torch.arange(128) * 2.0 ** -9
    x[11, 0], x[11, 1] = float("-inf"), 1e-3
    return x.to(dt)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("block", ["row", "tile"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 128), (5, 129), (130, 300)])
def test_quantize_is_the_definition(m, k, transposed, block, dt):
    x = values(m, k, dt)
    q = fp8_quantize(x, block, transposed)
    v = x.t() if transposed else x
    assert (q.rows, q.cols) == tuple(v.shape) and q.codes.shape[1] % 128 == 0 and q.scales.shape[1] % 4 == 0
    assert torch.equal(q.dequantize().double(), held(v, 128 if block == "tile" else 1, 128))
    assert (q.codes[:, q.cols:].float() == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_quantize_special_values(dt):
    x = special(dt)
    got, want = fp8_quantize(x).dequantize(), held(x, 1, 128).float()  # fp32's largest value is held as 2^128: infinity
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x))


def test_one_rounding_of_half_a_step():
    x = torch.randn(64, 256, generator=torch.Generator().manual_seed(2))
    d = (fp8_quantize(x).dequantize() - x).abs()
    big = x.abs().reshape(64, 2, 128).amax(2).repeat_interleave(128, 1)
    assert (d <= torch.maximum(x.abs() * 2.0 ** -4, big * 2.0 ** -17)).all()  # 2^-10 of 2^e, 2^e <= big / 224


def test_matmul_cpu():
    a, b = fp8_quantize(values(5, 300)), fp8_quantize(values(7, 300, seed=1), "tile")
    bias = torch.randn(7)
    for dt in (F32, BF16, F16):
        y = fp8_matmul(a, b, bias, dt)
        assert y.dtype == dt and y.shape == (5, 7)
        product_near(y, a.dequantize().double(), b.dequantize().double(), bias)


@pytest.mark.parametrize("dt,wt", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("m,k,o", [(1, 1, 1), (130, 72, 40), (5, 200, 129), (0, 8, 8)])
def test_fc_cpu(m, k, o, dt, wt):
    x, W = values(m, k, dt).requires_grad_(), (0.1 * values(k, o, seed=1)).to(wt).requires_grad_()
    b, dy = torch.randn(o, requires_grad=True), values(m, o, dt, seed=2)
    y = scaled_fp8fc(x, W, b)
    dx, dW, db = torch.autograd.grad(y, (x, W, b), dy)
    product_near(y, held(x, 1, 128), held(W, 128, 128).t(), b)
    product_near(dx, held(dy, 1, 128), held(W, 128, 128))
    product_near(dW, held(x, 128, 1).t(), held(dy, 128, 1).t())
    near(db, dy.double().sum(0), dy.double().abs().sum(0), roundings=(m + 1) * 2.0 ** -24)
    assert (dx.dtype, dW.dtype, db.dtype) == (dt, wt, F32)
    if m:
        p = scaled_fp8fc(x.detach(), fp8_quantize(W, "tile", transposed=True), b.detach())
        product_near(p, held(x, 1, 128), held(W, 128, 128).t(), b)


def test_fc_gradients_are_differences_on_held_values():
    """Where q() holds its argument exactly, fc is linear and its gradients are the differences of its outputs."""
    g = torch.Generator().manual_seed(0)
    x, W, dy = (torch.randint(-8, 9, s, generator=g).float() for s in ((6, 20), (20, 12), (6, 12)))
    x.requires_grad_(), W.requires_grad_()
    dx, dW = torch.autograd.grad(scaled_fp8fc(x, W), (x, W), dy)
    for t, grad, f in ((x, dx, lambda v: scaled_fp8fc(v, W)), (W, dW, lambda v: scaled_fp8fc(x, v))):
        for i in range(0, t.numel(), 7):
            e = torch.zeros(t.numel())
            e[i] = 1.0
            e = e.reshape(t.shape)
            with torch.no_grad():
                d = ((f(t + e) - f(t - e)) / 2 * dy).sum()
            assert float(d) == float(grad.flatten()[i])


X, Wt = torch.zeros(4, 8), torch.zeros(8, 6)


@pytest.mark.parametrize("call,err", [
    (lambda: scaled_fp8fc(X, torch.zeros(7, 6)), ValueError), (lambda: scaled_fp8fc(X[0], Wt), ValueError),
    (lambda: scaled_fp8fc(X.double(), Wt), TypeError), (lambda: scaled_fp8fc(X, Wt.double()), TypeError),
    (lambda: scaled_fp8fc(X, Wt, torch.zeros(5)), ValueError), (lambda: scaled_fp8fc(X, Wt, torch.zeros(6).half()), ValueError),
    (lambda: scaled_fp8fc(torch.zeros(4, 0), torch.zeros(0, 6)), ValueError),
    (lambda: scaled_fp8fc(X, torch.zeros(8, 0)), ValueError),
    (lambda: scaled_fp8fc(X, fp8_quantize(Wt, "tile")), ValueError),
    (lambda: scaled_fp8fc(X.clone().requires_grad_(), fp8_quantize(Wt, "tile", True)), ValueError),
    (lambda: fp8_quantize(X, "column"), ValueError), (lambda: fp8_quantize(torch.zeros(4, 0)), ValueError),
    (lambda: fp8_quantize(torch.zeros(0, 4), transposed=True), ValueError), (lambda: fp8_quantize(X.int()), TypeError),
    (lambda: fp8_matmul(fp8_quantize(X), fp8_quantize(torch.zeros(3, 9))), ValueError),
    (lambda: fp8_matmul(fp8_quantize(X), fp8_quantize(X), out_dtype=torch.float64), TypeError),
    (lambda: fp8_matmul(fp8_quantize(X), fp8_quantize(X), torch.zeros(3)), ValueError),
    (lambda: Fp8Blocks(torch.zeros(2, 100).to(torch.float8_e4m3fn), torch.zeros(2, 4, dtype=torch.uint8), 100), ValueError),
    (lambda: Fp8Blocks(torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8), 100), ValueError),
    (lambda: Fp8Blocks(torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.zeros(2, 4), 100), ValueError),
    (lambda: Fp8Blocks(torch.zeros(2, 128), torch.zeros(2, 4, dtype=torch.uint8), 100), ValueError),
    (lambda: Fp8Blocks(torch.zeros(128, 2).t().to(torch.float8_e4m3fn), torch.zeros(2, 4, dtype=torch.uint8), 100), ValueError)])
def test_refusals(call, err):
    with pytest.raises(err):
        call()


def test_second_order_is_refused():
    x = torch.randn(4, 8, requires_grad=True)
    (g,) = torch.autograd.grad(scaled_fp8fc(x, torch.ones(8, 6)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
