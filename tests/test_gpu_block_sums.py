"""How exactly the 8-bit products are summed on the GPU (csrc/hip/block_fp8.hip).

float32 and float16 results: no bits of a product are dropped, so a sum is off
by its additions' roundings and half a step of its type (tests/block_oracle.py,
product_near).  bfloat16 results: of each run of 8 products along K, the seven
others may lose what lies under 2^-13 of the run's largest, so at most 7 * 2^-13
of the sum of the runs' largest products."""
import pytest
import torch

from paddlebox_amd.ops.fp8 import fp8_matmul, fp8_quantize, scaled_fp8fc

from .block_oracle import held, near, product_near
from .test_block_fp8 import values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# a row of results each way: few rows, 128 x 128 tiles whole and with K in slices, 256 x 256 tiles
ROUTES = [(5, 40, 1024), (40, 3000, 200), (200, 130, 512), (400, 300, 1920), (3601, 3590, 200)]


def one_large_a_run(rows, k):
    """Each run of 8 along k: one 256 (its place differs by run and row) and seven values just under 2^-13 of it, all of
    which e4m3 holds exactly beside 256.  A row sums up to k / 8 * 256.205; without the small ones to k / 8 * 256, which
    float16 holds, 8.0e-4 of the sum too low: more than its half step of 2^-11 = 4.9e-4."""
    small = 1.875 * 2.0 ** -6
    assert small < 256 * 2.0 ** -13 and k % 8 == 0
    x = torch.full((rows, k // 8, 8), small)
    place = (torch.arange(rows)[:, None] + torch.arange(k // 8)) % 8
    return x.scatter_(2, place[..., None], 256.0).reshape(rows, k)


@pytest.mark.parametrize("m,n,k", ROUTES)
@pytest.mark.parametrize("dt", [F16, F32])
def test_small_products_beside_a_large_one(m, n, k, dt):
    x, w = one_large_a_run(m, k), torch.ones(n, k)
    assert torch.equal(held(x, 1, 128), x.double())
    y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV), "tile"), out_dtype=dt)
    product_near(y, x.double(), w.double())


@pytest.mark.parametrize("m,n,k", ROUTES)
@pytest.mark.parametrize("dt", [F16, F32])
def test_sums_hold_every_product(m, n, k, dt):
    x, w = values(m, k, seed=8), values(n, k, seed=9)
    x, w = x / x.abs().max(), w / w.abs().max()
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV)), bias.to(DEV), dt)
    product_near(y, held(x, 1, 128), held(w, 1, 128), bias)


@pytest.mark.parametrize("m", [24, 1024])
def test_fc_and_its_gradients_hold_every_product(m):
    """y, dx and dW of float16, each of one large value and seven small ones a run, in one launch or apart."""
    k, o = 200, 136
    x, W = one_large_a_run(m, k).to(F16).to(DEV).requires_grad_(), torch.ones(k, o, dtype=F16, device=DEV).requires_grad_()
    y = scaled_fp8fc(x, W)
    product_near(y, x.detach().double().cpu(), torch.ones(o, k).double())
    product_near(scaled_fp8fc(x.detach(), fp8_quantize(W, "tile", transposed=True)), x.detach().double().cpu(),
                 torch.ones(o, k).double())
    dy = one_large_a_run(m, o).to(F16)
    (dx,) = torch.autograd.grad(y, x, dy.to(DEV), retain_graph=True)
    product_near(dx, dy.double(), torch.ones(k, o).double())
    x1 = torch.ones(m, k, dtype=F16, device=DEV).requires_grad_()
    dy = one_large_a_run(o, m).t().contiguous().to(F16)
    dx, dW = torch.autograd.grad(scaled_fp8fc(x1, W), (x1, W), dy.to(DEV))
    assert dW.dtype == F16
    product_near(dW, torch.ones(k, m).double(), dy.t().double())
    product_near(dx, held(dy, 1, 128), torch.ones(k, o).double())


@pytest.mark.parametrize("m,n,k", ROUTES[:-1])
def test_bfloat16_sums_lose_no_more_than_is_said(m, n, k):
    for x, w in ((one_large_a_run(m, k), torch.ones(n, k)), (values(m, k, seed=8), values(n, k, seed=9))):
        a, b = held(x, 1, 128), held(w, 1, 128)
        y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV)), out_dtype=BF16)
        top = torch.zeros(m, n, dtype=torch.float64)  # the runs' largest products
        for i in range(0, k, 8):
            top += (a[:, None, i : i + 8] * b[None, :, i : i + 8]).abs().amax(2)
        r = (k + 64) * 2.0 ** -24
        near(y, a @ b.t(), a.abs() @ b.abs().t() + 7 * 2.0 ** -13 * top / r, roundings=r)


def test_a_bfloat16_input_has_the_codes_of_its_float32():
    """The way to sums that drop nothing for a bfloat16 input: the same held values, summed for a float32 result."""
    x, W = values(200, 300, BF16, 8).to(DEV), values(300, 40, BF16, 9).to(DEV)
    a, b = fp8_quantize(x), fp8_quantize(x.float())
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    product_near(scaled_fp8fc(x.float(), W.float()), held(x, 1, 128), held(W, 128, 128).t())


@pytest.mark.parametrize("m,n,k", [(8, 40, 300), (200, 40, 300), (400, 300, 1920), (3601, 3590, 200)])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_what_is_not_a_number_stays_in_its_row_and_column(m, n, k, dt):
    """By either route; the other rows and columns keep their values, and the scale of its block comes from the others."""
    x, w = values(m, k, seed=8), values(n, k, seed=9)
    x, w = x / x.abs().max(), w / w.abs().max()
    x[3, k - 10], w[7, 0], w[7, k - 1] = float("inf"), float("nan"), float("-inf")
    y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV)), out_dtype=dt).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[3], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(y), bad)
    rows, cols = [i for i in range(min(m, 64)) if i != 3], [i for i in range(n) if i != 7]
    product_near(y[rows][:, cols], held(x[rows], 1, 128), held(w[cols], 1, 128), exact_runs=dt != BF16)
