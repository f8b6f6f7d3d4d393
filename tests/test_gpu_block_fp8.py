"""The 8-bit fc on the GPU (csrc/hip/block_fp8.hip): codes against the format's
definition bit for bit, products against 64 bits (tests/block_oracle.py)."""
import pytest
import torch

from paddlebox_amd.ops.fp8 import Fp8Blocks, fp8_matmul, fp8_quantize, scaled_fp8fc

from .block_oracle import held, near
from .block_oracle import product_near as product_near_cpu
from .test_block_fp8 import special, values

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def product_near(got, a, b, bias=None):
    product_near_cpu(got, a, b, bias, exact_runs=False)


def same_blocks(q, want: Fp8Blocks):
    assert (q.rows, q.cols) == (want.rows, want.cols)
    nb = want.codes.shape[1] // 128
    assert torch.equal(q.scales[:, :nb].cpu(), want.scales[:, :nb])
    a, b = q.codes.float().cpu(), want.codes.float()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("block,transposed", [("row", False), ("row", True), ("tile", False), ("tile", True)])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 129), (16, 7), (128, 128), (130, 257), (300, 1000), (5, 4096), (1025, 40)])
def test_quantize(m, k, block, transposed, dt):
    x = values(m, k, dt)
    q = fp8_quantize(x.to(DEV), block, transposed)
    same_blocks(q, fp8_quantize(x, block, transposed))
    v = x.t() if transposed else x
    assert torch.equal(q.dequantize().double().cpu(), held(v, 128 if block == "tile" else 1, 128))
    assert (q.codes[:, q.cols:].float() == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_quantize_special_values(dt):
    x = special(dt)
    same_blocks(fp8_quantize(x.to(DEV)), fp8_quantize(x))
    same_blocks(fp8_quantize(x.t().contiguous().to(DEV), transposed=True), fp8_quantize(x))
    same_blocks(fp8_quantize(x.to(DEV), "tile"), fp8_quantize(x, "tile"))


def test_quantize_every_exponent():
    """Each power of two that fp32 has, and the values next to 448 times it."""
    x = torch.zeros(256, 128)
    for i in range(254):
        x[i, 0] = torch.tensor(1.75 * 2.0 ** (i - 126))
        x[i, 1] = x[i, 0] / 3
        if i % 2:
            x[i, 2] = torch.nextafter(x[i, 0], torch.tensor(float("inf")))
    q = fp8_quantize(x.to(DEV))
    same_blocks(q, fp8_quantize(x))
    assert torch.equal(q.dequantize().double().cpu(), held(x, 1, 128))


def test_quantize_strides():
    big = torch.randn(200, 300, device=DEV)
    for x in (big[:, 3:150], big[::3, 1:], big.t(), big[:1].expand(200, 300)):
        for kw in (dict(), dict(transposed=True), dict(block="tile")):
            a, b = fp8_quantize(x, **kw), fp8_quantize(x.contiguous(), **kw)
            assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("m", [1, 15, 17, 33, 49, 64, 65, 127, 129, 300])
@pytest.mark.parametrize("n", [1, 3, 16, 127, 130, 400])
def test_matmul_sizes(m, n):
    for k, dt in ((1, F32), (128, BF16), (129, F16), (500, F32), (1300, F32)):
        x, w = values(m, k), values(n, k, seed=1)
        a, b = fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV), "tile")
        bias = torch.randn(n, generator=torch.Generator().manual_seed(3)) if k % 2 else None
        y = fp8_matmul(a, b, bias.to(DEV) if bias is not None else None, dt)
        assert y.shape == (m, n) and y.dtype == dt
        product_near(y, held(x, 1, 128), held(w, 128, 128), bias)


@pytest.mark.parametrize("m,n,k", [(400, 400, 8192), (80, 33, 5000), (1000, 900, 128), (64, 64, 20000), (520, 260, 777),
                                   (2048, 2048, 256), (700, 2000, 1152)])
def test_matmul_tiles_and_slices(m, n, k):
    x, w = values(m, k, seed=4), values(n, k, seed=5)
    a, b = fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV))
    y = fp8_matmul(a, b)
    product_near(y, held(x, 1, 128), held(w, 1, 128))
    assert torch.equal(y, fp8_matmul(a, b))  # the same bits every time


@pytest.mark.parametrize("m", [8, 200])
def test_matmul_wide_scales(m):
    """Scales far apart in either operand: their exponents are added, not multiplied out one after the other."""
    x, w = torch.randn(m, 512), torch.randn(40, 512)
    for ex, ew in ((-100, 100), (100, -100), (-60, -60), (60, 55), (-110, -10), (0, -125)):
        a, b = x * 2.0 ** ex, w * 2.0 ** ew
        y = fp8_matmul(fp8_quantize(a.to(DEV)), fp8_quantize(b.to(DEV)))
        product_near(y, held(a, 1, 128), held(b, 1, 128))


@pytest.mark.parametrize("m", [8, 200])
def test_matmul_not_a_number_stays_in_its_row(m):
    x, w = torch.randn(m, 300), torch.randn(40, 300)
    x[3, 290], w[7, 0] = float("inf"), float("nan")
    y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV))).cpu()
    bad = torch.zeros(m, 40, dtype=torch.bool)
    bad[3], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(y), bad)


def test_matmul_reads_nothing_behind_its_operands():
    """Blocks whose neighbours in memory are NaN codes: rows and blocks past the end do not reach the result."""
    for m, n, k in ((70, 30, 200), (9, 5, 140), (200, 200, 900)):
        kp, sp = (k + 127) // 128 * 128, ((k + 127) // 128 + 3) // 4 * 4
        x, w = torch.randn(m, k), torch.randn(n, k)
        ops = []
        for v in (x, w):
            q = fp8_quantize(v)
            c = torch.full((v.shape[0] + 40, kp), 0x7F, dtype=torch.uint8)
            s = torch.full((v.shape[0] + 40, sp), 255, dtype=torch.uint8)
            c[:v.shape[0]], s[:v.shape[0], : kp // 128] = q.codes.view(torch.uint8), q.scales[:, : kp // 128]
            c, s = c.to(DEV), s.to(DEV)
            ops.append(Fp8Blocks(c[:v.shape[0]].view(torch.float8_e4m3fn), s[:v.shape[0]], k))
        product_near(fp8_matmul(*ops), held(x, 1, 128), held(w, 1, 128))


def check_fc(m, k, o, dt, wt=F32, bias=True, wrt=("x", "W", "b"), seed=0):
    t = {"x": values(m, k, dt, seed), "W": (0.1 * values(k, o, seed=seed + 1)).to(wt),
         "b": torch.randn(o, generator=torch.Generator().manual_seed(seed)) if bias else None}
    dy = values(m, o, dt, seed + 2)
    d = {n: v.to(DEV).requires_grad_(n in wrt) if v is not None else None for n, v in t.items()}
    y = scaled_fp8fc(d["x"], d["W"], d["b"])
    assert y.dtype == dt and y.shape == (m, o)
    product_near(y, held(t["x"], 1, 128), held(t["W"], 128, 128).t(), t["b"])
    names = [n for n in wrt if d[n] is not None]
    grads = dict(zip(names, torch.autograd.grad(y, [d[n] for n in names], dy.to(DEV)))) if names else {}
    for n, g in grads.items():
        assert g.shape == t[n].shape and g.dtype == t[n].dtype
    if "x" in grads:
        product_near(grads["x"], held(dy, 1, 128), held(t["W"], 128, 128))
    if "W" in grads:
        product_near(grads["W"], held(t["x"], 128, 1).t(), held(dy, 128, 1).t())
    if "b" in grads:
        near(grads["b"], dy.double().sum(0), dy.double().abs().sum(0), roundings=(m + 8) * 2.0 ** -24)
    return d, y, grads


@pytest.mark.parametrize("dt,wt", [(F32, F32), (BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("m,k,o", [(1, 1, 1), (7, 40, 3), (64, 200, 129), (130, 72, 300), (777, 400, 33), (2048, 400, 400)])
def test_fc(m, k, o, dt, wt):
    check_fc(m, k, o, dt, wt)


@pytest.mark.parametrize("wrt", [("x",), ("W",), ("b",), ("x", "b"), ("W", "b"), ()])
def test_fc_some_gradients(wrt):
    check_fc(200, 72, 140, F32, wrt=wrt)
    check_fc(30, 72, 140, BF16, wrt=[n for n in wrt if n != "b"], bias=False)


def test_fc_no_rows():
    d, y, g = check_fc(0, 24, 40, F32)
    assert y.shape == (0, 40) and (g["W"] == 0).all() and (g["b"] == 0).all() and g["x"].shape == (0, 24)
    assert scaled_fp8fc(d["x"].detach(), fp8_quantize(d["W"], "tile", transposed=True)).shape == (0, 40)
    assert fp8_quantize(d["x"].detach()).codes.shape == (0, 128)


@pytest.mark.parametrize("m", [1, 3, 16, 48, 64, 65, 200])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_fc_packed_is_the_forward(m, dt):
    W, b = torch.randn(300, 130, device=DEV), torch.randn(130, device=DEV)
    x = values(m, 300, dt).to(DEV)
    packed = fp8_quantize(W, "tile", transposed=True)
    y = scaled_fp8fc(x, packed, b)
    product_near(y, held(x, 1, 128), held(W, 128, 128).t(), b)
    assert torch.equal(y, scaled_fp8fc(x, W, b))


def test_fc_follows_its_weight():
    """Nothing is kept from one call for the next: a weight that changes in place counts at once."""
    W = torch.randn(64, 48, device=DEV)
    x = torch.randn(100, 64, device=DEV)
    a = scaled_fp8fc(x, W)
    W.mul_(3.0)
    b = scaled_fp8fc(x, W)
    product_near(b, held(x, 1, 128), held(W, 128, 128).t())
    assert not torch.equal(a, b)


def test_fc_strides():
    big = torch.randn(300, 300, device=DEV)
    for x, W in ((big[:, 5:77], big[:72, 9:50]), (big.t()[:, :64], big[::2][:64, :40]), (big[:1, :40].expand(70, 40), big[:40])):
        x, W = x.detach().requires_grad_(), W.detach().requires_grad_()
        y = scaled_fp8fc(x, W)
        xc, Wc = x.detach().contiguous().requires_grad_(), W.detach().contiguous().requires_grad_()
        yc = scaled_fp8fc(xc, Wc)
        assert torch.equal(y, yc)
        for dy in (torch.randn(y.shape[1], y.shape[0], device=DEV).t(), torch.ones(1, 1, device=DEV).expand(y.shape)):
            for a, b in zip(torch.autograd.grad(y, (x, W), dy, retain_graph=True),
                            torch.autograd.grad(yc, (xc, Wc), dy.contiguous(), retain_graph=True)):
                assert torch.equal(a, b)


def test_fc_same_bits_every_time():
    a, b = (check_fc(2048, 400, 400, F32)[2] for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_fc_refusals():
    x, W = torch.zeros(4, 8, device=DEV), torch.zeros(8, 6, device=DEV)
    for call in (lambda: scaled_fp8fc(x, W.cpu()), lambda: scaled_fp8fc(x, W, torch.zeros(6)),
                 lambda: scaled_fp8fc(x, fp8_quantize(W.cpu(), "tile", True)),
                 lambda: fp8_matmul(fp8_quantize(x), fp8_quantize(x.cpu()))):
        with pytest.raises(ValueError):
            call()
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(scaled_fp8fc(x, W).sum(), x, create_graph=True)


def test_fc_two_streams():
    x, W = torch.randn(3000, 400, device=DEV), torch.randn(400, 400, device=DEV)
    want = scaled_fp8fc(x, W)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(scaled_fp8fc(x, W))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_fc_captured_step_replays():
    """Forward and backward in a graph: with slices of K, and the weight changing between replays."""
    W = (0.1 * torch.randn(400, 400, device=DEV)).requires_grad_()
    b = torch.randn(400, device=DEV).requires_grad_()
    x, dy = torch.randn(2048, 400, device=DEV).requires_grad_(), torch.randn(2048, 400, device=DEV)

    def step():
        y = scaled_fp8fc(x, W, b)
        return (y,) + torch.autograd.grad(y, (x, W, b), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        with torch.no_grad():
            W.add_(0.01 * i)
        want = [v.clone() for v in step()]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c), i


@pytest.mark.parametrize("m,n,k", [(3601, 3590, 200), (12700, 1000, 128), (300, 50000, 520)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_matmul_large_tiles(m, n, k, dt):
    """Results over 2^23.6 values take 256 x 256 tiles: ragged ones, one block of K, more than one group of exponents."""
    x, w = values(m, k, seed=6), values(n, k, seed=7)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3))
    y = fp8_matmul(fp8_quantize(x.to(DEV)), fp8_quantize(w.to(DEV)), bias.to(DEV), dt)
    product_near(y, held(x, 1, 128), held(w, 1, 128), bias)


@pytest.mark.parametrize("m,k,o", [(65, 500, 40), (4000, 130, 3300)])
def test_fc_mixed_launches(m, k, o):
    """dx and dW in one launch, each in slices or not, and apart where one of them takes large tiles."""
    check_fc(m, k, o, BF16)
    check_fc(m, k, o, F32)


def test_two_graphs_share_nothing():
    """Two captured steps of one layer replayed in turn and against eager work keep their own temporaries."""
    W = torch.randn(400, 400, device=DEV)
    xs = [torch.randn(m, 400, device=DEV) for m in (700, 1300)]
    want = [scaled_fp8fc(x, W) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(scaled_fp8fc(x, W))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = scaled_fp8fc(xs[0], W)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(a, b) for a, b in zip(outs, want))


def test_capture_beside_a_live_eager_graph_is_refused():
    """The backward of a captured step may not meet a leaf that an eager graph on the default stream still holds."""
    W = torch.randn(40, 40, device=DEV).requires_grad_()
    x = torch.randn(70, 40, device=DEV)
    alive = scaled_fp8fc(x, W)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(g):
            scaled_fp8fc(x, W)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(g):
            scaled_fp8fc(alive, torch.empty(40, 8, device=DEV))
    del alive, g
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = scaled_fp8fc(x, W)
        (dW,) = torch.autograd.grad(y, W, torch.ones_like(y))
    g.replay()
    torch.cuda.synchronize()
    product_near(dW, held(x, 128, 1).t(), torch.ones(40, 70, dtype=torch.float64))


def test_block_of_a_tower():
    """The operators as they are used together: stream, branch -> residual_norm with dropout -> fc -> relu -> fc, forward
    and backward; each is held to its oracle on what the one before it gave."""
    from paddlebox_amd.ops.dropout import keep_mask
    from paddlebox_amd.ops.residual import residual_norm

    from .block_oracle import Residual

    M, D, H = 300, 136, 264
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g).to(DEV).requires_grad_()  # noqa: E731
    x, y, w, W1, W2, b1 = mk(M, D), mk(M, D), mk(D), mk(D, H), mk(H, D), mk(H)
    r, h = residual_norm(x, y, y_scale=0.5, post="rms", post_weight=w, pre="rms", pre_weight=w, p=0.25, seed=3, offset=4)
    a = scaled_fp8fc(h, W1, b1)
    z = torch.relu(a)
    out = scaled_fp8fc(z, W2)
    dout, dr = torch.randn(M, D, generator=g).to(DEV), torch.randn(M, D, generator=g).to(DEV)
    names = dict(z=z, a=a, h=h, x=x, y=y, w=w, W1=W1, W2=W2, b1=b1)
    grads = dict(zip(names, torch.autograd.grad((out, r), list(names.values()), (dout, dr))))
    o = Residual(x, y, x_scale=1.0, y_scale=0.5, gate=None, gate_kind=None, sigmoid=False, post="rms", pre="rms",
                 w={"post_weight": w, "pre_weight": w}, eps=1e-6, keep=keep_mask((M, D), 16384, None, 3, 4, torch.device("cpu")),
                 up=4 / 3)
    near(r, o.r, o.r_mag)
    near(h, o.h, o.h_mag)
    product_near(a, held(h, 1, 128), held(W1, 128, 128).t(), b1)
    product_near(out, held(z, 1, 128), held(W2, 128, 128).t())
    product_near(grads["z"], held(dout, 1, 128), held(W2, 128, 128))
    product_near(grads["W2"], held(z, 128, 1).t(), held(dout, 128, 1).t())
    product_near(grads["h"], held(grads["a"], 1, 128), held(W1, 128, 128))
    product_near(grads["W1"], held(h, 128, 1).t(), held(grads["a"], 128, 1).t())
    want = o.backward(dr, grads["h"])
    near(grads["x"], *want["x"])
    near(grads["y"], *want["y"])
    ww, wm = (p + q for p, q in zip(want["pre_weight"], want["post_weight"]))
    near(grads["w"], ww, wm, roundings=Residual.ROUNDINGS + (M + 64) * 2.0 ** -24)


@pytest.mark.parametrize("m,n", [(0, 40), (200, 0), (3, 0), (0, 0)])
def test_empty_products(m, n):
    a, b = fp8_quantize(torch.randn(m, 600, device=DEV)), fp8_quantize(torch.randn(n, 600, device=DEV))
    assert fp8_matmul(a, b).shape == (m, n)
    assert scaled_fp8fc(torch.randn(m, 600, device=DEV), b).shape == (m, n)


def test_quantize_more_blocks_than_a_launch_dimension():
    """2^24 + 8 blocks and more: the grid's second dimension; each row is the row 4096 before it."""
    part = values(4096, 1025, seed=11).to(BF16).to(DEV)
    m = 465 * 4096 + 7
    q, want = fp8_quantize(part.repeat(466, 1)[:m]), fp8_quantize(part)
    codes, scales = q.codes.view(torch.uint8), want.scales[:, :9]
    for at in range(0, m, 4096):
        n = min(4096, m - at)
        assert torch.equal(codes[at : at + n], want.codes.view(torch.uint8)[:n])
        assert torch.equal(q.scales[at : at + n, :9], scales[:n])


@pytest.mark.parametrize("m", [5, 200])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_matmul_outermost_exponent_bytes(m, dt):
    """Blocks of exponent bytes at both ends, made by hand: what they stand for, NaN for 255."""
    g = torch.Generator().manual_seed(2)
    for byte, other in ((0, 227), (1, 227), (254, 27), (255, 127)):
        # magnitudes 2 .. 3.75 (byte 0, 1: held values of 2^-126 and more) or 1 .. 1.875 (254: finite ones)
        mag = torch.randint(8, 16, (m, 256), generator=g) / (8 if byte == 254 else 4)
        a = (mag * (torch.randint(0, 2, (m, 256), generator=g) * 2 - 1)).to(torch.float8_e4m3fn)
        b = (torch.randint(8, 16, (40, 256), generator=g) / 8).to(torch.float8_e4m3fn)
        qa = Fp8Blocks(a.to(DEV), torch.full((m, 4), byte, dtype=torch.uint8, device=DEV), 256)
        qb = Fp8Blocks(b.to(DEV), torch.full((40, 4), other, dtype=torch.uint8, device=DEV), 256)
        y = fp8_matmul(qa, qb, out_dtype=dt)
        if byte == 255:
            assert y.isnan().all() and qa.dequantize().isnan().all()
        else:
            product_near(y, qa.dequantize().cpu().double(), qb.dequantize().cpu().double())
