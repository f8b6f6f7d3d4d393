"""64-bit oracles of the dense-block operators, written from their formulas
(no code of ops/dropout.py, ops/residual.py or ops/fp8.py)."""
import torch

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}  # half a step, relative


def philox_words(block, offset, seed):
    """Philox4x32-10 of one counter on Python integers."""
    m = 0xFFFFFFFF
    c = [block & m, block >> 32 & m, offset & m, offset >> 32 & m]
    k = [seed & m, seed >> 32 & m]
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & m, (p0 >> 32) ^ c[3] ^ k[1], p0 & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def keep(n, p, seed, offset):
    """The mask of n elements, element by element."""
    thr, out = round(p * 65536), []
    for b in range((n + 7) // 8):
        for w in philox_words(b, offset, seed):
            out += [(w & 0xFFFF) >= thr, (w >> 16) >= thr]
    return torch.tensor(out[:n], dtype=torch.bool)


class Residual:
    """One residual_norm in 64 bits: its outputs, the gradients' formulas and
    bounds on what 32-bit arithmetic may be off by.

    A row sum over D columns runs as at most 16 additions in a thread and 10
    levels of a tree; with the products and the final steps every normalised
    value and every gradient of one carries under 64 roundings (2^-24 each) of
    terms no larger than the ones that ``mag`` adds up in absolute value."""

    ROUNDINGS = 64 * 2.0 ** -24

    def __init__(self, x, y, *, x_scale, y_scale, gate, gate_kind, sigmoid, post, pre, w, eps, keep, up):
        d = lambda t: t.detach().double().cpu() if t is not None else None  # noqa: E731
        self.x, self.y, self.w = d(x), d(y), {k: d(v) for k, v in w.items()}
        self.xs, self.ys, self.eps, self.post, self.pre = x_scale, y_scale, eps, post, pre
        self.gate_kind, self.sigmoid = gate_kind, sigmoid
        self.raw = d(gate)
        self.g = torch.ones(()).double() if gate is None else torch.sigmoid(self.raw) if sigmoid else self.raw
        self.k = keep.reshape(self.y.shape).double() * up if keep is not None else torch.ones_like(self.y)
        self.n_post, self.inv_post, self.u, self.u_mag = self._norm(self.y, post, "post", self.y.abs())
        self.r = self.xs * self.x + self.ys * self.g * self.k * self.u
        self.r_mag = (self.xs * self.x).abs() + (self.ys * self.g * self.k).abs() * self.u_mag
        self.n_pre, self.inv_pre, self.h, self.h_mag = self._norm(self.r, pre, "pre", self.r_mag)

    def _norm(self, v, kind, which, mag):
        """(normalised, 1/dev, output, magnitude) of a norm whose input carries errors in proportion to `mag`."""
        if kind == "none":
            return v, None, v, mag
        mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
        c = v - mean
        inv = 1 / (c.square().mean(-1, keepdim=True) + self.eps).sqrt()
        n, w = c * inv, self.w[which + "_weight"]
        out = n * w
        # the input's error, the mean's (it averages the errors) and the deviation's, which scales n
        m = (mag + mag.mean(-1, keepdim=True)) * inv + n.abs() * (1 + (mag * c.abs()).mean(-1, keepdim=True) * inv * inv)
        mag = m * w.abs()
        if kind == "layer":
            out, mag = out + self.w[which + "_bias"], mag + self.w[which + "_bias"].abs()
        return n, inv, out, mag

    @staticmethod
    def _back(g, n, inv, kind, g_mag, n_mag):
        """(gradient of the norm's input, magnitude) from g = d(out) * weight."""
        if kind == "none":
            return g, g_mag
        m = (lambda t: t.mean(-1, keepdim=True))
        v = inv * (g - n * m(g * n) - (m(g) if kind == "layer" else 0.0))
        mag = inv * (g_mag + n_mag * m((g * n).abs()) + n.abs() * m(g_mag * n.abs() + g.abs() * n_mag) + m(g_mag))
        return v, mag * (1 + m(n_mag * n.abs()))

    def backward(self, dr, dh):
        """Gradients and their magnitudes: {name: (value, magnitude)}."""
        z = torch.zeros_like(self.y)
        dr = z if dr is None else dr.double().cpu()
        dh = z if dh is None else dh.double().cpu()
        out = {}
        t, t_mag = dr, dr.abs()
        if self.pre != "none":
            mean = self.r.mean(-1, keepdim=True) if self.pre == "layer" else 0.0
            n = (self.r - mean) * self.inv_pre
            n_mag = (self.r_mag + self.r_mag.mean(-1, keepdim=True)) * self.inv_pre + n.abs() * (
                1 + (self.r_mag * n.abs()).mean(-1, keepdim=True) * self.inv_pre)
            g = dh * self.w["pre_weight"]
            v, v_mag = self._back(g, n, self.inv_pre, self.pre, g.abs(), n_mag)
            t, t_mag = t + v, t_mag + v_mag
            out["pre_weight"] = ((dh * n).reshape(-1, n.shape[-1]).sum(0), (dh.abs() * n_mag).reshape(-1, n.shape[-1]).sum(0))
            if self.pre == "layer":
                out["pre_bias"] = (dh.reshape(-1, n.shape[-1]).sum(0), dh.abs().reshape(-1, n.shape[-1]).sum(0))
        out["x"] = (self.xs * t, abs(self.xs) * t_mag)
        d, d_mag = self.k * self.u, self.k * self.u_mag
        if self.gate_kind:
            s = self.g * (1 - self.g) if self.sigmoid else torch.ones(()).double()
            dg, dg_mag = self.ys * t * d * s, abs(self.ys) * (t_mag * d.abs() + t.abs() * d_mag) * (2 * s.abs() + 2 * 2.0 ** -24)
            if self.gate_kind == "channel":
                dg, dg_mag = dg.reshape(-1, d.shape[-1]).sum(0), dg_mag.reshape(-1, d.shape[-1]).sum(0)
            elif self.gate_kind == "row":
                dg, dg_mag = dg.sum(-1, keepdim=True), dg_mag.sum(-1, keepdim=True)
            out["gate"] = (dg, dg_mag)
        c = (self.ys * self.g * self.k).expand_as(t)
        du, du_mag = t * c, t_mag * c.abs()
        if self.post != "none":
            n_mag = (self.y.abs() + self.y.abs().mean(-1, keepdim=True)) * self.inv_post + 2 * self.n_post.abs()
            D = t.shape[-1]
            out["post_weight"] = ((du * self.n_post).reshape(-1, D).sum(0),
                                  (du_mag * self.n_post.abs() + du.abs() * n_mag).reshape(-1, D).sum(0))
            if self.post == "layer":
                out["post_bias"] = (du.reshape(-1, D).sum(0), du_mag.reshape(-1, D).sum(0))
            g = du * self.w["post_weight"]
            g_mag = du_mag * self.w["post_weight"].abs()
            out["y"] = self._back(g, self.n_post, self.inv_post, self.post, g_mag, n_mag)
        else:
            out["y"] = (du, du_mag)
        return out


def near(got, want, mag, roundings=Residual.ROUNDINGS):
    """Asserts |got - want| <= half a step of got's type + roundings * mag; where that reaches past the type's largest
    value, infinity is right too."""
    got64, f = got.detach().double().cpu(), torch.finfo(got.dtype)
    half_subnormal = f.smallest_normal * f.eps / 2
    lim = HALF[got.dtype] * want.abs() + roundings * mag * (1 + HALF[got.dtype]) + half_subnormal
    over = (got64 == torch.sign(want) * float("inf")) & (want.abs() + lim > f.max)
    bad = ~(((got64 - want).abs() <= lim) | over)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, worst "
                           f"{float(((got64 - want).abs() / lim).nan_to_num(1e30).max()):.3g} x the bound")


# ------------------------------------------------------------------ 8-bit blocks
def held(x, rows, cols):
    """x (any float type) as blocks of rows x cols hold it in e4m3 with a power-of-two scale, in 64 bits, from the
    format's definition: three mantissa bits, least exponent -6, largest value 448, halves to even; the scale is the
    least 2^e, e >= -127, with which the block's largest finite value is at most 448."""
    x = x.detach().double().cpu()
    m, k = x.shape
    p = x.new_zeros(m + -m % rows, k + -k % cols)
    p[:m, :k] = x
    v = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    big = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(dim=(1, 3), keepdim=True) if v.numel() else v.new_zeros(
        v.shape[0], 1, v.shape[2], 1)
    f, n = torch.frexp(big / 448)  # big / 448 may be rounded: 2^e * 448 is compared exactly below
    e = n.double()
    e = torch.where(big <= 448 * 2.0 ** (e - 1), e - 1, e)
    e = torch.where(big > 448 * 2.0 ** e, e + 1, e).clamp(min=-127)
    v = v / 2.0 ** e
    _, n = torch.frexp(v)  # |v| in [2^(n-1), 2^n)
    step = 2.0 ** ((n.double() - 1).clamp(min=-6) - 3)
    out = torch.round(v / step) * step * 2.0 ** e
    return torch.where(torch.isfinite(v), out, float("nan")).view(p.shape)[:m, :k]


def product_near(got, a, b, bias=None, exact_runs=True):
    """got = a b^T (+ bias), a [M, K] and b [N, K] the held values (64 bits).  Products of e4m3 values are exact in 32
    bits, so a sum is off by at most one rounding (2^-24 of the terms so far) an addition -- K of them, a few for slices
    and the bias -- and half a step of got's type.  With exact_runs=False (the GPU) a 16-bit result may lose, of each
    product, what lies below 2^-13 of the largest in its run of 8, and a 32-bit result a subnormal operand: the held
    values become bf16 operands, whose least normal value is 2^-126, so up to the value itself times the other operand."""
    want = a @ b.t()
    mag = a.abs() @ b.abs().t()
    lost = 0.0
    if not exact_runs and got.dtype == torch.float32:
        asub, bsub = (torch.where(t.abs() < 2.0 ** -126, t.abs(), 0.0) for t in (a, b))
        lost = asub @ b.abs().t() + a.abs() @ bsub.t()
    if not exact_runs and got.dtype != torch.float32:
        pad = torch.nn.functional.pad
        k = a.shape[1]
        ar, br = (pad(t.abs(), (0, -k % 8)).reshape(t.shape[0], -1, 8) for t in (a, b))
        for i in range(ar.shape[1]):
            lost = lost + (ar[:, None, i] * br[None, :, i]).amax(2)
        lost = lost * 8 * 2.0 ** -13
    if bias is not None:
        want = want + bias.detach().double().cpu()
        mag = mag + bias.detach().double().cpu().abs()
    r = (a.shape[1] + 64) * 2.0 ** -24
    near(got, want, mag + lost / r, roundings=r)
