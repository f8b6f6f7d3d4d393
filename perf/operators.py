"""Cases of the dense-block operators: what a deep CTR tower runs between its embeddings and its loss.

Three operators, each with a plain form (elementary torch operations in 32 bits, rounded once at the end) and the
framework's own call:

  fp8 fc         y = q(x) q(W) + b, operands in e4m3 with one power-of-two scale for each block of 128
                 (paddlebox_amd.ops.fp8: scaled_fp8fc, fp8_matmul)
  residual norm  r = x_scale x + y_scale gate * drop(norm_post(y)),  h = norm_pre(r)
                 (paddlebox_amd.ops.residual: residual_norm)
  dropout        a counter-based mask that is never stored  (paddlebox_amd.ops.dropout: dropout)

``own`` False: the plain forms.  ``own`` True: the calls a user makes.
"""
import torch

own = False

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one request's row through a packed layer: latency of a served token
        {"name": "fc serve 1 row", "op": "fc_serve", "rows": 1, "k": 1024, "o": 1024, "type": "bf16"},
        # a small serving batch against a wide layer: the weight's bytes are the cost
        {"name": "fc serve 48 rows", "op": "fc_serve", "rows": 48, "k": 8192, "o": 8192, "type": "bf16"},
        # one 400 -> 400 layer of the click model's tower at its batch, forward and backward
        {"name": "fc train tower", "op": "fc_train", "rows": 8192, "k": 400, "o": 400, "type": "fp32"},
        # the last, short batch of a pass through a layer of odd widths
        {"name": "fc train ragged", "op": "fc_train", "rows": 777, "k": 1023, "o": 333, "type": "fp16"},
        # a large dense layer, forward and backward
        {"name": "fc train large", "op": "fc_train", "rows": 16384, "k": 4096, "o": 4096, "type": "bf16"},
        # the product alone on operands that are held in 8 bits
        {"name": "matmul large", "op": "matmul", "rows": 8192, "k": 8192, "o": 8192, "type": "bf16"},
        # one token between two blocks at serving time
        {"name": "residual serve 1 row", "op": "residual", "rows": 1, "d": 4096, "type": "bf16", "stream": "bf16",
         "post": "rms", "pre": "rms", "gate": "channel", "act": "none", "p": 0.0, "train": False},
        # a residual tower block at the click model's batch: sandwich layer norms, a sigmoid gate, dropout
        {"name": "residual train tower", "op": "residual", "rows": 8192, "d": 400, "type": "fp32", "stream": "fp32",
         "post": "layer", "pre": "layer", "gate": "full", "act": "sigmoid", "p": 0.1, "train": True},
        # half-precision blocks on an fp32 stream, odd width, a gate for each row
        {"name": "residual train ragged", "op": "residual", "rows": 1000, "d": 1537, "type": "fp16", "stream": "fp32",
         "post": "none", "pre": "layer", "gate": "row", "act": "none", "p": 0.0, "train": True},
        # a large dense model's block boundary, forward and backward
        {"name": "residual train large", "op": "residual", "rows": 32768, "d": 4096, "type": "bf16", "stream": "bf16",
         "post": "rms", "pre": "rms", "gate": "channel", "act": "none", "p": 0.0, "train": True},
        # the activations of one tower layer
        {"name": "dropout tower", "op": "dropout", "rows": 8192, "d": 400, "type": "fp32", "p": 0.1},
        # the activations of a large layer
        {"name": "dropout large", "op": "dropout", "rows": 32768, "d": 8192, "type": "bf16", "p": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["fc_serve", "fc_train", "fc_train", "matmul", "residual", "residual", "dropout"])
    t = rng.choice(["fp32", "bf16", "fp16"])
    if op == "fc_serve":
        return {"op": op, "rows": _log(rng, 1, 64), "k": _log(rng, 256, 8192), "o": _log(rng, 256, 8192), "type": t}
    if op in ("fc_train", "matmul"):
        return {"op": op, "rows": _log(rng, 256, 16384), "k": _log(rng, 64, 4096), "o": _log(rng, 64, 4096), "type": t}
    if op == "dropout":
        return {"op": op, "rows": _log(rng, 1, 32768), "d": _log(rng, 64, 8192), "type": t,
                "p": rng.choice([0.0, 0.1, 0.25, 0.5, 0.9])}
    return {"op": op, "rows": _log(rng, 1, 16384), "d": _log(rng, 64, 4096), "type": t,
            "stream": rng.choice([t, "fp32"]), "post": rng.choice(["none", "rms", "layer"]),
            "pre": rng.choice(["rms", "layer"]), "gate": rng.choice(["none", "channel", "row", "full"]),
            "act": rng.choice(["none", "sigmoid"]), "p": rng.choice([0.0, 0.1, 0.5]),
            "train": rng.choice([True, True, False])}


def work(case):
    op, es = case["op"], SIZE[case["type"]]
    m = case["rows"]
    if op in ("fc_serve", "fc_train", "matmul"):
        k, o = case["k"], case["o"]
        if op == "matmul":  # codes and their scale bytes in, the product out
            return {"bytes": (m * k + o * k) * (1 + 1 / 128) + m * o * es, "flops": 2.0 * m * k * o}
        if op == "fc_serve":
            return {"bytes": m * k * es + o * k * (1 + 1 / 128) + 4 * o + m * o * es, "flops": 2.0 * m * k * o}
        # x, dy, W, b in; y, dx, dW, db out (W, b and their gradients are fp32 parameters)
        return {"bytes": 2 * m * k * es + 2 * m * o * es + 8 * k * o + 8 * o, "flops": 6.0 * m * k * o}
    n = m * case["d"]
    if op == "dropout":  # x, dy in; y, dx out
        return {"bytes": 4.0 * n * es, "flops": 2.0 * n}
    ss = SIZE[case["stream"]]
    full = case["gate"] == "full"
    fwd = 2 * n * ss + 2 * n * es + (n * es if full else 0)  # x, y (, gate) in; r, h out
    if not case["train"]:
        return {"bytes": float(fwd), "flops": 12.0 * n}
    # backward: dr, r, dh, y (, gate) in; dx, dy (, dgate) out
    bwd = 3 * n * ss + 3 * n * es + (2 * n * es if full else 0)
    return {"bytes": float(fwd + bwd), "flops": 40.0 * n}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _activations(g, m, k, dtype):
    """Activations as a tower has them: columns of very different scale, and a few that are zero."""
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32)
    x *= torch.exp(torch.randn(k, generator=g, device="cuda"))
    x *= torch.rand(k, generator=g, device="cuda") > 0.02
    return x.to(dtype)


def prepare(case, seed):
    g, op, dt, m = _gen(seed), case["op"], DT[case["type"]], case["rows"]
    s = {"case": case}
    if op in ("fc_serve", "fc_train", "matmul"):
        k, o = case["k"], case["o"]
        x = _activations(g, m, k, dt)
        w = _randn(g, k, o, scale=k ** -0.5)
        if op == "fc_train":
            s["x"], s["w"] = x.requires_grad_(), w.requires_grad_()
            s["b"] = _randn(g, o, scale=0.1).requires_grad_()
            s["dy"] = _randn(g, m, o, scale=1.0 / m, dtype=dt)
            return s
        # the weight as a checkpoint of packed layers holds it: codes and exponent bytes of W^T
        s["w_codes"], s["w_scales"] = _pack(w.t(), tile=True)
        if op == "matmul":
            s["x_codes"], s["x_scales"] = _pack(x.float(), tile=False)
        else:
            s["x"], s["b"] = x, _randn(g, o, scale=0.1)
        return s
    d = case["d"]
    s["seed"] = torch.tensor([seed * 0x9E3779B1 + 12345, seed + 7], dtype=torch.int64, device="cuda")
    if op == "dropout":
        s["x"] = _randn(g, m, d, dtype=dt).requires_grad_()
        s["dy"] = _randn(g, m, d, dtype=dt)
        return s
    st = DT[case["stream"]]
    s["x"], s["y"] = _randn(g, m, d, dtype=st), _randn(g, m, d, scale=2.0, dtype=dt)
    for name in ("post", "pre"):
        s[name + "_weight"] = 1 + _randn(g, d, scale=0.1) if case[name] != "none" else None
        s[name + "_bias"] = _randn(g, d, scale=0.1) if case[name] == "layer" else None
    kind = case["gate"]
    s["gate"] = (None if kind == "none" else _randn(g, d) if kind == "channel" else _randn(g, m, 1) if kind == "row"
                 else _randn(g, m, d, dtype=dt))
    if case["train"]:
        for name in ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias"):
            if s[name] is not None:
                s[name].requires_grad_()
        s["dr"], s["dh"] = _randn(g, m, d, dtype=st), _randn(g, m, d, dtype=dt)
    return s


X_SCALE, Y_SCALE, EPS = 1.0, 0.5, 1e-6


# ------------------------------------------------------------------ plain forms: 8-bit blocks
def _exponents(amax):
    """The least e with amax <= 448 * 2^e, within a byte: amax = f 2^n with f in [0.5, 1), 448 = 0.875 * 2^9."""
    f, n = torch.frexp(amax)
    return (n - 9 + (f > 0.875).to(n.dtype)).clamp(-127, 127)


def _blocks(x, tile):
    """x padded to whole blocks, and the exponent of each block's scale (tile: 128 x 128, else 1 x 128)."""
    m, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % 128, 0, -m % 128 if tile else 0))
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).reshape(x.shape[0], -1, 128).amax(2)
    if tile:
        a = a.reshape(-1, 128, a.shape[1]).amax(1).repeat_interleave(128, 0)
    return x, _exponents(a)


def _two_to(e):
    """2^e for whole e in [-127, 127], exactly (a power function may be off by a bit)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _codes(x, e):
    v = x * _two_to(-e).repeat_interleave(128, 1)
    return torch.where(torch.isfinite(v), v, torch.full_like(v, float("nan"))).to(torch.float8_e4m3fn)


def _pack(x, tile):
    """Codes [rows, K up to a whole block] and exponent bytes [rows, blocks up to a multiple of 4] of a float matrix."""
    m = x.shape[0]
    x, e = _blocks(x, tile)
    c = _codes(x, e)[:m].contiguous()
    s = torch.nn.functional.pad((e[:m] + 127).to(torch.uint8), (0, -e.shape[1] % 4), value=127)
    return c, s.contiguous()


def _values(codes, scales):
    e = scales[:, : codes.shape[1] // 128].to(torch.int32) - 127
    return codes.float() * _two_to(e).repeat_interleave(128, 1)


def _q(x, tile=False):
    """What x stands for once it is held in 8 bits, its own shape, fp32."""
    m, k = x.shape
    p, e = _blocks(x, tile)
    return (_codes(p, e).float() * _two_to(e).repeat_interleave(128, 1))[:m, :k]


def _fc_plain(s):
    case, dt = s["case"], DT[s["case"]["type"]]
    if case["op"] == "matmul":
        return (_values(s["x_codes"], s["x_scales"]) @ _values(s["w_codes"], s["w_scales"]).t()).to(dt)
    x = s["x"].detach().float()
    if case["op"] == "fc_serve":
        return (_q(x) @ _values(s["w_codes"], s["w_scales"])[:, : case["k"]].t() + s["b"]).to(dt)
    w, dy = _q(s["w"].detach(), tile=True), s["dy"].float()
    y = _q(x) @ w + s["b"].detach()
    dx = _q(dy) @ w.t()
    dw = _q(x.t()) @ _q(dy.t()).t()  # both run over the batch: blocks of 128 rows
    return {"y": y.to(dt), "dx": dx.to(dt), "dw": dw, "db": dy.sum(0)}


# ------------------------------------------------------------------ plain forms: counter-based mask
def _rounds(c, k0, k1):
    """Ten rounds of Philox 4x32 (Salmon et al., 2011) on four int64 tensors that hold 32-bit words."""
    low = 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32 & low) ^ c[1] ^ k0, p1 & low, (p0 >> 32 & low) ^ c[3] ^ k1, p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _keep(seed, n, p):
    """The mask of n elements: element i takes 16 bits of block i // 8, and stays where they are not under p 2^16."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 7) // 8, dtype=torch.int64, device=seed.device)
    z = torch.zeros_like(i)
    words = _rounds([i & low, i >> 32, z + (seed[1] & low), z + (seed[1] >> 32 & low)], seed[0] & low, seed[0] >> 32 & low)
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).reshape(-1)[:n]
    return bits >= round(p * 65536)


def _mask(s, shape):
    p = s["case"]["p"]
    return _keep(s["seed"], shape[0] * shape[1], p).reshape(shape), 65536.0 / (65536 - round(p * 65536))


def _dropout_plain(s):
    dt = DT[s["case"]["type"]]
    keep, up = _mask(s, s["x"].shape)
    y = torch.where(keep, s["x"].detach().float() * up, 0.0)
    dx = torch.where(keep, s["dy"].float() * up, 0.0)
    return {"y": y.to(dt), "dx": dx.to(dt)}


# ------------------------------------------------------------------ plain forms: residual norm
def _norm(v, kind, weight, bias):
    """(output, normalised value, 1 / deviation) in fp32."""
    if kind == "none":
        return v, v, None
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    inv = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    n = c * inv
    return (n * weight + bias if bias is not None else n * weight), n, inv


def _norm_back(d, kind, n, inv, weight):
    """Gradients of the norm's input, weight and bias."""
    if kind == "none":
        return d, None, None
    g = d * weight
    dv = inv * (g - n * (g * n).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if kind == "layer" else 0.0))
    return dv, (d * n).sum(0), (d.sum(0) if kind == "layer" else None)


def _residual_plain(s):
    c = s["case"]
    dt, st = DT[c["type"]], DT[c["stream"]]
    f = {k: v.detach().float() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    get = f.get
    u, un, uinv = _norm(f["y"], c["post"], get("post_weight"), get("post_bias"))
    keep, up = _mask(s, u.shape) if c["p"] > 0 else (torch.ones_like(u, dtype=torch.bool), 1.0)
    du_f = torch.where(keep, u * up, 0.0)
    raw = get("gate")
    gate = torch.ones((), device=u.device) if raw is None else 1 / (1 + torch.exp(-raw)) if c["act"] == "sigmoid" else raw
    r = X_SCALE * f["x"] + Y_SCALE * gate * du_f
    h, hn, hinv = _norm(r, c["pre"], get("pre_weight"), get("pre_bias"))
    if not c["train"]:
        return {"r": r.to(st), "h": h.to(dt)}
    dv, dpw, dpb = _norm_back(f["dh"], c["pre"], hn, hinv, get("pre_weight"))
    t = f["dr"] + dv
    out = {"r": r.to(st), "h": h.to(dt), "dx": (X_SCALE * t).to(st), "dpre_weight": dpw, "dpre_bias": dpb}
    if raw is not None:
        dg = Y_SCALE * t * du_f
        if c["act"] == "sigmoid":
            dg = dg * gate * (1 - gate)
        out["dgate"] = dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True) if c["gate"] == "row" else dg.to(dt)
    du = torch.where(keep, Y_SCALE * t * gate * up, 0.0)
    dy, out["dpost_weight"], out["dpost_bias"] = _norm_back(du, c["post"], un, uinv, get("post_weight"))
    out["dy"] = dy.to(dt)
    return out


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return _dropout_plain(s) if op == "dropout" else _residual_plain(s) if op == "residual" else _fc_plain(s)
    if op == "dropout":
        from paddlebox_amd.ops.dropout import dropout

        y = dropout(s["x"], case["p"], s["seed"])
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "dx": dx}
    if op == "residual":
        from paddlebox_amd.ops.residual import residual_norm

        r, h = residual_norm(s["x"], s["y"], x_scale=X_SCALE, y_scale=Y_SCALE, gate=s["gate"], gate_act=case["act"],
                             post=case["post"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                             pre=case["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], eps=EPS,
                             p=case["p"], seed=s["seed"])
        out = {"r": r.detach(), "h": h.detach()}
        if case["train"]:
            names = [n for n in ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[n] is not None]
            grads = torch.autograd.grad((r, h), [s[n] for n in names], (s["dr"], s["dh"]))
            out.update({"d" + n: g for n, g in zip(names, grads)})
        return out
    from paddlebox_amd.ops.fp8 import Fp8Blocks, fp8_matmul, scaled_fp8fc

    if op == "matmul":
        return fp8_matmul(Fp8Blocks(s["x_codes"], s["x_scales"], case["k"]),
                          Fp8Blocks(s["w_codes"], s["w_scales"], case["k"]), out_dtype=DT[case["type"]])
    if op == "fc_serve":
        return scaled_fp8fc(s["x"], Fp8Blocks(s["w_codes"], s["w_scales"], case["k"]), s["b"])
    y = scaled_fp8fc(s["x"], s["w"], s["b"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _power(e):
    """2^e in 64 bits for whole e between -200 and 200, from a table."""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=e.device)[e.long() + 200]


def _held(x, rows, cols):
    """x (float64) as blocks of rows x cols hold it in e4m3 with a power-of-two scale, from the format's definition:
    three mantissa bits, least exponent -6, largest value 448, halves to even."""
    m, k = x.shape
    p = x.new_zeros(m + -m % rows, k + -k % cols)
    p[:m, :k] = x
    v = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    big = v.abs().amax(dim=(1, 3), keepdim=True)
    e = torch.ceil(torch.log2(torch.where(big > 0, big, torch.ones_like(big)) / 448))
    e = e + (big > 448 * _power(e)).double() - (big <= 448 * _power(e - 1)).double()  # the logarithm may be off next to a border
    v = v / _power(e)
    a = v.abs().clamp(min=2.0 ** -6)
    lg = torch.floor(torch.log2(a))
    lg = lg + (_power(lg + 1) <= a).double() - (_power(lg) > a).double()
    step = _power(lg - 3)
    return (torch.round(v / step) * step * _power(e)).view(p.shape)[:m, :k]


def _exact_values(c, e):
    return c.double() * _power(e[:, : c.shape[1] // 128].double() - 127).repeat_interleave(128, 1)


def _exact_words(seed, offset, n, device):
    """Philox 4x32-10 on 16-bit halves, so that no product leaves 53 bits."""
    def mul(a, m):
        al, ah, ml, mh = a % 65536, a // 65536, m % 65536, m // 65536
        low, mid1, mid2, high = al * ml, ah * ml, al * mh, ah * mh
        mid = low // 65536 + mid1 % 65536 + mid2 % 65536
        return high + mid1 // 65536 + mid2 // 65536 + mid // 65536, (mid % 65536) * 65536 + low % 65536

    i = torch.arange(n, dtype=torch.int64, device=device)
    c0, c1 = i % 2 ** 32, i // 2 ** 32
    c2, c3 = torch.full_like(i, offset % 2 ** 32), torch.full_like(i, offset // 2 ** 32 % 2 ** 32)
    k0, k1 = seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32
    for _ in range(10):
        h0, l0 = mul(c0, 0xD2511F53)
        h1, l1 = mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return c0, c1, c2, c3


def _exact_scale(s, m, d):
    """0 or 1 / (1 - p), p in steps of 2^-16, for each element, in 64 bits."""
    t = round(s["case"]["p"] * 65536)
    seed, offset = (int(v) for v in s["seed"].tolist())
    n = m * d
    out = torch.empty((n + 7) // 8, 8, dtype=torch.float64, device=s["seed"].device)
    for j, w in enumerate(_exact_words(seed, offset, out.shape[0], out.device)):
        out[:, 2 * j] = (w % 65536 >= t).double()
        out[:, 2 * j + 1] = (w // 65536 >= t).double()
    return out.reshape(-1)[:n].reshape(m, d) * (65536.0 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    op, m = case["op"], case["rows"]
    if op == "matmul":
        return _exact_values(s["x_codes"], s["x_scales"]) @ _exact_values(s["w_codes"], s["w_scales"]).t()
    if op == "fc_serve":
        w = _exact_values(s["w_codes"], s["w_scales"])[:, : case["k"]]
        return _held(s["x"].double(), 1, 128) @ w.t() + s["b"].double()
    if op == "fc_train":
        x, w, dy = (s[n].detach().double() for n in ("x", "w", "dy"))
        y = _held(x, 1, 128) @ _held(w, 128, 128) + s["b"].detach().double()
        dx = _held(dy, 1, 128) @ _held(w, 128, 128).t()
        dw = _held(x, 128, 1).t() @ _held(dy, 128, 1)
        return {"y": y, "dx": dx, "dw": dw, "db": dy.sum(0)}
    if op == "dropout":
        k = _exact_scale(s, m, case["d"])
        return {"y": s["x"].detach().double() * k, "dx": s["dy"].double() * k}
    # residual norm: the definition, differentiated in 64 bits
    names = [n for n in ("x", "y", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[n] is not None]
    v = {n: s[n].detach().double().requires_grad_(case["train"]) for n in names}

    def norm(t, which):
        kind = case[which]
        if kind == "none":
            return t
        if kind == "layer":
            return (t - t.mean(1, keepdim=True)) / (t.var(1, keepdim=True, correction=0) + EPS).sqrt() \
                * v[which + "_weight"] + v[which + "_bias"]
        return t / (t.square().mean(1, keepdim=True) + EPS).sqrt() * v[which + "_weight"]

    branch = norm(v["y"], "post")
    if case["p"] > 0:
        branch = branch * _exact_scale(s, m, case["d"])
    if s["gate"] is not None:
        branch = branch * (torch.sigmoid(v["gate"]) if case["act"] == "sigmoid" else v["gate"])
    r = X_SCALE * v["x"] + Y_SCALE * branch
    h = norm(r, "pre")
    out = {"r": r.detach(), "h": h.detach()}
    if case["train"]:
        grads = torch.autograd.grad((r, h), [v[n] for n in names], (s["dr"].double(), s["dh"].double()))
        out.update({"d" + n: g for n, g in zip(names, grads)})
    return out
