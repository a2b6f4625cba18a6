"""What is measured of the 8-bit linear layer: its operators' cases, their plain form in elementary torch operations, and the
framework's calls.

Numbers are held as e4m3 with one power-of-two scale (e8m0) for each block: 128 neighbouring values of a row ("row"), or a tile of
128 x 128 ("tile").  A block's scale is the smallest 2^e with max|v| <= 448 * 2^e, 1 for a block of zeros, NaN for a block that
holds an infinity or a NaN; the values are v / 2^e, rounded once, to nearest even.

  quantize   x -> (q, scale): the 8-bit form of activations ("row", also how they are kept for the backward pass) and weights ("tile")
  norm       h = x + residual; y = h * rstd * weight, rstd = 1 / sqrt(mean(h^2) + eps); (q, scale) of y by rows, h, rstd
  norm_back  the gradients of x (and of the residual, which is the same) and of weight, from dy and the gradient of h
  gemm       C = A * B^T or A * B of 8-bit operands
  wgrad      dW = dY^T * X, dY in 16 bits and X kept in 8 bits by the forward pass
"""
import math

import torch

own = False

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decoding step: latency
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "residual": True},
        # a prompt's tokens, with a count that divides by nothing
        {"name": "norm_4001x5120", "op": "norm", "rows": 4001, "cols": 5120, "type": "f16", "residual": True},
        # a training step's norm, its residual stream's gradient added
        {"name": "norm_back_8192x8192", "op": "norm_back", "rows": 8192, "cols": 8192, "type": "bf16", "residual": True},
        # a small batch with a ragged width, first layer (nothing to add)
        {"name": "norm_back_777x1000", "op": "norm_back", "rows": 777, "cols": 1000, "type": "f16", "residual": False},
        # activations kept in 8 bits for the backward pass, ragged
        {"name": "quantize_row_4000x3000", "op": "quantize", "rows": 4000, "cols": 3000, "type": "f16", "tile": False},
        # a layer's weights after an optimizer step
        {"name": "quantize_tile_16384x4096", "op": "quantize", "rows": 16384, "cols": 4096, "type": "bf16", "tile": True},
        # one decoding step of a few sequences: bound by the weights' bytes
        {"name": "gemm_8x4096x4096", "op": "gemm", "m": 8, "n": 4096, "k": 4096, "type": "bf16", "trans_b": True, "tile": True},
        # a layer's forward product in training
        {"name": "gemm_8192x8192x8192", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "trans_b": True, "tile": True},
        # ragged in every size, weights with a scale for each row
        {"name": "gemm_4000x5120x3000", "op": "gemm", "m": 4000, "n": 5120, "k": 3000, "type": "f16", "trans_b": True, "tile": False},
        # the input's gradient: the same weights, not transposed
        {"name": "gemm_nn_4096x4096x4096", "op": "gemm", "m": 4096, "n": 4096, "k": 4096, "type": "f16", "trans_b": False, "tile": True},
        # the weights' gradient over a training step's tokens
        {"name": "wgrad_8192x4096x4096", "op": "wgrad", "tokens": 8192, "n": 4096, "k": 4096, "type": "bf16"},
        # the same with ragged sizes and few output tiles for its tokens
        {"name": "wgrad_5000x1000x1032", "op": "wgrad", "tokens": 5000, "n": 1000, "k": 1032, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_back", "quantize", "gemm", "gemm", "wgrad"])
    kind = rng.choice(sorted(TYPES))
    if op in ("norm", "norm_back"):
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 64, 8192), "type": kind, "residual": rng.random() < 0.7}
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 64, 8192), "type": kind, "tile": rng.random() < 0.5}
    if op == "gemm":
        trans = rng.random() < 0.7
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 128, 8192), "k": _log(rng, 128, 8192), "type": kind,
                "trans_b": trans, "tile": not trans or rng.random() < 0.5}
    # dY's rows are whole 16-byte units
    return {"op": op, "tokens": _log(rng, 64, 8192), "n": 8 * _log(rng, 16, 640), "k": _log(rng, 128, 5120), "type": kind}


def work(case):
    if case["op"] in ("norm", "norm_back", "quantize"):
        n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
        blocks = -(-cols // 128)
        if case["op"] == "quantize":
            return {"bytes": 3 * n + (-(-rows // 128) if case["tile"] else rows) * blocks, "flops": 3 * n}
        if case["op"] == "norm":  # x (and residual in, h out), 8 bits out
            return {"bytes": (7 if case["residual"] else 3) * n + rows * blocks + 4 * rows + 2 * cols, "flops": 8 * n}
        return {"bytes": (8 if case["residual"] else 6) * n + 4 * rows + 6 * cols, "flops": 12 * n}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // 128)
        return {"bytes": m * k + n * k + 2 * m * n + m * blocks + (-(-n // 128) if case["tile"] else n) * blocks, "flops": 2 * m * n * k}
    t, n, k = case["tokens"], case["n"], case["k"]
    return {"bytes": 2 * t * n + t * k + t * -(-k // 128) + 2 * n * k, "flops": 2 * t * n * k}


# ------------------------------------------------------------------------------------------------ plain forms
def _blocks(v, tile):
    """v as [row blocks, rows of one, column blocks, 128], filled up with zeros."""
    rows, cols = v.shape
    r = 128 if tile else 1
    v = torch.nn.functional.pad(v, (0, -cols % 128, 0, -rows % r))
    return v.reshape(v.shape[0] // r, r, v.shape[1] // 128, 128)


def _quantize(v, tile):
    """The 8-bit form of float32 values: (e4m3, e8m0)."""
    rows, cols = v.shape
    b = _blocks(v, tile)
    top = b.abs().amax(dim=(1, 3))
    part, e = torch.frexp(top)  # top = part * 2^e, part in [1/2, 1): 448 = 0.875 * 2^9
    e = torch.where(part <= 0.875, e - 9, e - 8).clamp(-127, 127)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    fine = torch.isfinite(top)
    e = torch.where(fine, e, torch.full_like(e, 128))
    half = torch.div(-e, 2, rounding_mode="floor")  # 2^-e in two factors: each is a normal number
    y = b * torch.exp2(half.float())[:, None, :, None] * torch.exp2((-e - half).float())[:, None, :, None]
    y = torch.where(fine[:, None, :, None], y, torch.full_like(y, float("nan")))
    q = y.reshape(-1, b.shape[2] * 128)[:rows, :cols].to(F8)
    return q, (e + 127).to(torch.uint8).view(E8)


def _values(q, scale, tile):
    """The float32 values that an 8-bit matrix stands for."""
    s = scale.float()
    if tile:
        s = s.repeat_interleave(128, dim=0)[: q.shape[0]]
    return q.float() * s.repeat_interleave(128, dim=1)[:, : q.shape[1]]


def _plain_norm(s):
    x = s["x"].float()
    h = s["x"]
    if s["residual"] is not None:
        h = (x + s["residual"].float()).to(s["x"].dtype)
    hf = h.float()
    rstd = 1.0 / torch.sqrt((hf * hf).mean(dim=1) + EPS)
    q, scale = _quantize(hf * rstd[:, None] * s["weight"].float(), False)
    return {"q": q, "scale": scale, "h": h, "rstd": rstd}


def _plain_norm_back(s):
    dy, h = s["dy"].float(), s["h"].float()
    xhat = h * s["rstd"][:, None]
    g = dy * s["weight"].float()
    dx = s["rstd"][:, None] * (g - xhat * (g * xhat).mean(dim=1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["dy"].dtype), "dweight": (dy * xhat).sum(dim=0)}


def _plain_quantize(s):
    q, scale = _quantize(s["x"].float(), s["tile"])
    return {"q": q, "scale": scale}


def _plain_gemm(s):
    a, b = _values(s["a"], s["a_scale"], False), _values(s["b"], s["b_scale"], s["tile"])
    return (a @ (b.t() if s["trans_b"] else b)).to(s["type"])


def _plain_wgrad(s):
    return (s["dy"].float().t() @ _values(s["x"], s["x_scale"], False)).to(s["type"])


# ------------------------------------------------------------------------------------------------ inputs
def _normal(gen, rows, cols, std, kind):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * std).to(kind)


def _activations(gen, rows, cols, kind):
    """Hidden states: some channels are much larger than the rest."""
    channel = torch.exp(0.5 * torch.randn(1, cols, generator=gen, device="cuda"))
    channel = torch.where(torch.rand(1, cols, generator=gen, device="cuda") < 0.01, channel * 16, channel)
    return (torch.randn(rows, cols, generator=gen, device="cuda") * channel).to(kind)


def _padded(v):
    """An 8-bit matrix as the framework's quantizers lay it out: rows start at multiples of 16 bytes."""
    rows, cols = v.shape
    room = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=v.device).view(F8)
    room[:, :cols].copy_(v)
    return room[:, :cols]


def _kept(v, tile):
    q, scale = _quantize(v.float(), tile)
    return _padded(q), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, op = TYPES[case["type"]], case["op"]
    s = {"op": op, "type": kind}
    if op in ("norm", "norm_back"):
        rows, cols = case["rows"], case["cols"]
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(kind)
    if op == "norm":
        s["x"] = _normal(gen, rows, cols, 0.5, kind)
        s["residual"] = _activations(gen, rows, cols, kind) if case["residual"] else None
    elif op == "norm_back":
        s["h"] = _activations(gen, rows, cols, kind)
        s["rstd"] = 1.0 / torch.sqrt(s["h"].float().square().mean(dim=1) + EPS)
        s["dy"] = _normal(gen, rows, cols, 0.1, kind)
        s["dres"] = _normal(gen, rows, cols, 0.1, kind) if case["residual"] else None
    elif op == "quantize":
        s["tile"] = case["tile"]
        s["x"] = _normal(gen, case["rows"], case["cols"], 0.02, kind) if case["tile"] else _activations(gen, case["rows"], case["cols"], kind)
    elif op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        s["trans_b"], s["tile"] = case["trans_b"], case["tile"]
        s["a"], s["a_scale"] = _kept(_activations(gen, m, k, kind), False)
        s["b"], s["b_scale"] = _kept(_normal(gen, *((n, k) if case["trans_b"] else (k, n)), 0.02, kind), case["tile"])
    else:
        s["dy"] = _normal(gen, case["tokens"], case["n"], 0.1, kind)
        s["x"], s["x_scale"] = _kept(_activations(gen, case["tokens"], case["k"], kind), False)
    return s


# ------------------------------------------------------------------------------------------------ a pass
def run(state):
    s, op = state, state["op"]
    if own:
        import vibekernel_b200 as vk
        if op == "norm":
            q, scale, h, rstd = vk.rmsnorm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
            return {"q": q, "scale": scale, "h": h, "rstd": rstd}
        if op == "norm_back":
            dx, dweight = vk.rmsnorm_fp8_backward(s["dy"], s["h"], s["weight"], s["rstd"], dres=s["dres"])
            return {"dx": dx, "dweight": dweight}
        if op == "quantize":
            q, scale = vk.quantize_fp8(s["x"], tile=s["tile"])
            return {"q": q, "scale": scale}
        if op == "gemm":
            return vk.gemm_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], trans_b=s["trans_b"], out_dtype=s["type"])
        return vk.wgrad_fp8(s["dy"], s["x"], s["x_scale"], out_dtype=s["type"])
    return {"norm": _plain_norm, "norm_back": _plain_norm_back, "quantize": _plain_quantize, "gemm": _plain_gemm, "wgrad": _plain_wgrad}[op](s)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_quantize(v, r):
    """q before its rounding and scale, in 64 bits, of blocks of r rows and 128 columns."""
    rows, cols = v.shape
    top = torch.zeros(-(-rows // r) * r, -(-cols // 128) * 128, dtype=torch.float64, device=v.device)
    top[:rows, :cols] = v.abs()
    top = top.unflatten(1, (-1, 128)).amax(dim=2).unflatten(0, (-1, r)).amax(dim=1)
    step = torch.exp2(torch.ceil(torch.log2(top / 448)))
    step = torch.where(top > 448 * step, 2 * step, torch.where(top <= 224 * step, step / 2, step))  # log2's own rounding
    step = torch.where(top == 0, torch.ones_like(step), step)
    wide = step.repeat_interleave(r, dim=0)[:rows].repeat_interleave(128, dim=1)[:, :cols]
    return v / wide, step


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "quantize":
        q, scale = _exact_quantize(d["x"], 128 if case["tile"] else 1)
        return {"q": q, "scale": scale}
    if case["op"] == "norm":
        total = d["x"] + d["residual"] if case["residual"] else d["x"]
        h = total.to(s["type"]).double()  # the norm is that of h as it is stored
        rstd = (h.square().sum(dim=1) / case["cols"] + EPS).pow(-0.5)
        q, scale = _exact_quantize(h * d["weight"] * rstd.unsqueeze(1), 1)
        return {"q": q, "scale": scale, "h": total, "rstd": rstd}
    if case["op"] == "norm_back":
        n = case["cols"]
        r = d["rstd"].unsqueeze(1)
        inner = torch.einsum("ij,j,ij->i", d["dy"], d["weight"], d["h"]).unsqueeze(1)
        dx = r * d["weight"] * d["dy"] - r.pow(3) / n * inner * d["h"]
        if case["residual"]:
            dx += d["dres"]
        return {"dx": dx, "dweight": torch.einsum("ij,ij,i->j", d["dy"], d["h"], d["rstd"])}

    def wide(q, scale, tile):
        col = torch.arange(q.shape[1], device=q.device) // 128
        row = torch.arange(q.shape[0], device=q.device) // (128 if tile else 1)
        return q * scale[row][:, col]

    if case["op"] == "gemm":
        a, b = wide(d["a"], d["a_scale"], False), wide(d["b"], d["b_scale"], case["tile"])
        return torch.einsum("mk,nk->mn" if case["trans_b"] else "mk,kn->mn", a, b)
    return torch.einsum("tn,tk->nk", d["dy"], wide(d["x"], d["x_scale"], False))
