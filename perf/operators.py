"""The training-step operators around the NVFP4 cast, as measured cases.

Each operator is computed two ways: `own` false gives its plain form in
elementary torch operations, `own` true makes the calls of the
fp4_sm120a_b200 package.  Operators:

  gemm                  D = act(A B^T + bias) + residual of two NVFP4 operands
  gemm_dact             D = (A B^T) * act'(aux) and its column sums (the bias gradient)
  layernorm             layer norm, with the amax that the cast of its output needs
  layernorm_backward    its input gradient (plus a residual's) and the weights' gradients
  adamw                 an AdamW step over many tensors, states in 32 or in 8 bits
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = 128  # elements that share one scale in the 8-bit optimizer states
EPS = 1e-5
ADAM = {"lr": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8}


# ----------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------

def gemm(m, n, k, out="bf16", act="none", bias=False, residual=False, aux=False, amax=False):
    return {"op": "gemm", "m": m, "n": n, "k": k, "out": out, "act": act, "bias": bias,
            "residual": residual, "aux": aux, "amax": amax}


def gemm_dact(m, n, k, out="bf16", act="gelu", dbias=True, amax=True):
    return {"op": "gemm_dact", "m": m, "n": n, "k": k, "out": out, "act": act, "dbias": dbias,
            "amax": amax}


def layernorm(rows, cols, dtype="bf16", weight="f32", amax=True):
    return {"op": "layernorm", "rows": rows, "cols": cols, "dtype": dtype, "weight": weight,
            "amax": amax}


def layernorm_backward(rows, cols, dtype="bf16", weight="f32", residual=True):
    return {"op": "layernorm_backward", "rows": rows, "cols": cols, "dtype": dtype,
            "weight": weight, "residual": residual}


def adamw(layers, width, ffn, state, grad="bf16"):
    return {"op": "adamw", "layers": layers, "width": width, "ffn": ffn, "state": state,
            "grad": grad}


def listed():
    return [
        # One token through one linear layer: the weights' bytes and the launch count.
        {"name": "gemm one token", **gemm(1, 5120, 5120, bias=True)},
        # A handful of sequences decoded together, ragged in both directions.
        {"name": "gemm 37 tokens ragged", **gemm(37, 5000, 8192, act="silu", bias=True,
                                                 residual=True)},
        # The first product of an MLP block: activation, its argument for the
        # backward pass, and the amax for the cast of its output.
        {"name": "gemm mlp up", **gemm(8192, 14336, 5120, act="gelu", bias=True, aux=True,
                                       amax=True)},
        # A weight gradient over 8192 tokens, added to an fp32 accumulator.
        {"name": "gemm weight gradient", **gemm(5120, 14336, 8192, out="f32", residual=True)},
        # The gradient at an MLP's inner activation for a short fine-tuning batch.
        {"name": "gemm dact short", **gemm_dact(200, 5120, 1280)},
        # The same at an odd number of tokens of the full model.
        {"name": "gemm dact long", **gemm_dact(4099, 14336, 5120)},
        # A decode step's layer norm: latency.
        {"name": "layernorm 16 rows", **layernorm(16, 5120)},
        # A training batch's layer norm.
        {"name": "layernorm training", **layernorm(16384, 8192)},
        # Odd rows and columns in 32 bits: nothing divides a vector.
        {"name": "layernorm backward odd", **layernorm_backward(1003, 4099, dtype="f32")},
        # A training batch's backward pass, joined with the residual stream's gradient.
        {"name": "layernorm backward training", **layernorm_backward(16384, 5120)},
        # A small adapter's parameters: many short tensors, states in 32 bits.
        {"name": "adamw adapters", **adamw(16, 257, 130, "32", grad="f32")},
        # Two MLP layers' master weights, gradients in bf16, states in 8 bits.
        {"name": "adamw mlp 8 bits", **adamw(2, 5120, 14336, "8")},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm_dact", "layernorm", "layernorm_backward", "adamw"])
    if op in ("gemm", "gemm_dact"):
        m, n = _log(rng, 1, 8192), _log(rng, 64, 14336)
        k = 32 * _log(rng, 1, 256)
        out = rng.choice(["bf16", "bf16", "f16", "f32"])
        act = rng.choice(["none", "relu", "gelu", "silu"])
        flag = [rng.random() < 0.5 for _ in range(4)]
        if op == "gemm":
            return gemm(m, n, k, out, act, flag[0], flag[1], flag[2], flag[3])
        return gemm_dact(m, n, k, out, act, flag[0], flag[1])
    if op in ("layernorm", "layernorm_backward"):
        rows, cols = _log(rng, 1, 16384), _log(rng, 16, 8192)
        if rng.random() < 0.5:
            cols = max(16, cols // 64 * 64)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        weight = rng.choice(["f32", dtype])
        flag = rng.random() < 0.5
        return (layernorm if op == "layernorm" else layernorm_backward)(rows, cols, dtype, weight,
                                                                        flag)
    layers, width = rng.randint(1, 8), _log(rng, 16, 2560)
    return adamw(layers, width, _log(rng, 16, 6144), rng.choice(["32", "8"]),
                 rng.choice(["f32", "bf16"]))


def work(case):
    op = case["op"]
    if op in ("gemm", "gemm_dact"):
        m, n, k, out = case["m"], case["n"], case["k"], BYTES[case["out"]]
        total = (m + n) * (k // 2 + k // 16) + 8 + m * n * out
        if op == "gemm":
            total += n * 4 * case["bias"] + m * n * out * (case["residual"] + case["aux"])
        else:
            total += m * n * out + n * 4 * case["dbias"]
        return {"bytes": total + 4 * case["amax"], "flops": 2 * m * n * k}
    if op == "layernorm":
        r, c, w = case["rows"], case["cols"], BYTES[case["weight"]]
        return {"bytes": 2 * r * c * BYTES[case["dtype"]] + 2 * c * w + 8 * r, "flops": 8 * r * c}
    if op == "layernorm_backward":
        r, c, w = case["rows"], case["cols"], BYTES[case["weight"]]
        return {"bytes": (3 + case["residual"]) * r * c * BYTES[case["dtype"]] + 3 * c * w + 8 * r,
                "flops": 16 * r * c}
    n = sum(size for size, _ in _tensors(case))
    # master weight read and written, gradient read, bf16 weight written; the
    # states read and written, and in 8 bits read back as values
    states = 16 if case["state"] == "32" else 4 + 2 + 4 + 6 / BLOCK
    return {"bytes": n * (8 + BYTES[case["grad"]] + 2 + states), "flops": 20 * n}


# ----------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------

def _nvfp4(g, rows, k, spread):
    """A random matrix as the cast leaves it: packed E2M1 codes (rows x k/2), E4M3
    scales of 16-element blocks (rows x k/16) and the amax they were derived from."""
    x = torch.randn(rows, k, device="cuda", generator=g) * spread
    x[torch.rand(rows, k, device="cuda", generator=g) < 0.001] *= 10.0
    amax = x.abs().amax().reshape(1)
    enc = 2688.0 / amax
    blocks = x.view(rows, k // 16, 16)
    scale = (blocks.abs().amax(2) * (enc / 6.0)).to(torch.float8_e4m3fn)
    inv = enc / scale.float().clamp_min(2.0 ** -9)
    blocks.mul_(inv[:, :, None])
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    code = torch.bucketize(x.abs(), edges, out_int32=True).to(torch.uint8)
    code |= (x < 0).to(torch.uint8) << 3
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    return codes, scale.view(torch.uint8), amax


def _tensors(case):
    """(elements, weight decay) of each tensor: per layer a norm's two vectors, two
    matrices and their biases."""
    w, f = case["width"], case["ffn"]
    return [(w, 0.0), (w, 0.0), (f * w, 0.1), (f, 0.0), (w * f, 0.1), (w, 0.0)] * case["layers"]


def _blocks8(x, levels):
    """Codes and scale bytes of a flat tensor in the 8-bit state format (sign apart):
    a power of two for each block, `levels` mantissa steps, rounded to nearest."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1)
    scale = (torch.frexp(top)[1] + 126 - 7).clamp(1, 254)
    y = torch.ldexp(b.abs(), (127 - scale)[:, None])
    exponent = (torch.frexp(y)[1] - 1).clamp_min(-6)
    q = torch.round(torch.ldexp(y, -exponent) * levels).to(torch.int32)
    code = (exponent + 6) * levels + q
    return torch.where(y > 0, code, torch.zeros_like(code)).to(torch.uint8).view(-1), scale.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s, op = dict(case), case["op"]
    if op in ("gemm", "gemm_dact"):
        m, n, k, out = case["m"], case["n"], case["k"], DTYPES[case["out"]]
        s["a"] = _nvfp4(g, m, k, 1.0)
        s["b"] = _nvfp4(g, n, k, 1.0 / math.sqrt(k))
        if op == "gemm":
            s["bias_t"] = rand(n) if case["bias"] else None
            s["residual_t"] = rand(m, n).to(out) if case["residual"] else None
        else:
            s["aux_t"] = rand(m, n).to(out)
    elif op == "layernorm":
        r, c = case["rows"], case["cols"]
        s["x"] = (rand(r, c) * (rand(c).abs() + 0.3) + 0.5).to(DTYPES[case["dtype"]])
        s["gamma"], s["beta"] = ((rand(c) * 0.2 + o).to(DTYPES[case["weight"]]) for o in (1.0, 0.0))
    elif op == "layernorm_backward":
        r, c, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]
        s["x"] = (rand(r, c) * (rand(c).abs() + 0.3) + 0.5).to(dtype)
        wide = s["x"].double()
        mean = wide.mean(1)
        s["mean"] = mean.float()
        s["rstd"] = (wide.var(1, unbiased=False) + EPS).rsqrt().float()
        s["gamma"] = (rand(c) * 0.2 + 1.0).to(DTYPES[case["weight"]])
        s["dy"] = rand(r, c).to(dtype)
        s["residual_t"] = rand(r, c).to(dtype) if case["residual"] else None
    else:
        # One flat buffer of each kind; every tensor starts at a multiple of BLOCK.
        tensors = _tensors(case)
        starts, at = [], 0
        for size, _ in tensors:
            starts.append(at)
            at += -(-size // BLOCK) * BLOCK
        live = torch.zeros(at, dtype=torch.bool, device="cuda")
        owner = torch.empty(at // BLOCK, dtype=torch.int64, device="cuda")
        for t, ((size, _), start) in enumerate(zip(tensors, starts)):
            live[start:start + size] = True
            owner[start // BLOCK:-(-(start + size) // BLOCK)] = t
        s["sizes"], s["starts"] = [size for size, _ in tensors], starts
        s["decays"] = [d for _, d in tensors]
        s["owner"] = owner
        s["decay"] = torch.tensor(s["decays"], device="cuda")[owner]
        s["step"] = 100
        s["rng"] = torch.tensor([seed, 7], dtype=torch.int64, device="cuda")
        s["p"] = rand(at) * 0.02 * live
        s["g"] = (rand(at) * 1e-3 * live).to(DTYPES[case["grad"]])
        s["copy"] = s["p"].to(torch.bfloat16)
        s["amax"] = torch.zeros(len(tensors), device="cuda")
        mean, square = rand(at) * 3e-4 * live, (rand(at) * 1e-3).square() * live
        if case["state"] == "32":
            s["m"], s["v"] = mean, square
        else:
            code, s["m_scale"] = _blocks8(mean, 8)
            s["m"] = code | ((mean < 0).to(torch.uint8) << 7)
            s["v"], s["v_scale"] = _blocks8(square, 16)
    return s


# ----------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------

def _values(codes, scales):
    """The fp32 matrix that codes and block scales stand for (times the encode scale)."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device="cuda")
    pairs = torch.stack((codes & 15, codes >> 4), dim=2).int()
    x = table[pairs].view(codes.shape[0], -1, 16)
    return (x * scales.view(torch.float8_e4m3fn).float()[:, :, None]).view(codes.shape[0], -1)


def _decode_scale(amax):
    enc = (2688.0 / amax).clamp_max(torch.finfo(torch.float32).max)
    return 1.0 / torch.where(amax == 0, torch.ones_like(enc), enc)


def _product(s):
    (a, sfa, amax_a), (b, sfb, amax_b) = s["a"], s["b"]
    return (_values(a, sfa) @ _values(b, sfb).t()) * (_decode_scale(amax_a) * _decode_scale(amax_b))


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


def _plain_gemm(s):
    out = DTYPES[s["out"]]
    z = _product(s)
    if s["bias"]:
        z = z + s["bias_t"]
    d = _act(z, s["act"])
    if s["residual"]:
        d = d + s["residual_t"].float()
    d = d.to(out)
    return {"d": d, "aux": z.to(out) if s["aux"] else None,
            "amax": d.abs().amax().float().reshape(1) if s["amax"] else None}


def _plain_gemm_dact(s):
    wide = _product(s) * _act_slope(s["aux_t"].float(), s["act"])
    d = wide.to(DTYPES[s["out"]])
    return {"d": d, "dbias": wide.sum(0) if s["dbias"] else None,
            "amax": d.abs().amax().float().reshape(1) if s["amax"] else None}


def _plain_layernorm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    y = (d * rstd * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype)
    return {"y": y, "mean": mean.view(-1), "rstd": rstd.view(-1),
            "amax": y.abs().amax().float().reshape(1) if s["amax"] else None}


def _plain_layernorm_backward(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    wdy = dy * s["gamma"].float()
    dx = rstd * (wdy - wdy.mean(1, keepdim=True) - xhat * (wdy * xhat).mean(1, keepdim=True))
    if s["residual"]:
        dx = dx + s["residual_t"].float()
    weight = s["gamma"].dtype
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0).to(weight),
            "dbeta": dy.sum(0).to(weight)}


def _philox(n, rng, step):
    """Philox4x32-10 words (n x 4, int64) of counters (offset + step, 0..n-1) under the seed."""
    mask = 0xFFFFFFFF
    i = torch.arange(n, device="cuda")
    offset = (rng[1] + step).expand(n)
    c0, c1, c2, c3 = offset & mask, (offset >> 32) & mask, i & mask, (i >> 32) & mask
    k0, k1 = rng[0] & mask, (rng[0] >> 32) & mask
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask,
                          ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask)
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack((c0, c1, c2, c3), dim=1)


def _plain_pack8(x, bits16, drop):
    """Stochastic rounding to 8-bit blocks: `drop` of the fraction's 23 bits are cut after
    the 16 random bits were added to their upper part; below 2^-6 steps stay equal."""
    b = x.abs().view(-1, BLOCK)
    top = b.amax(1, keepdim=True).view(torch.int32) >> 23
    scale = torch.where(top == 255, top, (top - 7).clamp_min(1))
    y = b * ((254 - scale).clamp_min(0) << 23).view(torch.float32)
    low = y < 2.0 ** -6
    t = torch.where(low, y + 2.0 ** -6, y).view(torch.int32) + (bits16.view(-1, BLOCK) << (drop - 16))
    code = (t >> drop) - ((120 + low.int()) << (23 - drop))
    return torch.where(scale == 255, torch.zeros_like(code), code), scale.view(-1).to(torch.uint8)


def _plain_unpack8(code, scale, drop):
    code = code.view(-1, BLOCK).int()
    low = code < (1 << (23 - drop))
    t = ((code << drop) + ((120 + low.int()) << 23)).view(torch.float32)
    y = torch.where(low, t - 2.0 ** -6, t)
    return (y * (scale.int() << 23).view(torch.float32)[:, None]).view(-1)


def _plain_adamw(s):
    s["step"] += 1
    step, h, eight = s["step"], ADAM, s["state"] == "8"
    g = s["g"].float()
    if eight:
        m = _plain_unpack8(s["m"] & 127, s["m_scale"], 20)
        m = torch.where(s["m"] >= 128, -m, m)
        v = _plain_unpack8(s["v"], s["v_scale"], 19)
    else:
        m, v = s["m"], s["v"]
    m = m * h["beta1"] + g * (1 - h["beta1"])
    v = v * h["beta2"] + (g * g) * (1 - h["beta2"])
    denominator = torch.sqrt(v) * (1 / math.sqrt(1 - h["beta2"] ** step)) + h["eps"]
    p = s["p"].view(-1, BLOCK)
    p = p * (1 - h["lr"] * s["decay"])[:, None]
    p = p.view(-1) - (m / denominator) * (h["lr"] / (1 - h["beta1"] ** step))
    s["p"].copy_(p)
    s["copy"].copy_(p)
    top = s["copy"].abs().view(-1, BLOCK).amax(1).float()
    s["amax"].zero_().scatter_reduce_(0, s["owner"], top, "amax")
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": s["p"], "copy": s["copy"], "amax": s["amax"], "m": s["m"], "v": s["v"]}
    words = _philox(m.numel() // 4, s["rng"], step).view(-1)
    code, scale = _plain_pack8(m, (words & 0xFFFF).int(), 20)
    s["m"].copy_(code.view(-1) | ((m < 0).int() << 7))
    s["m_scale"].copy_(scale)
    code, scale = _plain_pack8(v, (words >> 16).int(), 19)
    # a second moment above zero never becomes zero
    code = torch.where((v.view(-1, BLOCK) > 0) & (scale[:, None] != 255), code.clamp_min(1), code)
    s["v"].copy_(code.view(-1))
    s["v_scale"].copy_(scale)
    m = _plain_unpack8(s["m"] & 127, s["m_scale"], 20)
    return {"p": s["p"], "copy": s["copy"], "amax": s["amax"],
            "m": torch.where(s["m"] >= 128, -m, m).to(torch.bfloat16),
            "v": _plain_unpack8(s["v"], s["v_scale"], 19).to(torch.bfloat16)}


# ----------------------------------------------------------------------------
# The framework's calls
# ----------------------------------------------------------------------------

def _own_gemm(nv, s):
    amax = torch.empty(1, device="cuda") if s["amax"] else None
    d, aux = nv.matmul_nvfp4(*s["a"], *s["b"], bias=s["bias_t"], residual=s["residual_t"],
                             activation=s["act"], out_dtype=DTYPES[s["out"]],
                             with_aux=s["aux"], amax_out=amax)
    return {"d": d, "aux": aux, "amax": amax}


def _own_gemm_dact(nv, s):
    amax = torch.empty(1, device="cuda") if s["amax"] else None
    d, dbias = nv.matmul_nvfp4_dact(*s["a"], *s["b"], s["aux_t"], activation=s["act"],
                                    with_dbias=s["dbias"], amax_out=amax)
    return {"d": d, "dbias": dbias, "amax": amax}


def _own_layernorm(nv, s):
    amax = torch.empty(1, device="cuda") if s["amax"] else None
    y, mean, rstd = nv.layernorm(s["x"], s["gamma"], s["beta"], EPS, amax_out=amax)
    return {"y": y, "mean": mean, "rstd": rstd, "amax": amax}


def _own_layernorm_backward(nv, s):
    dx, dgamma, dbeta = nv.layernorm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"],
                                              residual=s["residual_t"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _own_adamw(nv, s):
    s["step"] += 1
    eight = s["state"] == "8"
    if "optimizer" not in s:
        # views of the flat buffers, one for each tensor: a user's program makes them once
        def cut(x, unit=1):
            return [x[a // unit:-(-(a + n) // unit)] for a, n in zip(s["starts"], s["sizes"])]
        s["optimizer"] = nv.AdamW(
            cut(s["p"]), cut(s["g"]), cut(s["m"]), cut(s["v"]),
            exp_avg_scales=cut(s["m_scale"], BLOCK) if eight else None,
            exp_avg_sq_scales=cut(s["v_scale"], BLOCK) if eight else None,
            copies=cut(s["copy"]), weight_decays=s["decays"], offsets=s["starts"],
            amax_out=s["amax"], rng_state=s["rng"])
    s["optimizer"].step(s["step"], lr=ADAM["lr"], beta1=ADAM["beta1"], beta2=ADAM["beta2"],
                        eps=ADAM["eps"])
    out = {"p": s["p"], "copy": s["copy"], "amax": s["amax"]}
    if not eight:
        return {**out, "m": s["m"], "v": s["v"]}
    return {**out, "m": nv.adamw_unpack_state(s["m"], s["m_scale"], "exp_avg"),
            "v": nv.adamw_unpack_state(s["v"], s["v_scale"], "exp_avg_sq")}


def run(state):
    op = state["op"]
    if own:
        import fp4_sm120a_b200 as nv
        return {"gemm": _own_gemm, "gemm_dact": _own_gemm_dact, "layernorm": _own_layernorm,
                "layernorm_backward": _own_layernorm_backward, "adamw": _own_adamw}[op](nv, state)
    return {"gemm": _plain_gemm, "gemm_dact": _plain_gemm_dact, "layernorm": _plain_layernorm,
            "layernorm_backward": _plain_layernorm_backward, "adamw": _plain_adamw}[op](state)


# ----------------------------------------------------------------------------
# The definition in 64 bits
# ----------------------------------------------------------------------------

def _exact_operand(operand):
    codes, scales, amax = operand
    mag = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    rows, half = codes.shape
    x = torch.empty(rows, 2 * half, dtype=torch.float64, device="cuda")
    for odd in (0, 1):
        c = (codes >> (4 * odd)) & 15
        x[:, odd::2] = mag[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).double())
    scale = scales.view(torch.float8_e4m3fn).double()
    x *= scale.repeat_interleave(16, dim=1)
    top = float(amax)
    return x * (top / 2688.0 if top else 1.0)


def _exact_gemm(s):
    z = _exact_operand(s["a"]) @ _exact_operand(s["b"]).t()
    if s["op"] == "gemm":
        if s["bias"]:
            z += s["bias_t"].double()
        act = s["act"]
        if act == "relu":
            d = torch.maximum(z, torch.zeros_like(z))
        elif act == "gelu":
            d = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))
        elif act == "silu":
            d = z * torch.sigmoid(z)
        else:
            d = z
        if s["residual"]:
            d = d + s["residual_t"].double()
        # the amax is that of the rounded product: no value of its own in 64 bits
        return {"d": d, "aux": z if s["aux"] else None, "amax": None}
    x, act = s["aux_t"].double(), s["act"]
    if act == "relu":
        slope = torch.where(x > 0, 1.0, 0.0).double()
    elif act == "gelu":
        c = math.sqrt(8 / math.pi)
        q = torch.sigmoid(c * (x + 0.044715 * x ** 3))
        slope = q + x * q * (1 - q) * c * (1 + 0.134145 * x ** 2)
    elif act == "silu":
        q = torch.sigmoid(x)
        slope = q + x * q * (1 - q)
    else:
        slope = torch.ones_like(x)
    d = z * slope
    return {"d": d, "dbias": d.sum(0) if s["dbias"] else None, "amax": None}


def _exact_layernorm(s):
    x = s["x"].double()
    mean, var = x.mean(1), x.var(1, unbiased=False)
    rstd = (var + EPS) ** -0.5
    y = (x - mean[:, None]) * rstd[:, None] * s["gamma"].double() + s["beta"].double()
    return {"y": y, "mean": mean, "rstd": rstd, "amax": None}


def _exact_layernorm_backward(s):
    x, dy, r = s["x"].double(), s["dy"].double(), s["rstd"].double()[:, None]
    h = (x - s["mean"].double()[:, None]) * r
    u = dy * s["gamma"].double()
    n = x.shape[1]
    dx = (u - u.sum(1, keepdim=True) / n - h * ((u * h).sum(1, keepdim=True) / n)) * r
    if s["residual"]:
        dx += s["residual_t"].double()
    return {"dx": dx, "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0)}


def _exact_adamw(s):
    t, h = s["step"] + 1, ADAM
    g = s["g"].double()
    if s["state"] == "32":
        m, v = s["m"].double(), s["v"].double()
    else:
        def decode(code, scale, steps):
            e, f = code // steps, (code % steps).double()
            y = torch.where(e == 0, f / steps * 2.0 ** -6, (1 + f / steps) * 2.0 ** (e.double() - 7))
            return y * (2.0 ** (scale.double() - 127)).repeat_interleave(BLOCK)
        m = decode(s["m"] % 128, s["m_scale"], 8) * (1 - 2.0 * (s["m"] // 128).double())
        v = decode(s["v"], s["v_scale"], 16)
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g ** 2
    p = s["p"].double()
    for start, size, decay in zip(s["starts"], s["sizes"], s["decays"]):
        p[start:start + size] *= 1 - h["lr"] * decay
    p -= h["lr"] * (m / (1 - h["beta1"] ** t)) / ((v / (1 - h["beta2"] ** t)).sqrt() + h["eps"])
    whole = s["state"] == "32"  # rounded states have no value of their own in 64 bits
    return {"p": p, "copy": p, "amax": None, "m": m if whole else None, "v": v if whole else None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gemm": _exact_gemm, "gemm_dact": _exact_gemm, "layernorm": _exact_layernorm,
            "layernorm_backward": _exact_layernorm_backward, "adamw": _exact_adamw}[s["op"]](s)
