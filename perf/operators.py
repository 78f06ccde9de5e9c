"""Timed cases of the trained-block operators: linear layer with its epilogue, layer norm, global gradient norm with clipping.

With `own` false `run` computes an operator in its plain form (elementary torch operations in 32 bits, one rounding at
the end); with `own` true it makes the calls that a user makes: `modules.linear`, `modules.layer_norm` (their backward
passes through autograd) and `training.clip_grad_norm_`.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def _linear(name, rows, width_in, width_out, dtype, activation, bias, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "in": width_in, "out": width_out, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual, "train": train}


def _norm(name, rows, width, dtype, affine_dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "affine_dtype": affine_dtype,
            "train": train}


def _clip(name, layout, width, layers, dtype, out, clipped, norm):
    return {"name": name, "op": "clip", "layout": layout, "width": width, "layers": layers, "dtype": dtype, "out": out,
            "clipped": clipped, "norm": norm, "seed": 0}


def listed():
    return [
        # one token through a block's widening layer while answering: the weight has to be read, latency counts
        _linear("linear_token_bf16", 1, 2048, 8192, "bfloat16", "gelu", True, False, False),
        # a few ragged prompts in half precision, no size a multiple of a tile
        _linear("linear_ragged_fp16", 77, 1000, 1531, "float16", "silu", True, True, False),
        # a long prompt (or many images' pixels) through the widening layer: the largest product
        _linear("linear_prompt_bf16", 8192, 2048, 8192, "bfloat16", "gelu", True, False, False),
        # training step of the widening layer
        _linear("linear_train_bf16", 4096, 1024, 4096, "bfloat16", "gelu", True, False, True),
        # training step of the narrowing layer that closes a residual block; an odd number of tokens
        _linear("linear_train_residual_bf16", 4001, 4096, 1024, "bfloat16", "none", True, True, True),
        # 1x1 layer over the pixels of four 64x64 images in the training path's own type
        _linear("linear_train_fp32", 16384, 256, 1024, "float32", "silu", True, False, True),
        # one token
        _norm("layer_norm_token_bf16", 1, 2048, "bfloat16", "bfloat16", False),
        # training step on a long batch with a wide model, scale and shift kept in 32 bits
        _norm("layer_norm_train_bf16", 16384, 4096, "bfloat16", "float32", True),
        # channels of the 64x64 level of sixteen images: very many short rows, the training path's own type
        _norm("layer_norm_train_fp32", 65536, 128, "float32", "float32", True),
        # odd rows and an odd width: no row starts on a 16-byte boundary
        _norm("layer_norm_train_ragged_fp16", 1237, 1111, "float16", "float16", True),
        # the default network's gradients (hundreds of tensors, most of them tiny) on a step that needs no clipping
        _clip("clip_unet_fp32", "unet", 32, 4, "float32", "in_place", False, "2"),
        # eight wide blocks' gradients in bfloat16, clipped into the optimiser's 32-bit buffers
        _clip("clip_blocks_bf16", "blocks", 2048, 8, "bfloat16", "float32", True, "2"),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]; every second one is odd or ragged as it falls."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 32 * 32
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "layer_norm", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "linear":
        train = rng.random() < 0.5
        rows, a, b = _spread(rng, 16 if train else 1, 8192), _spread(rng, 32, 8192), _spread(rng, 32, 8192)
        most = 2.7e11 / ((3 if train else 1) * (4 if dtype == "float32" else 1))
        rows = max(1, min(rows, int(most / (2.0 * a * b))))
        case = _linear("", rows, a, b, dtype, rng.choice(["none", "relu", "silu", "gelu"]), rng.random() < 0.7,
                       rng.random() < 0.4, train)
    elif op == "layer_norm":
        train = rng.random() < 0.7
        width = _spread(rng, 8, 16384)
        rows = min(_spread(rng, 1, 65536), 67108864 // width)
        case = _norm("", rows, width, dtype, rng.choice([dtype, "float32"]), train)
    else:
        layout = rng.choice(["unet", "blocks", "mixed"])
        out = rng.choice(["in_place", "same", "float32"])
        clipped = out != "in_place" and rng.random() < 0.5
        width, layers = {"unet": (rng.choice([16, 32, 64]), rng.randint(2, 4)), "blocks": (_spread(rng, 64, 1024), rng.randint(1, 12)),
                         "mixed": (_spread(rng, 100, 30000), rng.randint(1, 400))}[layout]
        case = _clip("", layout, width, layers, dtype, out, clipped, rng.choice(["2", "2", "inf"]))
        case["seed"] = rng.randrange(1 << 30)
    del case["name"]
    return case


def _unet_shapes(dim, levels):
    """Parameter shapes of the denoising network of base width `dim` with `levels` resolutions (widths dim * 1, 2, 4, ...)."""
    time = 4 * dim
    widths = [dim] + [dim << i for i in range(levels)]

    def conv(cin, cout, k, bias=True):
        return [(cout, cin, k, k)] + ([(cout,)] if bias else [])

    def block(cin, cout, embedded=True):
        return (([(cout, time), (cout,)] if embedded else []) + conv(cin, cout, 3) + [(cout,), (cout,)] + conv(cout, cout, 3)
                + [(cout,), (cout,)] + (conv(cin, cout, 1) if cin != cout else []))

    def attention(c, linear):
        return conv(c, 384, 1, False) + conv(128, c, 1) + ([(c,), (c,)] if linear else []) + [(c,), (c,)]

    shapes = conv(3, dim, 7) + [(time, dim), (time,), (time, time), (time,)]
    pairs = list(zip(widths[:-1], widths[1:]))
    for i, (a, b) in enumerate(pairs):
        shapes += block(a, b) + block(b, b) + attention(b, True) + (conv(b, b, 4) if i + 1 < len(pairs) else [])
    top = widths[-1]
    shapes += block(top, top) + attention(top, False) + block(top, top)
    for a, b in reversed(pairs[1:]):
        shapes += block(2 * b, a) + block(a, a) + attention(a, True) + conv(a, a, 4)
    return shapes + block(dim, dim, False) + [(dim,), (dim,)] + conv(dim, 3, 1)


def _gradient_shapes(case):
    w, n = case["width"], case["layers"]
    if case["layout"] == "unet":
        return _unet_shapes(w, n)
    if case["layout"] == "blocks":
        layer = [(w,), (w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
        return layer * n
    state, shapes = case["seed"] + 1, []
    for _ in range(n):   # sizes from one element up to about twice the width, none of them round
        state = (state * 6364136223846793005 + 1442695040888963407) % (1 << 64)
        shapes.append((1 + (state >> 33) % (2 * w),))
    return shapes + [(1001,)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(shape, generator=g, device=dev) * scale + shift).to(to)

    if case["op"] == "linear":
        m, k, n, train = case["rows"], case["in"], case["out"], case["train"]
        s = {"x": normal((m, k)), "weight": normal((n, k), k ** -0.5), "bias": normal((n,), 0.1) if case["bias"] else None,
             "residual": normal((m, n)) if case["residual"] else None, "activation": case["activation"], "train": train}
        if train:
            # as it comes back from the layers behind: small in the wide types, scaled up in half precision
            s["dy"] = normal((m, n), 0.5 if dtype == torch.float16 else 2e-3)
    elif case["op"] == "layer_norm":
        m, d, train = case["rows"], case["width"], case["train"]
        # a residual stream: an offset and a few channels far larger than the rest
        x = torch.randn((m, d), generator=g, device=dev) * 1.5 + 0.3
        x[:, ::97] *= 8
        a = DTYPES[case["affine_dtype"]]
        s = {"x": x.to(dtype), "weight": normal((d,), 0.1, 1.0, a), "bias": normal((d,), 0.1, 0.0, a), "train": train}
        if train:
            s["dy"] = normal((m, d), 0.5 if dtype == torch.float16 else 2e-3)
    else:
        shapes = _gradient_shapes(case)
        # the gradients that one backward pass hands out are views of one buffer: on 64-element steps, or packed tightly
        step = 1 if case["layout"] == "mixed" else 64
        starts, end = [], 0
        for shape in shapes:
            starts.append(end)
            end += -(-math.prod(shape) // step) * step
        flat, params = torch.zeros(end, dtype=dtype, device=dev), []
        for i, (shape, at) in enumerate(zip(shapes, starts)):
            p = torch.nn.Parameter(torch.empty(shape, dtype=dtype, device=dev))
            p.grad = flat[at:at + math.prod(shape)].view(shape)
            p.grad.copy_(normal(shape, 0.02 if i % 3 else 0.05))
            params.append(p)
        total = math.sqrt(sum(math.prod(sh) * (0.02 if i % 3 else 0.05) ** 2 for i, sh in enumerate(shapes)))
        biggest = 0.1 if case["norm"] == "inf" else total
        s = {"params": params, "max_norm": biggest * (0.3 if case["clipped"] else 4.0), "norm": case["norm"], "source": flat, "flat": flat, "out": None}
        if case["out"] != "in_place":   # the optimiser's own buffer of the same layout
            s["flat"] = torch.zeros(end, dtype=torch.float32 if case["out"] == "float32" else dtype, device=dev)
            s["out"] = [s["flat"][at:at + math.prod(shape)].view(shape) for shape, at in zip(shapes, starts)]
    s["op"] = case["op"]
    if s.get("train"):
        for key in ("x", "weight", "bias", "residual"):
            if s.get(key) is not None:
                s[key].requires_grad_(True)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _activate(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return z * 0.5 * torch.erfc(z * -math.sqrt(0.5))
    return z


def _slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _plain_linear(s):
    x, w, b, r = s["x"].detach().float(), s["weight"].detach().float(), s["bias"], s["residual"]
    to = s["x"].dtype
    z = x @ w.t()
    if b is not None:
        z = z + b.detach().float()
    y = _activate(z, s["activation"])
    if r is not None:
        y = y + r.detach().float()
    if not s["train"]:
        return {"y": y.to(to)}
    dy = s["dy"].float()
    dz = dy * _slope(z, s["activation"]) if s["activation"] != "none" else dy
    out = {"y": y.to(to), "dx": (dz @ w).to(to), "dweight": (dz.t() @ x).to(to)}
    if b is not None:
        out["dbias"] = dz.sum(0).to(to)
    if r is not None:
        out["dresidual"] = s["dy"]
    return out


def _plain_layer_norm(s):
    x, w, b, to = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float(), s["x"].dtype
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    xhat = (x - mean) * rstd
    y = xhat * w + b
    if not s["train"]:
        return {"y": y.to(to)}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return {"y": y.to(to), "dx": dx.to(to), "dweight": (dy * xhat).sum(0).to(s["weight"].dtype),
            "dbias": dy.sum(0).to(s["bias"].dtype)}


def _plain_clip(s):
    grads = [p.grad for p in s["params"]]
    if s["norm"] == "inf":
        norm = torch.stack([g.float().abs().max() for g in grads]).max()
    else:
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    scale = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    to = grads if s["out"] is None else s["out"]
    [o.copy_(g.float() * scale) for o, g in zip(to, grads)]
    return {"norm": norm, "grads": s["flat"]}


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _own_linear(s):
    from diffusion_model_nemo_amd.modules import linear
    activation = None if s["activation"] == "none" else s["activation"]
    if not s["train"]:
        with torch.no_grad():
            return {"y": linear(s["x"], s["weight"], s["bias"], activation=activation, residual=s["residual"])}
    y = linear(s["x"], s["weight"], s["bias"], activation=activation, residual=s["residual"])
    names = [k for k in ("x", "weight", "bias", "residual") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def _own_layer_norm(s):
    from diffusion_model_nemo_amd.modules import layer_norm
    if not s["train"]:
        with torch.no_grad():
            return {"y": layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)}
    y = layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
    dx, dw, db = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _own_clip(s):
    from diffusion_model_nemo_amd.training import clip_grad_norm_
    norm = clip_grad_norm_(s["params"], s["max_norm"], norm_type=float(s["norm"]), out=s["out"])
    return {"norm": norm, "grads": s["flat"]}


def run(state):
    if own:
        return {"linear": _own_linear, "layer_norm": _own_layer_norm, "clip": _own_clip}[state["op"]](state)
    return {"linear": _plain_linear, "layer_norm": _plain_layer_norm, "clip": _plain_clip}[state["op"]](state)


# ---- what a pass cannot do without, and the answers in 64 bits -----------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        b, r, train = n * case["bias"], m * n * case["residual"], case["train"]
        moved = m * k + n * k + b + r + m * n            # x, weight, bias, residual in; y out
        if train:
            moved += m * n + m * k + n * k + b           # dy in; dx, dweight, dbias out
        return {"bytes": moved * e, "flops": 2 * m * k * n * (3 if train else 1)}
    if case["op"] == "layer_norm":
        m, d, a, train = case["rows"], case["width"], BYTES[case["affine_dtype"]], case["train"]
        return {"bytes": (4 if train else 2) * m * d * e + (4 if train else 2) * d * a, "flops": (20 if train else 8) * m * d}
    total = sum(math.prod(s) for s in _gradient_shapes(case))
    out = {"in_place": 0, "same": e, "float32": 4}[case["out"]]
    return {"bytes": total * (e + out), "flops": total * (3 if out else 2)}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda t: t.detach().to(torch.float64)  # noqa: E731
    if case["op"] == "linear":
        x, w = f64(s["x"]), f64(s["weight"])
        z = torch.zeros((case["rows"], case["out"]), dtype=torch.float64, device=x.device)
        if s["bias"] is not None:
            z += f64(s["bias"])
        z.addmm_(x, w.transpose(0, 1).contiguous())
        kind = s["activation"]
        if kind == "gelu":
            # the normal distribution's lower tail through the scaled complementary error function: no cancellation
            tail = 0.5 * torch.exp(-0.5 * z * z) * torch.special.erfcx(z.abs() / math.sqrt(2.0))
            cdf = torch.where(z < 0, tail, 1.0 - tail)
            y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        elif kind == "silu":
            sig = torch.sigmoid(z)
            y, slope = z * sig, sig + z * sig * (1.0 - sig)
        elif kind == "relu":
            y, slope = z.clamp(min=0.0), torch.heaviside(z, torch.zeros((), dtype=torch.float64, device=z.device))
        else:
            y, slope = z.clone(), None
        if s["residual"] is not None:
            y += f64(s["residual"])
        if not s["train"]:
            return {"y": y}
        dz = f64(s["dy"]) if slope is None else slope.mul_(f64(s["dy"]))
        out = {"y": y, "dx": torch.mm(dz, w), "dweight": torch.mm(dz.transpose(0, 1).contiguous(), x)}
        if s["bias"] is not None:
            out["dbias"] = torch.mv(dz.transpose(0, 1), torch.ones(case["rows"], dtype=torch.float64, device=x.device))
        if s["residual"] is not None:
            out["dresidual"] = f64(s["dy"])
        return out
    if case["op"] == "layer_norm":
        x, w, b = f64(s["x"]).requires_grad_(True), f64(s["weight"]).requires_grad_(True), f64(s["bias"]).requires_grad_(True)
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = torch.addcmul(b, (x - mean) * torch.rsqrt(var + 1e-5), w)
        if not s["train"]:
            return {"y": y.detach()}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), f64(s["dy"]))
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    grads = [f64(p.grad) for p in s["params"]]
    if case["norm"] == "inf":
        norm = torch.stack([torch.linalg.vector_norm(g, math.inf) for g in grads]).max()
    else:
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in grads]))
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "grads": f64(s["source"]).mul_(factor)}
