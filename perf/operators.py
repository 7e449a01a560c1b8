"""Cases of the feature operators: a linear layer with bias, activation and
residual in its epilogue, and a group norm with an activation over
channel-last tensors, each forward and as a training step.

They are what decodes the feature channels that the rasterisers blend (rendered
channel-last, one row per pixel) or that the Gaussians carry (one row per
Gaussian).  Formulas, for rows x (M, K), W (N, K), b (N), r (M, N):

    linear:      y = act(x W^T + b) + r
    group norm:  y = act((x - mean_g) rstd_g w + b), mean and biased variance
                 over the positions of a sample and the channels of a group

and their gradients for an upstream dy.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5

# the largest listed pass of each operator bounds what is drawn
MOST_FLOPS = 131072 * 512 * 512
MOST_VALUES = 1600 * 1200 * 128


def linear_case(name, rows, k, n, dtype, act, *, bias=True, residual=False, train=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype,
            "act": act, "bias": bias, "residual": residual, "train": train}


def norm_case(name, views, height, width, channels, groups, dtype, act, *, train=False):
    return {"name": name, "op": "group_norm", "views": views, "height": height, "width": width,
            "channels": channels, "groups": groups, "dtype": dtype, "act": act, "train": train}


def listed():
    return [
        # a colour read for one picked pixel: latency only
        linear_case("linear one row", 1, 32, 3, "fp32", "sigmoid"),
        # a 256x256 render of RGB and 32 features into a first hidden layer
        linear_case("linear small image", 256 * 256, 35, 64, "fp32", "relu"),
        # the 32 features of a 1600x1200 render, widened
        linear_case("linear image", 1600 * 1200, 32, 64, "bf16", "silu"),
        # a residual layer at the same size
        linear_case("linear image residual", 1600 * 1200, 64, 64, "bf16", "silu", residual=True),
        # a head over the features of a million Gaussians, trained in fp32
        linear_case("linear gaussians train", 1000000, 35, 32, "fp32", "gelu", train=True),
        # the residual layer of a decoder in training
        linear_case("linear image residual train", 1600 * 1200, 64, 64, "bf16", "silu",
                    residual=True, train=True),
        # wide features: the products themselves count
        linear_case("linear wide train", 131072, 512, 512, "fp16", "gelu", train=True),
        # a small crop with odd sizes
        norm_case("norm crop", 1, 37, 53, 35, 5, "fp32", "none"),
        # a batch of eight views at 1296x840
        norm_case("norm views", 8, 840, 1296, 32, 8, "bf16", "silu"),
        # one 1920x1080 image in fp32
        norm_case("norm image", 1, 1080, 1920, 64, 16, "fp32", "silu"),
        # two crops in training
        norm_case("norm crops train", 2, 67, 101, 48, 4, "fp32", "gelu", train=True),
        # a 1600x1200 image in training
        norm_case("norm image train", 1, 1200, 1600, 64, 8, "bf16", "silu", train=True),
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    act = rng.choice(["none", "relu", "silu", "gelu", "sigmoid"])
    # relu's slope jumps: among 10^7 values one lies within an fp32 rounding of the border
    # and goes either way, so fp32 training is drawn with the smooth activations
    train = rng.random() < 0.5 and not (act == "relu" and dtype == "fp32")
    most = MOST_VALUES // (2 if dtype == "fp32" else 1)
    if rng.random() < 0.5:
        k, n = _spread(rng, 3, 512), _spread(rng, 3, 512)
        if rng.random() < 0.5:
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        rows = _spread(rng, 1, 1920 * 1080)
        rows = max(1, min(rows, most // (k + n), MOST_FLOPS // (k * n)))
        return {"op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act,
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.4, "train": train}
    groups = rng.choice([1, 2, 4, 5, 8, 16, 32])
    channels = groups * max(1, round(_spread(rng, 8, 256) / groups))
    views = rng.choice([1, 1, 2, 3, 8])
    height = _spread(rng, 4, 1200)
    width = max(1, round(height * rng.uniform(0.7, 1.8)))
    height = max(1, min(height, most // 2 // (views * width * channels)))
    return {"op": "group_norm", "views": views, "height": height, "width": width,
            "channels": channels, "groups": groups, "dtype": dtype, "act": act, "train": train}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = normal(rows, k)
        s["weight"] = normal(n, k, scale=1 / math.sqrt(k))
        s["bias"] = normal(n, scale=0.2) if case["bias"] else None
        s["residual"] = normal(rows, n) if case["residual"] else None
        s["upstream"] = normal(rows, n) if case["train"] else None
    else:
        shape = (case["views"], case["height"], case["width"], case["channels"])
        # blended features: each channel with a mean of its own
        means = torch.randn(shape[-1], generator=g, device="cuda")
        s["x"] = (torch.randn(shape, generator=g, device="cuda") * 1.5 + means).to(dtype)
        s["weight"] = normal(shape[-1], scale=0.2, shift=1.0)
        s["bias"] = normal(shape[-1], scale=0.2)
        s["upstream"] = normal(*shape) if case["train"] else None
    return s


def activate(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return z


def slope(z, act):
    """d activate / dz."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    if act == "gelu":
        density = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * density
    if act == "sigmoid":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 - sig)
    return torch.ones_like(z)


def plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = activate(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dz = s["upstream"].float() * slope(z, case["act"])
        out["dx"] = (dz @ w).to(dtype)
        out["dweight"] = (dz.t() @ x).to(dtype)
        if s["bias"] is not None:
            out["dbias"] = dz.sum(0).to(dtype)
        if s["residual"] is not None:
            out["dresidual"] = s["upstream"]
    return out


def plain_norm(s):
    case, dtype, shape = s["case"], s["x"].dtype, s["x"].shape
    groups, channels = case["groups"], case["channels"]
    x = s["x"].float().reshape(shape[0], -1, groups, channels // groups)
    w, b = (s[name].float().reshape(groups, -1) for name in ("weight", "bias"))
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + EPS)
    hat = (x - mean) * rstd
    u = hat * w + b
    out = {"y": activate(u, case["act"]).to(dtype).reshape(shape)}
    if case["train"]:
        du = s["upstream"].float().reshape(u.shape) * slope(u, case["act"])
        dhat = du * w
        dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True)
                     - hat * (dhat * hat).mean((1, 3), keepdim=True))
        out["dx"] = dx.to(dtype).reshape(shape)
        out["dweight"] = (du * hat).sum((0, 1)).to(dtype).reshape(-1)
        out["dbias"] = du.sum((0, 1)).to(dtype).reshape(-1)
    return out


def own_linear(s):
    from dsl_splat_b200 import features

    case = s["case"]
    if not case["train"]:
        return {"y": features.linear(s["x"], s["weight"], s["bias"], residual=s["residual"],
                                     activation=case["act"])}
    names = [m for m in ("x", "weight", "bias", "residual") if s[m] is not None]
    leaves = {m: s[m].detach().requires_grad_() for m in names}
    y = features.linear(leaves["x"], leaves["weight"], leaves.get("bias"),
                        residual=leaves.get("residual"), activation=case["act"])
    grads = torch.autograd.grad(y, [leaves[m] for m in names], s["upstream"])
    return {"y": y.detach(), **{"d" + m: v for m, v in zip(names, grads)}}


def own_norm(s):
    from dsl_splat_b200 import features

    case = s["case"]
    if not case["train"]:
        return {"y": features.group_norm(s["x"], case["groups"], s["weight"], s["bias"],
                                         eps=EPS, activation=case["act"])}
    names = ("x", "weight", "bias")
    leaves = [s[m].detach().requires_grad_() for m in names]
    y = features.group_norm(leaves[0], case["groups"], leaves[1], leaves[2], eps=EPS,
                            activation=case["act"])
    grads = torch.autograd.grad(y, leaves, s["upstream"])
    return {"y": y.detach(), **{"d" + m: v for m, v in zip(names, grads)}}


def run(state):
    linear = state["case"]["op"] == "linear"
    if own:
        return own_linear(state) if linear else own_norm(state)
    return plain_linear(state) if linear else plain_norm(state)


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        values = rows * (k + n) + n * k + n * case["bias"] + rows * n * case["residual"]
        if case["train"]:
            values += rows * (k + n) + n * k + n * case["bias"]
        return {"bytes": size * values, "flops": 2 * rows * n * k * (3 if case["train"] else 1)}
    values = case["views"] * case["height"] * case["width"] * case["channels"]
    passes = 4 if case["train"] else 2
    return {"bytes": size * (passes * values + passes * case["channels"]),
            "flops": (24 if case["train"] else 8) * values}


def exact(case, seed):
    """The definition in 64 bits, written with sums over einsum indices."""
    s = prepare(case, seed)
    wide = {m: None if s[m] is None else s[m].double() for m in s if m != "case"}
    x, w, b, dy = wide["x"], wide["weight"], wide["bias"], wide["upstream"]
    act = case["act"]

    def value_and_slope(z):
        if act == "none":
            return z, torch.ones_like(z)
        if act == "relu":
            return z.clamp(min=0), torch.heaviside(z, torch.zeros_like(z))
        if act == "gelu":
            upper = 0.5 * torch.special.erfc(-z / math.sqrt(2))
            return z * upper, upper + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        sig = torch.special.expit(z)
        if act == "sigmoid":
            return sig, sig * torch.special.expit(-z)
        return z * sig, sig + z * sig * torch.special.expit(-z)

    if case["op"] == "linear":
        z = torch.einsum("mk,nk->mn", x, w)
        value, rate = value_and_slope(z if b is None else z + b[None])
        out = {"y": value if wide["residual"] is None else value + wide["residual"]}
        if case["train"]:
            dz = dy * rate
            out["dx"] = torch.einsum("mn,nk->mk", dz, w)
            out["dweight"] = torch.einsum("mn,mk->nk", dz, x)
            if b is not None:
                out["dbias"] = torch.einsum("mn->n", dz)
            if wide["residual"] is not None:
                out["dresidual"] = dy
        return out
    shape, groups = x.shape, case["groups"]
    # one row per sample and group
    split = (shape[0], shape[1] * shape[2], groups, shape[3] // groups)

    def gather(v):
        return v.reshape(split).permute(0, 2, 1, 3).reshape(shape[0] * groups, -1)

    def scatter(v):
        return (v.reshape(split[0], split[2], split[1], split[3]).permute(0, 2, 1, 3)
                .reshape(shape))

    rows = gather(x)
    var, mean = torch.var_mean(rows, dim=1, correction=0, keepdim=True)
    deviation = (var + EPS).sqrt()
    hat = scatter((rows - mean) / deviation)
    value, rate = value_and_slope(hat * w + b)
    out = {"y": value}
    if case["train"]:
        du = dy * rate
        upstream, normal = gather(du * w), gather(hat)
        along = (upstream * normal).mean(1, keepdim=True)
        out["dx"] = scatter((upstream - upstream.mean(1, keepdim=True) - normal * along)
                            / deviation)
        out["dweight"] = torch.einsum("bhwc,bhwc->c", du, hat)
        out["dbias"] = torch.einsum("bhwc->c", du)
    return out
