"""Cases of the operators that train features and scenes: layer norm over
channel-last rows, a codebook's lookup and its gradient, the softmax cross entropy
of a linear head over a vocabulary, and AdamW over a scene's tensors.

    layer norm:     y = act((x - mean) rstd w + b), mean and biased variance of a row
    embedding:      y_i = s T[id_i];  dT[v] = s sum of dy_i over id_i = v
    cross entropy:  z = x W^T + b, l_i = log sum_j exp z_ij - z_i,t_i, summed, averaged over
                    the rows that count or kept apart; the rows whose target is the ignored
                    index have no loss and no gradient;
                    dz_ij = u_i (exp(z_ij - lse_i) - [j = t_i]), dx = dz W, dW = dz^T x,
                    db = sum_i dz_i
    AdamW:          m' = b1 m + (1 - b1) g, v' = b2 v + (1 - b2) g^2,
                    p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)

States in 8 bits: the runs of 256 values of a flattened tensor have an exponent E
each, from their largest magnitude.  m is held as a sign, 4 bits of exponent and 3 of
mantissa; of v the root is held, without a sign, with 4 and 4.  A code c of M mantissa
bits stands for 2^E (1 + (c mod 2^M) / 2^M) 2^(c div 2^M - 15), or, below 2^M, for
2^E c 2^(-14 - M).  E is the least exponent in [-126, 127] whose largest code reaches the
run's largest magnitude.  Values are rounded down after a dither below one step has been
added, a hash of the value's place and the step, so that the moving averages move by less
than a step on average; a root that is not zero has a code that is not zero.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-5
IGNORED = -100
BETAS = (0.9, 0.999)
RUN = 256

# the largest listed pass of each operator bounds what is drawn
MOST_VALUES = 1600 * 1200 * 64
MOST_LOOKED_UP = 1000000 * 64
MOST_PRODUCTS = 65536 * 512 * 32768
MOST_PARAMETERS = 1000000 * 59


def norm_case(name, rows, channels, dtype, act, *, train=False):
    return {"name": name, "op": "layer_norm", "rows": rows, "channels": channels, "dtype": dtype,
            "act": act, "train": train}


def embedding_case(name, ids, entries, channels, dtype, scale, *, train):
    return {"name": name, "op": "embedding", "ids": ids, "entries": entries,
            "channels": channels, "dtype": dtype, "scale": scale, "train": train}


def entropy_case(name, rows, k, vocabulary, dtype, reduction, *, bias=False, train=True,
                 ignored=0.1):
    return {"name": name, "op": "cross_entropy", "rows": rows, "k": k, "vocabulary": vocabulary,
            "dtype": dtype, "reduction": reduction, "bias": bias, "train": train,
            "ignored": ignored}


def adamw_case(name, kind, count, dtype, bits, decay, step):
    """kind: "scene" of `count` Gaussians, or "decoder" of layers `count` wide."""
    return {"name": name, "op": "adamw", "kind": kind, "count": count, "dtype": dtype,
            "bits": bits, "decay": decay, "step": step}


def listed():
    return [
        # a small crop of a rendered feature image: latency
        norm_case("layer norm crop", 37 * 53, 48, "fp32", "none"),
        # the 64 features of a 1600x1200 render
        norm_case("layer norm image", 1600 * 1200, 64, "bf16", "silu"),
        # the features of a million Gaussians, trained in fp32, of an odd width
        norm_case("layer norm gaussians train", 1000000, 35, "fp32", "gelu", train=True),
        # the appearance codes of a batch's eight views: latency
        embedding_case("embedding views train", 8, 300, 32, "fp32", 1.0, train=True),
        # a million Gaussians that share a codebook of features
        embedding_case("embedding gaussians train", 1000000, 8192, 64, "bf16", 0.125, train=True),
        # a few thousand labelled pixels, each with its own loss
        entropy_case("entropy pixels", 4000, 35, 150, "fp32", "none", bias=True, train=False,
                     ignored=0.3),
        # the labels of a 640x480 view over the words of a vocabulary
        entropy_case("entropy image train", 640 * 480, 64, 4096, "bf16", "mean", bias=True),
        # odd sizes in fp32
        entropy_case("entropy fp32 train", 20001, 100, 1203, "fp32", "none", bias=True),
        # wide language features against a large vocabulary: the products count
        entropy_case("entropy vocabulary train", 65536, 512, 32768, "bf16", "mean"),
        # a small feature decoder's layers: latency
        adamw_case("adamw decoder", "decoder", 64, "fp32", 32, 0.01, 7),
        # a scene of a million Gaussians with third-order spherical harmonics
        adamw_case("adamw scene", "scene", 1000000, "fp32", 32, 0.0, 1000),
        # the same with its states in 8 bits
        adamw_case("adamw scene 8 bits", "scene", 1000000, "fp32", 8, 0.0, 1000),
    ]


def _spread(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["layer_norm", "embedding", "cross_entropy", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "layer_norm":
        act = rng.choice(["none", "relu", "silu", "gelu", "sigmoid"])
        # relu's slope jumps: among 10^7 values one lies within an fp32 rounding of the border
        train = rng.random() < 0.5 and not (act == "relu" and dtype == "fp32")
        channels = _spread(rng, 4, 2048)
        if rng.random() < 0.5:
            channels = -(-channels // 8) * 8
        most = MOST_VALUES // (4 if train and dtype == "fp32" else 2)
        rows = min(_spread(rng, 1, 1600 * 1200), most // channels)
        return {"op": op, "rows": rows, "channels": channels, "dtype": dtype, "act": act,
                "train": train}
    if op == "embedding":
        channels = _spread(rng, 3, 512)
        if rng.random() < 0.5:
            channels = -(-channels // 8) * 8
        most = MOST_LOOKED_UP // (2 if dtype == "fp32" else 1)
        return {"op": op, "ids": min(_spread(rng, 1, 1000000), most // channels),
                "entries": min(_spread(rng, 2, 1 << 17), most // channels), "channels": channels,
                "dtype": dtype, "scale": rng.choice([1.0, 0.5, 0.3, math.sqrt(channels)]),
                "train": rng.random() < 0.7}
    if op == "cross_entropy":
        train = rng.random() < 0.7
        k, vocabulary = _spread(rng, 8, 512), _spread(rng, 20, 32768)
        if rng.random() < 0.5:
            k = -(-k // 8) * 8
        # fp32 products take six of bf16 parts
        rows = min(_spread(rng, 1, 640 * 480),
                   MOST_PRODUCTS // (16 if dtype == "fp32" else 2) // (k * vocabulary),
                   (1 << 30) // vocabulary)
        return {"op": op, "rows": max(1, rows), "k": k, "vocabulary": vocabulary, "dtype": dtype,
                "reduction": rng.choice(["none", "sum", "mean"]), "bias": rng.random() < 0.5,
                "train": train, "ignored": rng.choice([0.0, 0.1, 0.5])}
    kind = rng.choice(["scene", "scene", "decoder"])
    count = (_spread(rng, 100, MOST_PARAMETERS // 59) if kind == "scene"
             else _spread(rng, 8, 512))
    return {"op": op, "kind": kind, "count": count,
            "dtype": "fp32" if kind == "scene" else dtype, "bits": rng.choice([8, 32]),
            "decay": rng.choice([0.0, 0.01]), "step": _spread(rng, 1, 30000)}


def parameters(case):
    """The shapes and learning rates of a case's tensors."""
    n = case["count"]
    if case["kind"] == "scene":
        return [((n, 3), 1.6e-4), ((n, 4), 1e-3), ((n, 3), 5e-3), ((n,), 5e-2),
                ((n, 1, 3), 2.5e-3), ((n, 15, 3), 1.25e-4)]
    return [((n, 35), 1e-3), ((n,), 1e-3), ((n,), 1e-3), ((n,), 1e-3), ((n, n), 1e-3),
            ((n,), 1e-3), ((3, n), 1e-3), ((3,), 1e-3)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(to)

    def whole(low, high, *shape, to=torch.int64):
        return torch.randint(low, high, shape, generator=g, device="cuda").to(to)

    s = {"case": case}
    if op == "layer_norm":
        rows, channels = case["rows"], case["channels"]
        means = torch.randn(channels, generator=g, device="cuda")
        s["x"] = (torch.randn(rows, channels, generator=g, device="cuda") * 1.5 + means).to(dtype)
        s["weight"] = normal(channels, scale=0.2, shift=1.0)
        s["bias"] = normal(channels, scale=0.2)
        s["upstream"] = normal(rows, channels) if case["train"] else None
    elif op == "embedding":
        # some entries are far more common than others, and some never occur
        share = torch.rand(case["ids"], generator=g, device="cuda").square()
        s["ids"] = (share * case["entries"]).long().clamp(max=case["entries"] - 1)
        s["table"] = normal(case["entries"], case["channels"])
        s["upstream"] = normal(case["ids"], case["channels"]) if case["train"] else None
    elif op == "cross_entropy":
        rows, k, vocabulary = case["rows"], case["k"], case["vocabulary"]
        s["x"] = normal(rows, k)
        s["weight"] = normal(vocabulary, k, scale=2 / math.sqrt(k))
        s["bias"] = normal(vocabulary, scale=0.5) if case["bias"] else None
        target = whole(0, vocabulary, rows)
        out = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        s["target"] = torch.where(out, torch.full_like(target, IGNORED), target)
        s["upstream"] = normal(*([rows] if case["reduction"] == "none" else []), scale=0.5,
                               shift=1.0, to=torch.float32) if case["train"] else None
    else:
        sizes = parameters(case)
        s["lr"] = [lr for _, lr in sizes]
        s["step"] = case["step"]
        s["params"] = [normal(*shape) for shape, _ in sizes]
        s["grads"] = [normal(*shape, scale=2.0 ** (-3 - i)) for i, (shape, _) in enumerate(sizes)]
        if case["bits"] == 32:
            s["first"] = [normal(*shape, scale=0.3 * 2.0 ** (-3 - i), to=torch.float32)
                          for i, (shape, _) in enumerate(sizes)]
            s["second"] = [normal(*shape, scale=2.0 ** (-3 - i), to=torch.float32).square() + 1e-8
                           for i, (shape, _) in enumerate(sizes)]
        else:
            runs = [-(-math.prod(shape) // RUN) for shape, _ in sizes]
            s["first"] = [(whole(0, 256, *shape, to=torch.uint8),
                           whole(-8 - i, -5 - i, n, to=torch.int8))
                          for i, ((shape, _), n) in enumerate(zip(sizes, runs))]
            s["second"] = [(whole(160, 256, *shape, to=torch.uint8),
                            whole(-6 - i, -3 - i, n, to=torch.int8))
                           for i, ((shape, _), n) in enumerate(zip(sizes, runs))]
    return s


# ---- plain forms -----------------------------------------------------------------

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


def plain_norm(s):
    act, dtype = s["case"]["act"], s["x"].dtype
    x, w, b = (s[name].float() for name in ("x", "weight", "bias"))
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
    hat = centred * rstd
    u = hat * w + b
    out = {"y": activate(u, act).to(dtype)}
    if s["upstream"] is not None:
        du = s["upstream"].float() * slope(u, act)
        dhat = du * w
        dx = rstd * (dhat - dhat.mean(1, keepdim=True) - hat * (dhat * hat).mean(1, keepdim=True))
        out["dx"] = dx.to(dtype)
        out["dweight"] = (du * hat).sum(0).to(dtype)
        out["dbias"] = du.sum(0).to(dtype)
    return out


def plain_embedding(s):
    scale, table = s["case"]["scale"], s["table"]
    out = {"y": (table.float()[s["ids"]] * scale).to(table.dtype)}
    if s["upstream"] is not None:
        # sums of many rows, in 64 bits
        sums = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
        sums.index_add_(0, s["ids"], s["upstream"].double())
        out["dtable"] = (sums * scale).to(table.dtype)
    return out


def plain_entropy(s):
    case, dtype = s["case"], s["x"].dtype
    x, w, target = s["x"].float(), s["weight"].float(), s["target"]
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    counts = target != IGNORED
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total) + top
    rows = torch.where(counts, (lse - z.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    del z
    number = counts.sum().clamp(min=1).float()
    loss = rows
    if case["reduction"] != "none":
        loss = rows.double().sum()
        loss = (loss / number if case["reduction"] == "mean" else loss).float()
    out = {"loss": loss}
    if s["upstream"] is not None:
        up = s["upstream"] * counts
        if case["reduction"] == "mean":
            up = up / number
        e /= total
        e.scatter_add_(1, at, torch.full_like(e[:, :1], -1.0))
        e *= up[:, None]
        out["dx"] = (e @ w).to(dtype)
        out["dweight"] = (e.t() @ x).to(dtype)
        if s["bias"] is not None:
            out["dbias"] = e.sum(0).to(dtype)
    return out


def dither(count, step, device):
    """16 bits for each of the two moments at every place: a hash of place and step."""
    low = 0xffffffff
    h = torch.arange(count, device=device)
    h = (h * 0x9e3779b9 + (step & low) * 0x6a09e667 + (h >> 32) * 0xbb67ae85) & low
    h = ((h ^ (h >> 16)) * 0x3c6ef373) & low
    h = ((h ^ (h >> 15)) * 0x510e527f) & low
    h = h ^ (h >> 16)
    return h & 0xffff, h >> 16


def power(exponents):
    """2^E as fp32, each exactly, of exponents in [-127, 127]."""
    return torch.ldexp(torch.ones_like(exponents, dtype=torch.float64), exponents).float()


def decode(codes, exponents, bits):
    """The values that 8-bit codes stand for: magnitudes of `bits` bits of mantissa."""
    c, shape = codes.reshape(-1).int(), codes.shape
    sign = None
    if bits == 3:
        sign = 1 - 2 * (c >> 7)
        c = c & 127
    normal = (((c >> bits) + 112) << 23) | ((c & (2 ** bits - 1)) << (23 - bits))
    value = torch.where(c < 2 ** bits, c.float() * 2.0 ** (-14 - bits), normal.view(torch.float32))
    if sign is not None:
        value = value * sign
    scale = power(exponents.int()).repeat_interleave(RUN)[:value.numel()]
    return (value * scale).reshape(shape)


def encode(values, bits, noise):
    """Codes and exponents of fp32 values."""
    x = values.reshape(-1)
    n = x.numel()
    runs = torch.nn.functional.pad(x, (0, -n % RUN)).reshape(-1, RUN)
    most = runs.abs().amax(1).view(torch.int32)
    top = (1 << 23) - (1 << (23 - bits))  # the largest code's mantissa
    exponents = ((most >> 23) - 127 + ((most & 0x7fffff) > top)).clamp(-126, 127)
    y = x.abs() * power(-exponents).repeat_interleave(RUN)[:n]
    drop = 23 - bits
    normal = ((y.view(torch.int32).long() + (noise << (drop - 16))) >> drop) - (112 << bits)
    small = torch.floor(y * 2.0 ** (14 + bits) + noise.float() * 2.0 ** -16).long()
    c = torch.where(y < 2.0 ** -14, small, normal)
    if bits == 3:
        c = c.clamp(max=127) | ((x < 0).long() << 7)
    else:
        c = torch.where((x > 0) & (c == 0), torch.ones_like(c), c.clamp(max=255))
    return c.to(torch.uint8).reshape(values.shape), exponents.to(torch.int8)


def plain_adamw(s):
    case, step = s["case"], s["step"]
    held = case["bits"] == 8
    fix1, fix2 = 1 - BETAS[0] ** step, 1 - BETAS[1] ** step
    out = {"params": [], "first": [], "second": []}
    for i, (p, g, lr) in enumerate(zip(s["params"], s["grads"], s["lr"])):
        m, v = s["first"][i], s["second"][i]
        if held:
            m, v = decode(*m, 3), decode(*v, 4).square()
        wide = g.float()
        # single fp32 operations: values next to a border between codes depend on each
        m = m * BETAS[0] + wide * (1 - BETAS[0])
        v = v * BETAS[1] + (wide * (1 - BETAS[1])) * wide
        root = torch.sqrt(v)
        update = m / (root / math.sqrt(fix2) + 1e-15)
        p.copy_(p.float() * (1 - lr * case["decay"]) - update * (lr / fix1))
        if held:
            noise = dither(p.numel(), step, p.device)
            for t, u in zip(s["first"][i], encode(m, 3, noise[0])):
                t.copy_(u)
            for t, u in zip(s["second"][i], encode(root, 4, noise[1])):
                t.copy_(u)
            m, v = decode(*s["first"][i], 3), decode(*s["second"][i], 4).square()
        else:
            m, v = s["first"][i].copy_(m), s["second"][i].copy_(v)
        out["params"].append(p)
        out["first"].append(m)
        out["second"].append(v)
    s["step"] = step + 1
    return out


# ---- the framework's operators ---------------------------------------------------

def own_norm(s):
    from dsl_splat_b200 import features

    act = s["case"]["act"]
    if s["upstream"] is None:
        return {"y": features.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, activation=act)}
    leaves = [s[m].detach().requires_grad_() for m in ("x", "weight", "bias")]
    y = features.layer_norm(*leaves, eps=EPS, activation=act)
    dx, dweight, dbias = torch.autograd.grad(y, leaves, s["upstream"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def own_embedding(s):
    from dsl_splat_b200 import features

    scale = s["case"]["scale"]
    if s["upstream"] is None:
        return {"y": features.embedding(s["ids"], s["table"], scale=scale)}
    table = s["table"].detach().requires_grad_()
    y = features.embedding(s["ids"], table, scale=scale)
    return {"y": y.detach(), "dtable": torch.autograd.grad(y, table, s["upstream"])[0]}


def own_entropy(s):
    from dsl_splat_b200 import features

    reduction = s["case"]["reduction"]
    if s["upstream"] is None:
        return {"loss": features.linear_cross_entropy(s["x"], s["weight"], s["target"], s["bias"],
                                                      ignore_index=IGNORED, reduction=reduction)}
    names = [m for m in ("x", "weight", "bias") if s[m] is not None]
    leaves = {m: s[m].detach().requires_grad_() for m in names}
    loss = features.linear_cross_entropy(leaves["x"], leaves["weight"], s["target"],
                                         leaves.get("bias"), ignore_index=IGNORED,
                                         reduction=reduction)
    grads = torch.autograd.grad(loss, list(leaves.values()), s["upstream"])
    return {"loss": loss.detach(), **{"d" + m: v for m, v in zip(names, grads)}}


def own_adamw(s):
    from dsl_splat_b200 import optim

    first, second = s["first"], s["second"]
    if s["case"]["bits"] == 8:
        first = [optim.Moment8(*t) for t in first]
        second = [optim.Moment8(*t, squared=True) for t in second]
    optim.adamw(s["params"], s["grads"], first, second, step=s["step"], lr=s["lr"], betas=BETAS,
                eps=1e-15, weight_decay=s["case"]["decay"])
    s["step"] += 1
    if s["case"]["bits"] == 8:
        first, second = ([t.values() for t in moments] for moments in (first, second))
    return {"params": s["params"], "first": first, "second": second}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": own_norm, "embedding": own_embedding, "cross_entropy": own_entropy,
                "adamw": own_adamw}[op](state)
    return {"layer_norm": plain_norm, "embedding": plain_embedding,
            "cross_entropy": plain_entropy, "adamw": plain_adamw}[op](state)


def work(case):
    size, op = SIZES[case["dtype"]], case["op"]
    if op == "layer_norm":
        values, channels = case["rows"] * case["channels"], case["channels"]
        passes = 4 if case["train"] else 2
        return {"bytes": size * passes * (values + channels),
                "flops": (24 if case["train"] else 8) * values}
    if op == "embedding":
        looked_up, held = case["ids"] * case["channels"], case["entries"] * case["channels"]
        # every entry is read once at most, every looked-up row written once
        read = min(looked_up, held)
        if not case["train"]:
            return {"bytes": size * (looked_up + read) + 8 * case["ids"], "flops": looked_up}
        return {"bytes": size * (2 * looked_up + read + held) + 8 * case["ids"],
                "flops": 2 * looked_up}
    if op == "cross_entropy":
        rows, k, vocabulary = case["rows"], case["k"], case["vocabulary"]
        values = (rows + vocabulary) * k + vocabulary * case["bias"]
        losses = rows if case["reduction"] == "none" else 1
        return {"bytes": (2 if case["train"] else 1) * (size * values + 4 * losses) + 8 * rows,
                "flops": (6 if case["train"] else 2) * rows * k * vocabulary}
    values = sum(math.prod(shape) for shape, _ in parameters(case))
    # gradient, parameter and both moments; 8-bit moments are read back as values besides
    moments = 16 if case["bits"] == 32 else 4 + 4 / RUN + 8
    return {"bytes": values * (3 * size + moments), "flops": 16 * values}


# ---- the definitions in 64 bits --------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "layer_norm":
        return exact_norm(case, s)
    if op == "embedding":
        table, ids, scale = s["table"].double(), s["ids"], case["scale"]
        out = {"y": scale * table.index_select(0, ids)}
        if case["train"]:
            # sums between the ends of each entry's run among the sorted rows
            order = torch.argsort(ids, stable=True)
            ends = torch.searchsorted(ids[order], torch.arange(len(table), device=ids.device),
                                      right=True)
            along = torch.cumsum(s["upstream"].double()[order], 0)
            along = torch.cat([torch.zeros_like(along[:1]), along])[ends]
            out["dtable"] = scale * torch.diff(along, dim=0, prepend=torch.zeros_like(along[:1]))
        return out
    if op == "cross_entropy":
        return exact_entropy(case, s)
    return exact_adamw(case, s)


def exact_norm(case, s):
    x, w, b = (s[m].double() for m in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    deviation = torch.sqrt(var + EPS)
    hat = (x - mean) / deviation
    u = w * hat + b
    sig = torch.special.expit(u)
    cdf = 0.5 * torch.special.erfc(-u / math.sqrt(2))
    value, rate = {
        "none": lambda: (u, torch.ones_like(u)),
        "relu": lambda: (u.clamp(min=0), torch.heaviside(u, torch.zeros_like(u))),
        "silu": lambda: (u * sig, sig + u * sig * torch.special.expit(-u)),
        "gelu": lambda: (u * cdf, cdf + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)),
        "sigmoid": lambda: (sig, sig * torch.special.expit(-u)),
    }[case["act"]]()
    out = {"y": value}
    if case["train"]:
        du = s["upstream"].double() * rate
        n = case["channels"]
        d = du * w
        along = torch.einsum("rc,rc->r", d, hat)[:, None] / n
        out["dx"] = (d - torch.einsum("rc->r", d)[:, None] / n - hat * along) / deviation
        out["dweight"] = torch.einsum("rc,rc->c", du, hat)
        out["dbias"] = torch.einsum("rc->c", du)
    return out


def exact_entropy(case, s):
    x, w = s["x"].double(), s["weight"].double()
    b = None if s["bias"] is None else s["bias"].double()
    target, rows = s["target"], case["rows"]
    used = (target != IGNORED).double()
    share = torch.ones_like(used)
    if case["reduction"] == "mean":
        share = share / max(1.0, float(used.sum()))
    up = used * share * s["upstream"].double() if case["train"] else None
    losses, dx = [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(w[:, 0])
    step = max(1, (1 << 28) // case["vocabulary"])
    for r in range(0, rows, step):
        piece = slice(r, min(rows, r + step))
        z = torch.einsum("rk,vk->rv", x[piece], w)
        if b is not None:
            z += b
        lse = torch.logsumexp(z, 1)
        label = target[piece].clamp(min=0)
        losses.append((lse - z[torch.arange(len(z), device=z.device), label]) * used[piece])
        if not case["train"]:
            continue
        z = torch.exp(z - lse[:, None])
        z[torch.arange(len(z), device=z.device), label] -= 1
        z *= up[piece, None]
        dx.append(torch.einsum("rv,vk->rk", z, w))
        dw += torch.einsum("rv,rk->vk", z, x[piece])
        db += z.sum(0)
    loss = torch.cat(losses)
    out = {"loss": loss if case["reduction"] == "none" else (loss * share).sum()}
    if case["train"]:
        out["dx"], out["dweight"] = torch.cat(dx), dw
        if b is not None:
            out["dbias"] = db
    return out


def exact_adamw(case, s):
    def value(moment, mantissa):
        """Of a code's sign, exponent and mantissa."""
        codes, exponents = moment
        c = codes.double().reshape(-1)
        negative = (c >= 128) if mantissa == 8 else torch.zeros_like(c, dtype=torch.bool)
        c = torch.where(negative, c - 128, c)
        e, f = torch.div(c, mantissa, rounding_mode="floor"), torch.remainder(c, mantissa)
        size = torch.where(e == 0, f / mantissa * 2.0 ** -14, (1 + f / mantissa) * 2.0 ** (e - 15))
        run = torch.arange(len(c), device=c.device) // RUN
        return (torch.where(negative, -size, size) * 2.0 ** exponents.double()[run]).reshape(
            codes.shape)

    t, (b1, b2) = case["step"], BETAS
    out = {"params": [], "first": [], "second": []}
    for p, g, lr, m, v in zip(s["params"], s["grads"], s["lr"], s["first"], s["second"]):
        p, g = p.double(), g.double()
        if case["bits"] == 8:
            m, v = value(m, 8), value(v, 16) ** 2
        m, v = b1 * m.double() + (1 - b1) * g, b2 * v.double() + (1 - b2) * g ** 2
        step = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + 1e-15)
        out["params"].append(p - lr * case["decay"] * p - lr * step)
        # what is rounded to 8 bits has no value in 64
        out["first"].append(m if case["bits"] == 32 else None)
        out["second"].append(v if case["bits"] == 32 else None)
    return out
