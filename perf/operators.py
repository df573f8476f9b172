"""Workloads over the transformer operators of ``cltorch_amd``: layer norm, the linear layer (matrix product with
bias, activation and residual) and the matrix product grouped by expert, each forward alone and as a training pass.

``run`` computes a case with elementary torch operations, or, with ``own`` true, through ``cltorch_amd``'s entry
points on tensors of its own.  Both get the same values.
"""
import math

import torch

own = False

EPS = 1e-5


# ---------------------------------------------------------------- cases ---
def listed():
    return [
        # the norm in front of a block while one token is generated: one row, latency counts
        {"name": "norm 1x4096", "op": "norm", "train": False, "rows": 1, "width": 4096},
        # the same over a batch of prompts
        {"name": "norm 16384x4096", "op": "norm", "train": False, "rows": 16384, "width": 4096},
        # a training step's norm with a ragged batch and a width that is no multiple of a vector load
        {"name": "norm train 2047x1537", "op": "norm", "train": True, "rows": 2047, "width": 1537},
        # a training step's norm of a wide model
        {"name": "norm train 8192x8192", "op": "norm", "train": True, "rows": 8192, "width": 8192},
        # the first half of a feed-forward block for one generated token: the weights are read once
        {"name": "linear 1x4096x16384", "op": "linear", "train": False, "rows": 1, "inner": 4096, "outer": 16384,
         "act": "gelu", "bias": True, "residual": False},
        # the same for 64 sequences that generate together
        {"name": "linear 64x4096x16384", "op": "linear", "train": False, "rows": 64, "inner": 4096, "outer": 16384,
         "act": "silu", "bias": True, "residual": False},
        # the projection that closes a block, added to the residual stream, over a prompt
        {"name": "linear 2048x4096x4096", "op": "linear", "train": False, "rows": 2048, "inner": 4096, "outer": 4096,
         "act": "none", "bias": True, "residual": True},
        # a training step on a ragged batch with odd widths
        {"name": "linear train 1531x1027x2053", "op": "linear", "train": True, "rows": 1531, "inner": 1027, "outer": 2053,
         "act": "gelu", "bias": True, "residual": True},
        # a training step of a large layer
        {"name": "linear train 8192x8192x8192", "op": "linear", "train": True, "rows": 8192, "inner": 8192, "outer": 8192,
         "act": "silu", "bias": True, "residual": False},
        # 32 generated tokens, two experts each: most experts see a few rows, some none
        {"name": "grouped 64x1024x2048 of 16", "op": "grouped", "train": False, "rows": 64, "inner": 1024, "outer": 2048, "groups": 16},
        # a prompt's tokens over the experts of one layer
        {"name": "grouped 8192x2048x4096 of 16", "op": "grouped", "train": False, "rows": 8192, "inner": 2048, "outer": 4096, "groups": 16},
        # a training step of ragged experts with odd widths
        {"name": "grouped train 4095x1023x2049 of 8", "op": "grouped", "train": True, "rows": 4095, "inner": 1023, "outer": 2049, "groups": 8},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of its range; a third are multiples of 64, a third of 4, the rest anything."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    step = rng.choice((1, 4, 64))
    return min(high, max(low, n // step * step))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "grouped"))
    train = rng.random() < 0.5
    while True:
        rows = _size(rng, 1, 16384)
        if op == "norm":
            width = _size(rng, 64, 8192)
            if rows * width <= 1 << 26:
                return {"op": op, "train": train, "rows": rows, "width": width}
            continue
        inner, outer = _size(rng, 64, 16384), _size(rng, 64, 16384)
        if op == "linear":
            if rows * inner * outer <= 1 << 38 and max(rows, inner) * outer <= 1 << 27:
                # relu forward only: the two sides of its step at 0 differ by more than any rounding of what feeds it
                act = rng.choice(("none", "gelu", "silu") if train else ("none", "relu", "gelu", "silu"))
                return {"op": op, "train": train, "rows": rows, "inner": inner, "outer": outer,
                        "act": act, "bias": rng.random() < 0.8, "residual": rng.random() < 0.4}
            continue
        groups = _size(rng, 2, 64)
        if rows >= 16 and rows * inner * outer <= 1 << 36 and groups * inner * outer <= 1 << 28 and rows * max(inner, outer) <= 1 << 26:
            return {"op": op, "train": train, "rows": rows, "inner": inner, "outer": outer, "groups": groups}


def _group_sizes(case, seed):
    """Rows of each group as a router leaves them: uneven shares, and with few rows some groups get none."""
    g = torch.Generator().manual_seed(int(seed) * 7919 + 1)
    share = torch.softmax(0.7 * torch.randn(case["groups"], generator=g), 0)
    pick = torch.multinomial(share, case["rows"], replacement=True, generator=g)
    return torch.bincount(pick, minlength=case["groups"]).tolist()


def work(case):
    r = case["rows"]
    if case["op"] == "norm":
        d = case["width"]
        return {"bytes": 4 * (4 * r * d + 4 * d) if case["train"] else 4 * (2 * r * d + 2 * d), "flops": (20 if case["train"] else 8) * r * d}
    k, n = case["inner"], case["outer"]
    weights = k * n
    if case["op"] == "grouped":
        weights *= min(case["groups"], r)
        extra = 0
    else:
        extra = (n if case["bias"] else 0) + (r * n if case["residual"] else 0)
    forward = 4 * (r * k + weights + r * n + extra)
    if not case["train"]:
        return {"bytes": forward, "flops": 2 * r * k * n}
    backward = 4 * (r * n + r * k + weights + (n if case.get("bias") else 0))
    return {"bytes": forward + backward, "flops": 6 * r * k * n}


# --------------------------------------------------------------- inputs ---
def _values(case, seed):
    """The inputs of a case as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(mean)

    r, t = case["rows"], {}
    if case["op"] == "norm":
        d = case["width"]
        # a residual stream: rows of different scale around a small offset of their own
        t["x"] = normal(r, d) * torch.exp(normal(r, 1, scale=0.5)) + normal(r, 1, scale=0.3)
        t["weight"], t["bias"] = normal(d, scale=0.2, mean=1.0), normal(d, scale=0.1)
        if case["train"]:
            t["gy"] = normal(r, d, scale=0.05)
        return t
    k, n = case["inner"], case["outer"]
    t["x"] = normal(r, k)
    if case["op"] == "linear":
        t["weight"] = normal(n, k, scale=k ** -0.5)
        if case["bias"]:
            t["bias"] = normal(n, scale=0.1)
        if case["residual"]:
            t["residual"] = normal(r, n)
    else:
        t["weight"] = normal(case["groups"], k, n, scale=k ** -0.5)
    if case["train"]:
        t["gy"] = normal(r, n, scale=0.05)
    return t


class _OnDevice:
    """Lets torch read and write a ClTensor's memory, and keeps the tensor alive meanwhile."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": tensor.size(), "typestr": "<f4", "data": (tensor.data_ptr(), False), "version": 3}


def _seen_by_torch(tensor):
    return torch.as_tensor(_OnDevice(tensor), device="cuda")


def _results(case):
    """Shapes of what a pass leaves, and of what a training pass keeps from its forward half for its backward half."""
    r = case["rows"]
    if case["op"] == "norm":
        d = case["width"]
        out, kept = {"y": (r, d)}, {}
        if case["train"]:
            out.update(gx=(r, d), gweight=(d,), gbias=(d,))
            kept.update(mean=(r,), rstd=(r,))
        return out, kept
    k, n = case["inner"], case["outer"]
    out, kept = {"y": (r, n)}, {}
    if case["train"]:
        out.update(gx=(r, k), gweight=(n, k) if case["op"] == "linear" else (case["groups"], k, n))
        if case.get("bias"):
            out["gbias"] = (n,)
        if case.get("act", "none") != "none":
            kept["z"] = (r, n)
    return out, kept


def prepare(case, seed):
    state = {"case": case}
    values = _values(case, seed)
    if case["op"] == "grouped":
        state["sizes"] = _group_sizes(case, seed)
        values["sizes"] = torch.tensor(state["sizes"], dtype=torch.float32, device="cuda")
    if own:
        # the library's tensors hold the same values, and its results go to tensors that a program keeps from step to step
        import cltorch_amd as cl
        for name in list(values):
            state[name] = cl.ClTensor(*values[name].shape)
            _seen_by_torch(state[name]).copy_(values.pop(name))
        out, kept = _results(case)
        for name, shape in {**out, **kept}.items():
            state[name] = cl.ClTensor(*shape)
        state["out"] = {name: _seen_by_torch(state[name]) for name in out}
        torch.cuda.synchronize()  # the library's stream does not wait for torch's
    else:
        sizes = state.pop("sizes", None)
        state.update(values)
        state["sizes"] = sizes
    return state


# ------------------------------------------------------------ plain form ---
def _act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(name, z):
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_norm(s):
    x = s["x"]
    away = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((away * away).mean(1, keepdim=True) + EPS)
    hat = away * rstd
    out = {"y": hat * s["weight"] + s["bias"]}
    if s["case"]["train"]:
        g = s["gy"] * s["weight"]
        out["gx"] = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        out["gweight"] = (s["gy"] * hat).sum(0)
        out["gbias"] = s["gy"].sum(0)
    return out


def _plain_linear(s):
    case = s["case"]
    z = s["x"] @ s["weight"].t()
    if case["bias"]:
        z = z + s["bias"]
    y = _act(case["act"], z)
    out = {"y": y + s["residual"] if case["residual"] else y}
    if case["train"]:
        gz = s["gy"] if case["act"] == "none" else s["gy"] * _act_slope(case["act"], z)
        out["gx"] = gz @ s["weight"]
        out["gweight"] = gz.t() @ s["x"]
        if case["bias"]:
            out["gbias"] = gz.sum(0)
    return out


def _plain_grouped(s):
    # one product per group, over the rows that are its own
    xs, ws = s["x"].split(s["sizes"]), s["weight"]
    out = {"y": torch.cat([x @ w for x, w in zip(xs, ws)])}
    if s["case"]["train"]:
        gs = s["gy"].split(s["sizes"])
        out["gx"] = torch.cat([g @ w.t() for g, w in zip(gs, ws)])
        out["gweight"] = torch.stack([x.t() @ g for x, g in zip(xs, gs)])
    return out


# -------------------------------------------------------- the library's ---
def _own_norm(s):
    import cltorch_amd as cl
    if not s["case"]["train"]:
        s["y"].layerNorm(s["x"], s["weight"], s["bias"], EPS)
    else:
        s["y"].layerNorm(s["x"], s["weight"], s["bias"], EPS, mean=s["mean"], rstd=s["rstd"])
        cl.layerNormBackward(s["gx"], s["gweight"], s["gbias"], s["gy"], s["x"], s["weight"], s["mean"], s["rstd"])
    return s["out"]


def _own_linear(s):
    import cltorch_amd as cl
    act = s["case"]["act"]
    s["y"].linear(s["x"], s["weight"], s.get("bias"), residual=s.get("residual"), activation=act, preact=s.get("z"))
    if s["case"]["train"]:
        cl.linearBackward(s["gx"], s["gweight"], s.get("gbias"), s["gy"], s["x"], s["weight"], preact=s.get("z"), activation=act)
    return s["out"]


def _own_grouped(s):
    import cltorch_amd as cl
    s["y"].groupedmm(s["x"], s["weight"], s["sizes"])
    if s["case"]["train"]:
        cl.groupedmmBackward(s["gx"], s["gweight"], s["gy"], s["x"], s["weight"], s["sizes"])
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "grouped": _own_grouped}[op](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "grouped": _plain_grouped}[op](state)


# ---------------------------------------------------------------- exact ---
def _exact_norm(case, t):
    x, w = t["x"], t["weight"]
    d = x.shape[1]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    inv = (var + EPS).rsqrt()
    out = {"y": torch.addcmul(t["bias"], (x - mean) * inv, w)}
    if case["train"]:
        gy = t["gy"]
        # through the Jacobian of the normalised row: inv * (1 - 1/d - hat hat^T / d)
        hat = (x - mean).mul_(inv)
        g = gy * w
        out["gx"] = (g - g.sum(1, keepdim=True) / d - hat * (torch.linalg.vecdot(g, hat)[:, None] / d)) * inv
        out["gweight"] = torch.linalg.vecdot(gy, hat, dim=0)
        out["gbias"] = torch.ones(1, x.shape[0], dtype=x.dtype, device=x.device).matmul(gy)[0]
    return out


def _exact_linear(case, t):
    z = torch.mm(t["x"], t["weight"].T.contiguous())
    if case["bias"]:
        z += t["bias"]
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2.0))
    y = {"none": lambda: z, "relu": lambda: z.clamp(min=0.0), "gelu": lambda: z * cdf, "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
    out = {"y": y + t["residual"] if case["residual"] else y}
    if case["train"]:
        if case["act"] == "gelu":
            slope = cdf + z * torch.exp(z.square() / -2.0) / math.sqrt(2.0 * math.pi)
        elif case["act"] == "silu":
            p = torch.sigmoid(z)
            slope = p + z * p * torch.sigmoid(-z)
        else:
            slope = torch.ones_like(z)
        gz = t["gy"] * slope
        out["gx"] = torch.mm(gz, t["weight"])
        out["gweight"] = torch.mm(t["x"].T.contiguous(), gz).T
        if case["bias"]:
            out["gbias"] = torch.ones(1, z.shape[0], dtype=z.dtype, device=z.device).matmul(gz)[0]
    return out


def _exact_grouped(case, t, sizes):
    x, w = t["x"], t["weight"]
    out = {"y": torch.empty(x.shape[0], w.shape[2], dtype=x.dtype, device=x.device)}
    if case["train"]:
        out["gx"], out["gweight"] = torch.empty_like(x), torch.zeros_like(w)
    at = 0
    for g, n in enumerate(sizes):
        if n == 0:
            continue
        rows = slice(at, at + n)
        out["y"][rows] = torch.mm(x[rows], w[g])
        if case["train"]:
            out["gx"][rows] = torch.mm(w[g], t["gy"][rows].T.contiguous()).T
            out["gweight"][g] = torch.mm(t["gy"][rows].T.contiguous(), x[rows]).T
        at += n
    return out


def exact(case, seed):
    t = {name: v.double() for name, v in _values(case, seed).items()}
    if case["op"] == "norm":
        return _exact_norm(case, t)
    if case["op"] == "linear":
        return _exact_linear(case, t)
    return _exact_grouped(case, t, _group_sizes(case, seed))
