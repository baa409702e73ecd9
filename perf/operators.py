"""What is measured of the training operators of ``torch_kunlun_b200.ops``:
``dropout`` (a counter-based mask that is never stored), ``residual_norm``
(the norms behind and before a transformer block with its dropout, gate and
residual scale) and ``linear_cross_entropy`` (a vocabulary projection and its
loss without the logits), each forward and with its gradients.

With ``own`` false the cases run in plain torch operations on the CUDA device;
with ``own`` true on the kunlun device, through the calls a user makes.
"""

import math

import torch

own = False

LOW = 0xFFFFFFFF
IGNORE = -100


def listed():
    return [
        # the hidden state of one generated or scored token: latency alone
        {"name": "dropout_token_fp16", "op": "dropout", "dtype": "float16", "rows": 1, "cols": 768, "p": 0.1, "grad": False},
        # FFN activations of a training step, 16384 tokens of 4096
        {"name": "dropout_tokens_fp16", "op": "dropout", "dtype": "float16", "rows": 16384, "cols": 4096, "p": 0.1, "grad": True},
        # a ragged fp32 batch, neither size a multiple of anything
        {"name": "dropout_odd_fp32", "op": "dropout", "dtype": "float32", "rows": 4097, "cols": 1023, "p": 0.5, "grad": True},
        # one token for each of four requests behind an encoder's attention
        {"name": "norm_token_fp16", "op": "norm", "dtype": "float16", "batch": 4, "tokens": 1, "cols": 768, "kind": "layer", "post": False,
         "gate": "none", "scale": 1.0, "p": 0.0, "grad": False},
        # the encoder block's add and LayerNorm with dropout, 32 sequences of 512 tokens in training
        {"name": "norm_encoder_fp16", "op": "norm", "dtype": "float16", "batch": 32, "tokens": 512, "cols": 768, "kind": "layer", "post": False,
         "gate": "none", "scale": 1.0, "p": 0.1, "grad": True},
        # norms on both sides of a block, a learned gate for each channel
        {"name": "norm_both_sides_fp16", "op": "norm", "dtype": "float16", "batch": 4, "tokens": 2048, "cols": 4096, "kind": "rms", "post": True,
         "gate": "channel", "scale": 1.0, "p": 0.0, "grad": True},
        # a gate for each sample (conditioned blocks), scaled residual, ragged sizes in fp32
        {"name": "norm_sample_gate_fp32", "op": "norm", "dtype": "float32", "batch": 7, "tokens": 333, "cols": 1151, "kind": "layer", "post": True,
         "gate": "sample", "scale": 1.25, "p": 0.1, "grad": True},
        # a wide model's prompt, forward only
        {"name": "norm_wide_fp16", "op": "norm", "dtype": "float16", "batch": 1, "tokens": 2048, "cols": 16384, "kind": "rms", "post": True,
         "gate": "channel", "scale": 1.0, "p": 0.0, "grad": False},
        # scoring a few tokens: one loss for each
        {"name": "loss_few_fp16", "op": "loss", "dtype": "float16", "rows": 8, "cols": 768, "vocab": 30011, "bias": False, "ignored": 0, "reduction": "none", "grad": False},
        # the step of a language model, every token a target
        {"name": "loss_tokens_fp16", "op": "loss", "dtype": "float16", "rows": 8192, "cols": 4096, "vocab": 65536, "bias": False, "ignored": 0, "reduction": "mean", "grad": True},
        # masked-token training of an encoder: about one target in seven, the others ignored
        {"name": "loss_masked_fp16", "op": "loss", "dtype": "float16", "rows": 16384, "cols": 768, "vocab": 30011, "bias": True, "ignored": 14000, "reduction": "mean", "grad": True},
        # a small fp32 model, ragged in every size
        {"name": "loss_odd_fp32", "op": "loss", "dtype": "float32", "rows": 1021, "cols": 1023, "vocab": 20011, "bias": True, "ignored": 37, "reduction": "sum", "grad": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "loss"])
    dtype = rng.choice(["float16", "float16", "float32"])
    grad = rng.random() < 0.7
    p = rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9])
    if op == "dropout":
        cols = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, max(1, 16384 * 4096 // (2 * cols)))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "p": p or 0.1, "grad": grad}
    if op == "norm":
        cols = _spread(rng, 8, 20000)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        batch = rng.randint(1, 33)
        tokens = _spread(rng, 1, max(1, 4 * 2048 * 4096 // (2 * cols * batch)))
        return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "cols": cols, "kind": rng.choice(["layer", "rms"]), "post": rng.random() < 0.6,
                "gate": rng.choice(["none", "channel", "sample"]), "scale": rng.choice([1.0, 1.0, 0.7, 2.5]), "p": rng.choice([0.0, p]), "grad": grad}
    cols = _spread(rng, 16, 6000)
    if rng.random() < 0.5:
        cols = max(64, cols // 64 * 64)
    vocab = _spread(rng, 100, 140000)
    rows = _spread(rng, 1, max(1, min(20000, 8192 * 65536 // (4 * vocab), 8192 * 4096 * 65536 // (2 * vocab * cols))))
    return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "vocab": vocab, "bias": rng.random() < 0.5,
            "ignored": rng.choice([0, 0, rows // 7, rows * 6 // 7]), "reduction": rng.choice(["mean", "mean", "sum", "none"]), "grad": grad}


# ---- inputs ---------------------------------------------------------------------


class _Memory:
    """A kunlun tensor's memory for torch.as_tensor: a kunlun device is a CUDA
    device, so its tensors can be read in place as CUDA tensors."""

    KINDS = {torch.float16: "<f2", torch.float32: "<f4", torch.int64: "<i8"}

    def __init__(self, t):
        self.t = t
        self.__cuda_array_interface__ = {"shape": tuple(t.shape), "typestr": self.KINDS[t.dtype], "data": (t.data_ptr(), False), "strides": None, "version": 3}


def _as_cuda(t):
    return torch.as_tensor(_Memory(t.detach()), device="cuda")


def _place(t, grad=False):
    """The tensor where the program keeps it: for the framework's calls on its own device."""
    if t is None:
        return None
    if own:
        import torch_kunlun_b200  # noqa: F401  (registers the device)

        k = torch.empty(t.shape, dtype=t.dtype, device="kunlun")
        _as_cuda(k).copy_(t)
        return k.requires_grad_(grad)
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    grad = case["grad"]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    s = {"case": case, "seed": 1_000_003 * seed + 17, "offset": 3}
    if case["op"] == "dropout":
        s["x"] = _place(normal(case["rows"], case["cols"]), grad)
        s["gy"] = _place(normal(case["rows"], case["cols"])) if grad else None
        return s
    if case["op"] == "norm":
        shape, d = (case["batch"], case["tokens"], case["cols"]), case["cols"]
        # a residual stream has channels with a mean of their own
        s["x"] = _place((normal(*shape).float() + torch.randn(d, generator=g, device="cuda")).to(dtype), grad)
        s["f"] = _place(normal(*shape, std=0.7), grad)
        s["weight"] = _place(normal(d, mean=1.0, std=0.1), grad)
        s["bias"] = _place(normal(d, std=0.1), grad) if case["kind"] == "layer" else None
        s["post_weight"] = _place(normal(d, mean=1.0, std=0.1), grad) if case["post"] else None
        s["post_bias"] = _place(normal(d, std=0.1), grad) if case["post"] and case["kind"] == "layer" else None
        shapes = {"none": None, "channel": (d,), "sample": (case["batch"], 1, d)}[case["gate"]]
        s["gate"] = _place(normal(*shapes, mean=0.5, std=0.3), grad) if shapes else None
        s["gx"] = _place(normal(*shape)) if grad else None
        s["gh"] = _place(normal(*shape)) if grad else None
        return s
    rows, d, v = case["rows"], case["cols"], case["vocab"]
    s["x"] = _place(normal(rows, d), grad)
    s["weight"] = _place(normal(v, d, std=2.0 / math.sqrt(d)), grad)
    s["bias"] = _place(normal(v, std=0.1), grad) if case["bias"] else None
    target = torch.randint(0, v, (rows,), generator=g, device="cuda")
    target[torch.randperm(rows, generator=g, device="cuda")[: case["ignored"]]] = IGNORE
    s["target"] = _place(target)
    # the loss's own gradient: one for each row, or the loss scale of fp16 training
    if case["reduction"] == "none":
        gl = torch.rand(rows, generator=g, device="cuda") + 0.5
    else:
        gl = torch.full((), 4096.0 if case["dtype"] == "float16" and case["reduction"] == "mean" else 1.0, device="cuda")
    s["gl"] = _place(gl) if grad else None
    return s


# ---- the plain forms --------------------------------------------------------------


def _words(n, seed, offset):
    """n words of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): element i
    is word i % 4 of counter (i // 4, offset) under the key `seed`."""
    i = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1 = i & LOW, i >> 32
    c2, c3 = torch.full_like(i, offset & LOW), torch.full_like(i, (offset >> 32) & LOW)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the 64-bit products' bits, kept under wrap-around
        c0, c1, c2, c3 = ((b >> 32) & LOW) ^ c1 ^ k0, b & LOW, ((a >> 32) & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    return torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)[:n]


def _keep(shape, p, seed, offset):
    return _words(math.prod(shape), seed, offset).view(shape) >= round(p * 2.0**32)


def _dropped(x, keep, p):
    return torch.where(keep, x * (1.0 / (1.0 - p)), 0.0)


def _plain_dropout(s):
    x, p = s["x"], s["case"]["p"]
    y = _dropped(x.float(), _keep(x.shape, p, s["seed"], s["offset"]), p).to(x.dtype)
    if s["gy"] is None:
        return y
    return y, _dropped(s["gy"].float(), _keep(x.shape, p, s["seed"], s["offset"]), p).to(x.dtype)


def _standardised(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    return v * r, r


def _standardised_grad(g, n, r, kind):
    g_mean = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return r * (g - g_mean - n * (g * n).mean(-1, keepdim=True))


def _plain_norm(s):
    c = s["case"]
    kind, eps, dtype = c["kind"], 1e-5, s["x"].dtype
    f32 = {k: s[k].float() for k in ("x", "f", "weight", "bias", "post_weight", "post_bias", "gate", "gx", "gh") if s[k] is not None}
    u = f32["f"]
    if c["post"]:
        pn, pr = _standardised(u, kind, eps)
        u = pn * f32["post_weight"] + f32.get("post_bias", 0.0)
    keep = _keep(u.shape, c["p"], s["seed"], s["offset"]) if c["p"] > 0 else None
    if keep is not None:
        u = _dropped(u, keep, c["p"])
    gate = f32.get("gate", 1.0)
    x_new = c["scale"] * f32["x"] + gate * u
    n, r = _standardised(x_new, kind, eps)
    h = n * f32["weight"] + f32.get("bias", 0.0)
    out = {"x_new": x_new.to(dtype), "h": h.to(dtype)}
    if not c["grad"]:
        return out
    gh = f32["gh"]
    g = f32["gx"] + _standardised_grad(gh * f32["weight"], n, r, kind)
    out["x"] = (c["scale"] * g).to(dtype)
    out["weight"] = (gh * n).sum((0, 1)).to(dtype)
    if "bias" in f32:
        out["bias"] = gh.sum((0, 1)).to(dtype)
    if "gate" in f32:
        out["gate"] = (g * u).sum(1, keepdim=True).to(dtype) if c["gate"] == "sample" else (g * u).sum((0, 1)).to(dtype)
    gu = gate * g
    if keep is not None:
        gu = _dropped(gu, keep, c["p"])
    if c["post"]:
        out["post_weight"] = (gu * pn).sum((0, 1)).to(dtype)
        if "post_bias" in f32:
            out["post_bias"] = gu.sum((0, 1)).to(dtype)
        gu = _standardised_grad(gu * f32["post_weight"], pn, pr, kind)
    out["f"] = gu.to(dtype)
    return out


def _plain_loss(s):
    c, dtype = s["case"], s["x"].dtype
    x, w, target = s["x"].float(), s["weight"].float(), s["target"]
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    top = z.amax(1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(1, keepdim=True)
    used = target != IGNORE
    at = torch.where(used, target, 0)[:, None]
    rows = torch.where(used, (total.log() + top - z.gather(1, at))[:, 0], 0.0)
    count = used.sum()
    out = {"loss": rows if c["reduction"] == "none" else rows.sum() if c["reduction"] == "sum" else rows.sum() / count}
    if not c["grad"]:
        return out
    g = torch.where(used, s["gl"] / count if c["reduction"] == "mean" else s["gl"], 0.0)[:, None]
    dz = e / total
    dz.scatter_add_(1, at, torch.full_like(g, -1.0))
    dz = dz * g
    out["x"] = (dz @ w).to(dtype)
    out["weight"] = (dz.t() @ x).to(dtype)
    if s["bias"] is not None:
        out["bias"] = dz.sum(0).to(dtype)
    return out


# ---- the framework's calls ----------------------------------------------------------


def _grads(outputs, inputs, grads):
    names = [k for k in inputs if inputs[k] is not None]
    return dict(zip(names, torch.autograd.grad(outputs, [inputs[k] for k in names], grads)))


def _own_dropout(s, ops):
    y = ops.dropout(s["x"], s["case"]["p"], s["seed"], s["offset"])
    if s["gy"] is None:
        return _as_cuda(y)
    (gx,) = torch.autograd.grad(y, s["x"], s["gy"])
    return _as_cuda(y), _as_cuda(gx)


def _own_norm(s, ops):
    c = s["case"]
    x_new, h = ops.residual_norm(s["x"], s["f"], s["weight"], s["bias"], norm=c["kind"], post_norm=c["post"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                                 gate=s["gate"], residual_scale=c["scale"], eps=1e-5, p=c["p"], seed=s["seed"], offset=s["offset"])
    out = {"x_new": x_new, "h": h}
    if c["grad"]:
        out.update(_grads((x_new, h), {k: s[k] for k in ("x", "f", "weight", "bias", "post_weight", "post_bias", "gate")}, (s["gx"], s["gh"])))
    return {k: _as_cuda(v) for k, v in out.items()}


def _own_loss(s, ops):
    c = s["case"]
    loss = ops.linear_cross_entropy(s["x"], s["weight"], s["target"], s["bias"], ignore_index=IGNORE, reduction=c["reduction"])
    out = {"loss": loss}
    if c["grad"]:
        out.update(_grads(loss, {k: s[k] for k in ("x", "weight", "bias")}, s["gl"]))
    return {k: _as_cuda(v) for k, v in out.items()}


def run(state):
    op = state["case"]["op"]
    if own:
        from torch_kunlun_b200 import ops

        return {"dropout": _own_dropout, "norm": _own_norm, "loss": _own_loss}[op](state, ops)
    return {"dropout": _plain_dropout, "norm": _plain_norm, "loss": _plain_loss}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------


def work(case):
    size = 2 if case["dtype"] == "float16" else 4
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": (4 if case["grad"] else 2) * n * size, "flops": (2 if case["grad"] else 1) * n}
    if case["op"] == "norm":
        n, d = case["batch"] * case["tokens"] * case["cols"], case["cols"]
        params = d * (1 + (case["kind"] == "layer")) * (1 + case["post"]) + d * {"none": 0, "channel": 1, "sample": case["batch"]}[case["gate"]]
        # x, f in and x_new, h out; then their two gradients in, dx and df out
        return {"bytes": size * ((8 if case["grad"] else 4) * n + (2 if case["grad"] else 1) * params), "flops": (40 if case["grad"] else 12) * n}
    rows, d, v = case["rows"] - case["ignored"], case["cols"], case["vocab"]
    values = rows * d + v * d + v * case["bias"]
    return {"bytes": size * (2 if case["grad"] else 1) * values + 8 * case["rows"], "flops": (6 if case["grad"] else 2) * rows * d * v}


# ---- the definitions in 64 bits -----------------------------------------------------------


def _times(a, m):
    """(high, low) words of a * m for 32-bit words, from 16-bit halves."""
    al, ah, ml, mh = a % 65536, a // 65536, m % 65536, m // 65536
    middle = ah * ml + (al * ml) // 65536
    other = al * mh + middle % 65536
    return ah * mh + middle // 65536 + other // 65536, (other % 65536) * 65536 + (al * ml) % 65536


def _kept64(shape, p, seed, offset):
    n = math.prod(shape)
    block = torch.arange(-(-n // 4), device="cuda", dtype=torch.int64)
    state = [block % 2**32, block // 2**32, torch.zeros_like(block) + offset % 2**32, torch.zeros_like(block) + offset // 2**32 % 2**32]
    for r in range(10):
        hi0, lo0 = _times(state[0], 0xD2511F53)
        hi1, lo1 = _times(state[2], 0xCD9E8D57)
        keys = (seed % 2**32 + r * 0x9E3779B9) % 2**32, (seed // 2**32 + r * 0xBB67AE85) % 2**32
        state = [hi1 ^ state[1] ^ keys[0], lo1, hi0 ^ state[3] ^ keys[1], lo0]
    words = torch.empty(4 * block.numel(), device="cuda", dtype=torch.int64)
    for k in range(4):
        words[k::4] = state[k]
    return (words[:n].reshape(shape) >= int(round(p * 4294967296.0))).double()


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    wide = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "dropout":
        m = _kept64(s["x"].shape, case["p"], s["seed"], s["offset"]) / (1 - case["p"])
        return (wide["x"] * m, wide["gy"] * m) if case["grad"] else wide["x"] * m
    leaves = {}
    for k in ("x", "f", "weight", "bias", "post_weight", "post_bias", "gate"):
        if torch.is_tensor(wide.get(k)):
            wide[k].requires_grad_(case["grad"])
            leaves[k] = wide[k]
    if case["op"] == "norm":
        def norm(v, w, b):
            if case["kind"] == "layer":
                y = (v - v.mean(-1, True)) / (v.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
            else:
                y = v / ((v * v).mean(-1, True) + 1e-5).sqrt()
            return y * w if b is None else y * w + b

        u = norm(wide["f"], wide["post_weight"], wide["post_bias"]) if case["post"] else wide["f"]
        if case["p"] > 0:
            u = u * (_kept64(u.shape, case["p"], s["seed"], s["offset"]) / (1 - case["p"]))
        x_new = case["scale"] * wide["x"] + (u if wide["gate"] is None else wide["gate"] * u)
        out = {"x_new": x_new, "h": norm(x_new, wide["weight"], wide["bias"])}
        ends, gs = (out["x_new"], out["h"]), (wide["gx"], wide["gh"])
    else:
        z = wide["x"] @ wide["weight"].T
        if wide["bias"] is not None:
            z = z + wide["bias"]
        used = (s["target"] != IGNORE).nonzero()[:, 0]
        rows = torch.zeros(case["rows"], device="cuda", dtype=torch.float64)
        rows = rows.index_put((used,), torch.logsumexp(z[used], 1) - z[used, s["target"][used]])
        loss = {"none": lambda: rows, "sum": rows.sum, "mean": lambda: rows.sum() / used.numel()}[case["reduction"]]()
        out = {"loss": loss}
        ends, gs = (loss,), (wide["gl"],)
    if case["grad"]:
        out.update(zip(leaves, torch.autograd.grad(ends, list(leaves.values()), gs)))
    return {k: v.detach() for k, v in out.items()}
