"""64-bit references of the training operators and the bounds their tests use.

`philox_words` is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011) in
numpy integers.  `residual_norm64` evaluates the residual norm and its
gradients from the formulas, with the sum of the absolute values of the terms
each result is built from: a result's error is at most one ulp of T (its
rounding, which a binary32 error can move across a boundary) plus a relative
error of those terms.
"""
import numpy as np
import torch

U32 = 2.0 ** -24          # half a binary32 step, relative
HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Roundings on a term's way through one row sum: at most 24 additions in a
# thread and 5 + 9 levels across threads, then a handful of products.
K = 48


def philox_words(n, seed, offset):
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    lo = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [i & lo, i >> s, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ np.uint64(k[0]), b & lo, (a >> s) ^ c[3] ^ np.uint64(k[1]), a & lo]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1).reshape(-1)[:n]


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    return torch.from_numpy(philox_words(n, seed, offset) >= np.uint64(round(p * 2.0 ** 32))).reshape(shape)


def ulp(v, dtype):
    bits, low = (10, -14) if dtype == torch.float16 else (23, -126)
    return 2.0 ** (torch.floor(torch.log2(v.abs().clamp_min(2.0 ** low))) - bits)


def assert_within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {err.numel()} beyond the bound, first at "
                           f"{bad.nonzero()[:3].tolist()}: got {got.double()[bad][:3].tolist()}, "
                           f"want {want[bad][:3].tolist()}, bound {bound.expand_as(err)[bad][:3].tolist()}")


def _norm64(v, rms, eps):
    mean = torch.zeros_like(v[..., :1]) if rms else v.mean(-1, keepdim=True)
    rstd = ((v - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    return (v - mean) * rstd, rstd, v.abs().amax(-1, keepdim=True) * rstd


def residual_norm64(x, f, weight=None, bias=None, post=False, post_weight=None, post_bias=None, gate=None,
                    rms=False, scale=1.0, eps=1e-5, keep=None, p=0.0, gx=None, gh=None, chain=None):
    """{name: (value, bound)} in float64 on the rounded inputs; gradients when
    gx / gh are given (the missing one counts as zero).

    `chain` None: bounds that also admit a backward pass from the rounded x_new
    and column sums of all rows one after the other.  A number: bounds for the
    unrounded x_new, with results rounded to nearest and at most `chain` additions
    on a term's way through a column sum."""
    dtype = x.dtype
    d = {n: t.double() for n, t in dict(x=x, f=f, w=weight, b=bias, pw=post_weight, pb=post_bias, gate=gate,
                                        gx=gx, gh=gh).items() if t is not None}
    one = torch.ones((), dtype=torch.float64)
    w, b, pw, pb, gt = d.get("w", one), d.get("b", 0 * one), d.get("pw", one), d.get("pb", 0 * one), d.get("gate", one)
    drop = one if keep is None else keep.double() / (1.0 - p) if p < 1 else torch.zeros_like(d["x"])
    u, m_u, c_u = d["f"], d["f"].abs(), 0.0
    if post:
        q, rq, aq = _norm64(d["f"], rms, eps)
        c_q = K * U32 * (1 + aq)
        u, m_u, c_u = q * pw + pb, (1 + q.abs()) * pw.abs() + pb.abs(), c_q
    x_new = scale * d["x"] + gt * drop * u
    m_x = abs(scale) * d["x"].abs() + (gt * drop).abs() * m_u
    e_x = (c_u + 8 * U32) * m_x                       # binary32 error of x_new
    n, rn, an = _norm64(x_new, rms, eps)
    # n moves with x_new's error, its own row sums and (in the backward pass) x_new's rounding
    c_n = K * U32 * (1 + an) + 2 * e_x.amax(-1, keepdim=True) * rn
    h = n * w + b
    out = {"x_new": (x_new, ulp(x_new, dtype) + e_x),
           "h": (h, ulp(h, dtype) + (c_n + 4 * U32) * ((1 + n.abs()) * w.abs() + b.abs()))}
    if gx is None and gh is None:
        return out
    zero = torch.zeros_like(x_new)
    vx, vh = d.get("gx", zero), d.get("gh", zero)
    c_b = c_n + (HALF_STEP[dtype] * an if chain is None else 0.0)  # n from the rounded x_new
    t = vh * w
    mean = (lambda v: torch.zeros_like(v[..., :1])) if rms else (lambda v: v.mean(-1, keepdim=True))
    both = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    g = vx + rn * (t - mean(t) - n * both(t * n))
    m_g = vx.abs() + rn * (t.abs() + (1 + n.abs()) * (both(t.abs()) + both((t * n).abs())))
    e_g = (c_b + K * U32) * 2 * m_g
    rows = x.numel() // x.shape[-1]
    dims = tuple(range(x.dim() - 1))

    def total(name, v, err, mag, over=dims, shape=None):
        s = v.sum(over, keepdim=shape is not None)
        e = (err + (rows + 64 if chain is None else chain) * U32 * mag).sum(over, keepdim=shape is not None)
        out[name] = (s, ulp(s, dtype) + e)

    out["x"] = (scale * g, ulp(scale * g, dtype) + abs(scale) * e_g)
    total("weight", vh * n, vh.abs() * c_b * (1 + n.abs()), (vh * n).abs())
    total("bias", vh, 0 * zero, vh.abs())
    e_u = (c_u + 8 * U32) * m_u * drop.abs()
    if gate is not None:
        v, e, m = g * drop * u, e_g * (drop * u).abs() + m_g * e_u, m_g * drop.abs() * m_u
        if gate.dim() == 1:
            total("gate", v, e, m)
        else:
            over = tuple(i for i in range(x.dim() - 1) if gate.shape[i] != x.shape[i])
            if over:
                total("gate", v, e, m, over, True)
            else:
                out["gate"] = (v, ulp(v, dtype) + e + 4 * U32 * m)
    gu, e_gu, m_gu = gt * drop * g, (gt * drop).abs() * (e_g + 4 * U32 * m_g), (gt * drop).abs() * m_g
    if post:
        total("post_weight", gu * q, e_gu * (1 + q.abs()) + m_gu * c_q * (1 + q.abs()), m_gu * (1 + q.abs()))
        total("post_bias", gu, e_gu, m_gu)
        t, e_t, m_t = gu * pw, e_gu * pw.abs(), m_gu * pw.abs()
        gu = rq * (t - mean(t) - q * both(t * q))
        spread = lambda v: v + (1 + q.abs()) * (both(v) + both(v * q.abs()))  # noqa: E731
        e_gu = rq * (spread(e_t) + 2 * (c_q + K * U32) * spread(m_t))
    out["f"] = (gu, ulp(gu, dtype) + e_gu)
    return out


def column_chain(rows, gate_rows=None):
    """Additions on a term's way through a column sum of `rows` rows of more than
    128 columns that one CTA holds: the rows of one of 148 or more row ranges, or of
    a gate row that a group takes whole, then the range's groups (up to 8), four to
    19 ranges per thread and 32 threads, and a product's rounding."""
    return max(-(-rows // 148), rows // gate_rows if gate_rows else 0) + 64


# Norm of the error over norm of the value.  Rounding a result is off by half a
# step at most, 2^-11 of the norm in binary16; binary32 errors of the terms, up to
# K half steps each with signs of their own, add sqrt(K) twice over (the
# statistics' and the sums'), 14 to 28 half steps: 32 in all.
NORM_ERROR = {torch.float16: 2.0 ** -11 + 32 * U32, torch.float32: 32 * U32}


def norm_error(got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-300))


def linear_ce64(x, w, target, bias=None, ignore=-100, reduction="mean", grad=None):
    """{name: (value, bound)} of the linear cross entropy and its gradients in
    float64 (on the tensors' device), from their rounded values.

    Bounds, from how the kernels compute:
    * a product sum over k terms in steps of 16 on the tensor cores, each step
      rounded (or cut) to binary32: (k / 16 + 16) 2^-23 of the terms' absolute
      sum; binary16 factors are exact, fp32 ones enter as two binary16 planes
      without the product of the low ones: three times the steps, and 4 * 2^-22
      of the terms' absolute sum, and 2^-39 of the largest values per term;
    * base-2 exponentials and logarithms: 2^-21 relative; the sums of
      exponentials: 32 in a row, then at most V / 2048 + 32 joins;
    * dz (softmax - onehot, at most 1) rounded to binary16 at 2^14 times its
      value: half a step or half the smallest subnormal, 2^-39; two planes
      keep 2^-22.
    """
    f16 = x.dtype == torch.float16
    X, W = x.double(), w.double()
    V, D = W.shape
    used = target != ignore
    X = torch.where(used[:, None], X, torch.zeros((), dtype=X.dtype, device=X.device))

    def product_error(k, mag, amax=0.0):
        e = (k * (1 if f16 else 3) / 16 + 16) * 2.0 ** -23 * mag
        return e if f16 else e + 4 * 2.0 ** -22 * mag + k * 2.0 ** -39 * amax

    z, mag = X @ W.T, X.abs() @ W.abs().T
    if bias is not None:
        z, mag = z + bias.double(), mag + bias.double().abs()
    xm, wm = float(X.abs().max()) if X.numel() else 0.0, float(W.abs().max())
    e_z = product_error(D, mag, xm * wm) + 2.0 ** -22 * z.abs()
    lse = torch.logsumexp(z, 1)
    at = torch.where(used, target, 0)[:, None]
    hit = z.gather(1, at)[:, 0]
    e_lse = e_z.amax(1) + 2.0 ** -20 + (64 + V / 2048) * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    rows = torch.where(used, lse - hit, 0.0)
    e_rows = torch.where(used, e_lse + (D / 64 + 12) * 2.0 ** -24 * mag.gather(1, at)[:, 0] + 2.0 ** -22 * (lse.abs() + hit.abs()), 0.0)
    count = int(used.sum())
    share = {"none": 1.0, "sum": 1.0, "mean": 1.0 / max(count, 1)}[reduction]
    if reduction == "none":
        out = {"loss": (rows, e_rows + ulp(rows, torch.float32))}
    else:
        total = rows.sum() * share
        out = {"loss": (total, e_rows.sum() * share + ulp(total, torch.float32))}
    if grad is None:
        return out
    g = torch.where(used, grad.double() * share, 0.0)
    gmax = float(g.abs().max()) if g.numel() else 0.0
    p = (z - lse[:, None]).exp()
    dz = p.clone()
    dz[torch.arange(len(dz), device=dz.device), at[:, 0]] -= 1.0
    e_dz = p * (e_z + e_lse[:, None] + 2.0 ** -20) + (2.0 ** -11 if f16 else 2.0 ** -22) * dz.abs() + 2.0 ** -22 * dz.abs()
    dz, e_dz = dz * g[:, None], e_dz * g.abs()[:, None] + torch.where(used, 2.0 ** -39 * gmax, 0.0)[:, None]
    for name, a, e, b, k in (("x", dz, e_dz, W, V), ("weight", dz.T, e_dz.T, X, len(X))):
        v, m = a @ b, a.abs() @ b.abs()
        out[name] = (v, ulp(v, x.dtype) + e @ b.abs() + product_error(k, m, gmax * float(b.abs().max()) if b.numel() else 0.0)
                     + 64 * 2.0 ** -24 * m)
    if bias is not None:
        s = dz.sum(0)
        out["bias"] = (s, ulp(s, x.dtype) + e_dz.sum(0) + (len(X) / 8 + 64) * 2.0 ** -24 * dz.abs().sum(0))
    return out
