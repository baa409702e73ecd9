"""Dropout and the residual norm against 64-bit references on the same rounded
inputs (tests/_train_helpers.py holds the references and derives the bounds),
their gradients against the formulas and against differences, and what they
refuse."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

torch_kunlun = pytest.importorskip("torch_kunlun")
kunlun = torch_kunlun.kunlun
from tests import _train_helpers as R  # noqa: E402
from torch_kunlun_b200 import _capi as C, ops  # noqa: E402

DEV = "kunlun"
F16, F32 = torch.float16, torch.float32


def rnd(shape, seed, dtype=F16, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + mean).to(dtype)


# ---- dropout ------------------------------------------------------------------------


def dropout_reference(x, p, seed, offset):
    keep = R.keep_mask(x.shape, p, seed, offset)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=F32)
    return torch.where(keep, x.float() * scale, torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (9,), (17, 5), (1, 768), (37, 1023), (515, 1024)])
def test_dropout_is_exact(shape, dtype):
    x = rnd(shape, 1, dtype)
    for p, seed, offset in [(0.1, 0, 0), (0.5, 0xFEDCBA9876543210, 2 ** 64 - 1), (0.0, 7, 3), (1.0, 7, 3), (0.999999, 5, 1 << 32)]:
        y = ops.dropout(x.to(DEV), p, seed, offset).cpu()
        assert torch.equal(y, dropout_reference(x, p, seed, offset)), (p, seed, offset)


def test_dropout_drops_non_finite_values_and_keeps_them():
    x = torch.full((4096,), float("inf"), dtype=F16)
    x[1::2] = float("nan")
    y = ops.dropout(x.to(DEV), 0.5, 11).cpu()
    keep = R.keep_mask((4096,), 0.5, 11, 0)
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum()), dtype=F16))
    assert not torch.isfinite(y[keep]).any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_dropout_off_boundary_and_strided_inputs(dtype):
    base = rnd((64, 70), 2, dtype).to(DEV)
    flat = base.view(-1)[3:3 + 1001]  # contiguous, off a 16-byte boundary
    assert torch.equal(ops.dropout(flat, 0.3, 5).cpu(), dropout_reference(flat.cpu(), 0.3, 5, 0))
    t = base.t()                      # element order is the view's own
    assert torch.equal(ops.dropout(t, 0.3, 5).cpu(), dropout_reference(t.cpu(), 0.3, 5, 0))


def test_dropout_gradient_uses_the_same_mask():
    x, g = rnd((33, 129), 3), rnd((33, 129), 4)
    xd = x.to(DEV).requires_grad_()
    y = ops.dropout(xd, 0.25, 9, 2)
    y.backward(g.to(DEV))
    assert torch.equal(y.detach().cpu(), dropout_reference(x, 0.25, 9, 2))
    assert torch.equal(xd.grad.cpu(), dropout_reference(g, 0.25, 9, 2))


def test_dropout_empty():
    assert ops.dropout(torch.empty(0, 5, dtype=F16).to(DEV), 0.5, 1).shape == (0, 5)


@pytest.mark.parametrize("n", [(1 << 32) + 4093, (1 << 34) + 4093])
def test_dropout_large_index_in_place(n):
    # element indices past 2^32, and past 2^34, where the block counter has a high word
    if torch.cuda.mem_get_info()[0] < 2 * n + (8 << 30):
        pytest.skip("needs the memory of one large tensor")
    x = torch.ones(n, dtype=F16, device="cuda")
    torch.cuda.synchronize()
    C.check(C.lib().tk_dropout(0, x.data_ptr(), x.data_ptr(), n, 0.5, 21, 4, None), "tk_dropout")
    torch.cuda.synchronize()
    tail, first = x[-4096:].cpu(), n - 4096
    del x
    torch.cuda.empty_cache()
    words = np.concatenate([_block(i, 21, 4) for i in range(first // 4, n // 4 + 1)])[first % 4:][:4096]
    assert torch.equal(tail, torch.from_numpy(np.where(words >= 1 << 31, 2.0, 0.0)).to(F16))


def _block(i, seed, offset):
    c, k = [i & 0xFFFFFFFF, i >> 32, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.array(c, dtype=np.uint64)


def test_dropout_rate_and_independence():
    n = 1 << 20
    one = torch.ones(n, dtype=F32).to(DEV)
    a = ops.dropout(one, 0.1, 1, 0).cpu() > 0
    b = ops.dropout(one, 0.1, 1, 1).cpu() > 0
    # binomial: 6 standard deviations of n trials at 0.9 and 0.81
    assert abs(a.double().mean() - 0.9) < 6 * (0.09 / n) ** 0.5
    assert abs((a & b).double().mean() - 0.81) < 6 * (0.81 * 0.19 / n) ** 0.5


# ---- residual norm ---------------------------------------------------------------------


def norm_inputs(shape, dtype, kind, post, gate, seed, with_params=True):
    d = shape[-1]
    t = {"x": rnd(shape, seed, dtype, 1.0, 0.5), "f": rnd(shape, seed + 1, dtype, 0.7)}
    if with_params:
        t["weight"] = rnd((d,), seed + 2, dtype, 0.1, 1.0)
        if kind == "layer":
            t["bias"] = rnd((d,), seed + 3, dtype, 0.1)
        if post:
            t["post_weight"] = rnd((d,), seed + 4, dtype, 0.1, 1.0)
            if kind == "layer":
                t["post_bias"] = rnd((d,), seed + 5, dtype, 0.1)
    shapes = {"none": None, "channel": (d,), "sample": shape[:1] + (1,) * (len(shape) - 2) + (d,), "token": shape}[gate]
    if shapes:
        t["gate"] = rnd(shapes, seed + 6, dtype, 0.3, 0.5)
    return t


def run_norm(t, kind, post, scale, p, gx=None, gh=None, seed=77, offset=5):
    dev = {k: v.to(DEV).requires_grad_(gx is not None or gh is not None) for k, v in t.items()}
    kw = {k: dev[k] for k in ("weight", "bias", "post_weight", "post_bias", "gate") if k in dev}
    x_new, h = ops.residual_norm(dev["x"], dev["f"], norm=kind, post_norm=post, residual_scale=scale, p=p, seed=seed, offset=offset, **kw)
    out = {"x_new": x_new, "h": h}
    ends = [(o, g.to(DEV)) for o, g in ((x_new, gx), (h, gh)) if g is not None]
    if ends:
        grads = torch.autograd.grad([e[0] for e in ends], list(dev.values()), [e[1] for e in ends])
        out.update(zip(dev, grads))
    return {k: v.detach().cpu() for k, v in out.items()}


def check_norm(shape, dtype, kind, post, gate, scale=1.0, p=0.0, grads="both", seed=0, with_params=True, t=None):
    t = t or norm_inputs(shape, dtype, kind, post, gate, seed, with_params)
    gx = rnd(shape, seed + 8, dtype) if grads in ("both", "x_new") else None
    gh = rnd(shape, seed + 9, dtype) if grads in ("both", "h") else None
    got = run_norm(t, kind, post, scale, p, gx, gh)
    keep = R.keep_mask(shape, p, 77, 5) if p > 0 else None
    want = R.residual_norm64(t["x"], t["f"], t.get("weight"), t.get("bias"), post, t.get("post_weight"), t.get("post_bias"),
                             t.get("gate"), kind == "rms", scale, 1e-5, keep, p, gx, gh)
    for k, v in got.items():
        value, bound = want[k]
        R.assert_within(v, value.reshape(v.shape), bound.expand_as(value).reshape(v.shape), f"{k} {shape} {dtype} {kind}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 7), (1, 5, 8), (3, 2, 33), (4, 1, 768), (3, 37, 768), (5, 31, 1000), (2, 130, 257), (3, 50, 256),
                                   (2, 9, 1536), (2, 11, 2048), (7, 33, 1151), (2, 5, 4096)])
@pytest.mark.parametrize("kind,post,gate,p", [("layer", False, "none", 0.0), ("layer", False, "none", 0.1), ("layer", True, "sample", 0.1),
                                              ("rms", True, "channel", 0.0), ("rms", False, "token", 0.5)])
def test_residual_norm(shape, dtype, kind, post, gate, p):
    check_norm(shape, dtype, kind, post, gate, 1.25 if post else 1.0, p, seed=sum(shape))


@pytest.mark.parametrize("dtype,cols", [(F16, 8192), (F16, 8200), (F16, 16384), (F16, 20001), (F16, 32768), (F32, 4104), (F32, 8192), (F32, 9999), (F32, 32768)])
@pytest.mark.parametrize("kind,post,gate", [("layer", True, "channel"), ("rms", False, "none")])
def test_residual_norm_wide_rows(dtype, cols, kind, post, gate):
    check_norm((2, 3, cols), dtype, kind, post, gate, p=0.1, seed=cols)


def test_residual_norm_many_rows_and_gate_segments():
    # more rows than resident groups; gate rows cut by the row ranges at every offset
    check_norm((3, 4001, 256), F16, "layer", True, "sample", p=0.1)
    check_norm((811, 13, 96), F32, "rms", False, "sample")
    check_norm((1, 9000, 64), F16, "rms", True, "channel")
    check_norm((2, 1500, 4096), F16, "rms", True, "sample", seed=3)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("cols", [1, 2, 3, 7, 8, 9, 16, 17, 24, 31, 40, 63, 64, 65, 100, 104, 120, 127, 128, 129])
@pytest.mark.parametrize("kind,post,gate,p", [("layer", False, "none", 0.1), ("rms", True, "sample", 0.2), ("layer", True, "token", 0.0)])
def test_residual_norm_narrow_rows(cols, dtype, kind, post, gate, p):
    # several rows to a warp; row counts that leave lanes of the last warp without one
    check_norm((3, 67, cols), dtype, kind, post, gate, p=p, seed=cols)
    check_norm((1, 1, cols), dtype, kind, post, gate, p=p, seed=cols + 1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(50, 3, 64), (301, 2, 8), (3001, 2, 5), (40, 5, 63), (33, 7, 256), (700, 4, 200), (2, 2, 1000), (9, 20, 129), (5000, 6, 16)])
@pytest.mark.parametrize("post,p", [(False, 0.0), (True, 0.1)])
def test_residual_norm_short_gate_rows(shape, dtype, post, p):
    # groups of a block that take whole gate rows, the last block's with fewer than the others
    check_norm(shape, dtype, "layer", post, "sample", p=p, seed=shape[0])


def test_residual_norm_gate_over_two_leading_dimensions():
    t = norm_inputs((3, 4, 5, 40), F32, "layer", True, "none", 2)
    t["gate"] = rnd((3, 4, 1, 40), 8, F32)
    check_norm((3, 4, 5, 40), F32, "layer", True, "none", p=0.2, t=t)


@pytest.mark.parametrize("grads", ["x_new", "h"])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_residual_norm_one_output_used(grads, dtype):
    check_norm((4, 19, 320), dtype, "layer", True, "channel", 0.5, 0.3, grads=grads)
    check_norm((4, 19, 321), dtype, "rms", False, "none", grads=grads, with_params=False)


def test_residual_norm_everything_dropped_and_zero_rows():
    check_norm((2, 6, 128), F16, "layer", False, "channel", p=1.0)
    for shape in [(0, 4, 16), (3, 0, 16)]:
        t = norm_inputs(shape, F16, "layer", True, "channel", 1)
        got = run_norm(t, "layer", True, 1.0, 0.1, torch.zeros(shape, dtype=F16), torch.zeros(shape, dtype=F16))
        assert got["h"].shape == shape and got["x"].shape == shape
        assert not got["weight"].any() and not got["gate"].any()


def test_residual_norm_constant_and_offset_rows():
    # a row of equal values normalises to the bias; a large mean costs no variance
    x = torch.full((2, 4, 64), 3.0, dtype=F32)
    t = {"x": x, "f": torch.zeros_like(x), "bias": rnd((64,), 1, F32)}
    got = run_norm(t, "layer", False, 1.0, 0.0)
    assert torch.equal(got["h"], t["bias"].expand(2, 4, 64))
    big = {"x": rnd((2, 4, 500), 2, F32, 1.0, 1000.0), "f": rnd((2, 4, 500), 3, F32)}
    check_norm((2, 4, 500), F32, "layer", False, "none", t=big)


def test_residual_norm_strided_and_misaligned_inputs():
    base = rnd((6, 4, 96), 5, F16)
    t = norm_inputs((4, 6, 96), F16, "layer", True, "channel", 6)
    t["x"] = base.transpose(0, 1)
    dev = base.to(DEV).transpose(0, 1)
    w = torch.empty(97, dtype=F16, device=DEV)
    w[1:].copy_(t["weight"].to(DEV))  # off a 16-byte boundary
    kw = {k: t[k].to(DEV) for k in ("bias", "post_weight", "post_bias", "gate")}
    x_new, h = ops.residual_norm(dev, t["f"].to(DEV), w[1:], post_norm=True, **kw)
    want = R.residual_norm64(t["x"], t["f"], t["weight"], t["bias"], True, t["post_weight"], t["post_bias"], t["gate"])
    R.assert_within(x_new.cpu(), *want["x_new"], "x_new")
    R.assert_within(h.cpu(), *want["h"], "h")


def test_residual_norm_vectors_shared_inputs_and_expanded_gates():
    # one row without leading dimensions
    t = {"x": rnd((70,), 1, F32), "f": rnd((70,), 2, F32), "weight": rnd((70,), 3, F32), "gate": rnd((70,), 4, F32)}
    gx, gh = rnd((70,), 5, F32), rnd((70,), 6, F32)
    got = run_norm(t, "layer", True, 1.0, 0.2, gx, gh)
    one = lambda v: v[None]  # noqa: E731
    want = R.residual_norm64(one(t["x"]), one(t["f"]), t["weight"], None, True, None, None, t["gate"], False, 1.0, 1e-5,
                             R.keep_mask((1, 70), 0.2, 77, 5), 0.2, one(gx), one(gh))
    for k, v in got.items():
        R.assert_within(v, want[k][0].reshape(v.shape), want[k][1].expand_as(want[k][0]).reshape(v.shape), k)
    # x and f one tensor: its gradient is the sum of both
    x = rnd((3, 4, 32), 7, F32)
    xd = x.to(DEV).requires_grad_()
    y, _ = ops.residual_norm(xd, xd, residual_scale=2.0)
    y.backward(torch.ones(3, 4, 32).to(DEV))
    assert torch.equal(xd.grad.cpu(), torch.full((3, 4, 32), 3.0))
    # a gate for all samples, with its leading ones
    check_norm((3, 4, 32), F32, "rms", False, "none", t={"x": x, "f": rnd((3, 4, 32), 8, F32), "gate": rnd((1, 1, 32), 9, F32)})


def test_train_ops_on_two_streams_at_once():
    t = norm_inputs((4, 500, 512), F16, "rms", True, "sample", 5)
    g = rnd((4, 500, 512), 6)
    x, w = rnd((600, 128), 7), rnd((3000, 128), 8, F16, 0.1)
    target = torch.randint(0, 3000, (600,), generator=torch.Generator().manual_seed(1)).to(DEV)

    def both():
        dev = {k: v.to(DEV).requires_grad_() for k, v in t.items()}
        xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        return dev, xd, wd

    def work(dev, xd, wd):
        y, h = ops.residual_norm(dev["x"], dev["f"], dev["weight"], norm="rms", post_norm=True, post_weight=dev["post_weight"], gate=dev["gate"], p=0.1, seed=3)
        loss = ops.linear_cross_entropy(xd, wd, target)
        return [y, h, loss] + list(torch.autograd.grad([y, h, loss], list(dev.values()) + [xd, wd], [gd, gd, one]))

    gd, one = g.to(DEV), torch.tensor(64.0).to(DEV)
    inputs = [both() for _ in range(4)]
    kunlun.synchronize()
    first = [v.detach().cpu() for v in work(*inputs[0])]
    streams = [kunlun.Stream() for _ in range(2)]
    results = []
    for i in range(6):
        with kunlun.stream(streams[i % 2]):
            results.append(work(*inputs[1 + i % 3]))
    for s in streams:
        s.synchronize()
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b.detach().cpu())


def test_residual_norm_non_finite_rows_stay_in_their_rows():
    x, f = rnd((1, 6, 800), 1), rnd((1, 6, 800), 2)
    x[0, 2, 5] = float("inf")
    f[0, 4, 7] = float("nan")
    x_new, h = ops.residual_norm(x.to(DEV), f.to(DEV), post_norm=True)
    h = h.cpu()
    assert torch.isfinite(h[0, [0, 1, 3, 5]]).all()
    assert torch.isnan(h[0, 2, 5]) and torch.isnan(h[0, 4]).all()


def test_residual_norm_gradient_against_differences():
    # central differences of the 64-bit forward in a random direction, per input
    shape = (2, 3, 40)
    t = norm_inputs(shape, F32, "layer", True, "sample", 4)
    gx, gh = rnd(shape, 8, F32), rnd(shape, 9, F32)
    got = run_norm(t, "layer", True, 0.8, 0.2, gx, gh)
    keep = R.keep_mask(shape, 0.2, 77, 5)

    def value(u):
        o = R.residual_norm64(u["x"], u["f"], u["weight"], u["bias"], True, u["post_weight"], u["post_bias"], u["gate"],
                              False, 0.8, 1e-5, keep, 0.2)
        return float((o["x_new"][0] * gx.double()).sum() + (o["h"][0] * gh.double()).sum())

    wide = {k: v.double() for k, v in t.items()}
    R.HALF_STEP.setdefault(torch.float64, 0.0)
    for k in t:
        v = torch.randn(t[k].shape, generator=torch.Generator().manual_seed(31), dtype=torch.float64)
        step = 1e-5
        slope = (value({**wide, k: wide[k] + step * v}) - value({**wide, k: wide[k] - step * v})) / (2 * step)
        have = float((got[k].double() * v).sum())
        # differences: step^2 truncation and 2^-52 / step cancellation, far below
        # the binary32 error of the gradient, 200 * 2^-24 of its terms' sum
        assert abs(have - slope) <= 200 * R.U32 * float((got[k].double() * v).abs().sum()) + 1e-6, k


def test_residual_norm_is_deterministic_and_stream_ordered():
    t = norm_inputs((8, 300, 768), F16, "layer", False, "channel", 12)
    g = rnd((8, 300, 768), 13)
    first = run_norm(t, "layer", False, 1.0, 0.1, g, g)
    s = kunlun.Stream()
    for _ in range(3):
        with kunlun.stream(s):
            again = run_norm(t, "layer", False, 1.0, 0.1, g, g)
        s.synchronize()
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_train_op_refusals():
    x = rnd((4, 16), 1).to(DEV)
    w = rnd((16,), 2).to(DEV)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(RuntimeError, match="p must be in"):
            ops.dropout(x, p, 1)
        with pytest.raises(RuntimeError, match="p must be in"):
            ops.residual_norm(x, x, p=p)
    with pytest.raises(ValueError, match="seed"):
        ops.dropout(x, 0.1, -1)
    with pytest.raises(ValueError, match="offset"):
        ops.dropout(x, 0.1, 1, 1 << 64)
    with pytest.raises(RuntimeError, match="float16/float32"):
        ops.dropout(torch.zeros(4, dtype=torch.int64).to(DEV), 0.1, 1)
    with pytest.raises(RuntimeError, match="kunlun tensors"):
        ops.dropout(torch.zeros(4), 0.1, 1)
    with pytest.raises(ValueError, match="norm must be"):
        ops.residual_norm(x, x, norm="batch")
    with pytest.raises(RuntimeError, match="f has shape"):
        ops.residual_norm(x, x[:2])
    with pytest.raises(RuntimeError, match="must be"):
        ops.residual_norm(x, x, w.float())
    with pytest.raises(RuntimeError, match="weights and biases"):
        ops.residual_norm(x, x, w[:8])
    with pytest.raises(RuntimeError, match="need post_norm"):
        ops.residual_norm(x, x, w, post_weight=w)
    with pytest.raises(RuntimeError, match="gate must be"):
        ops.residual_norm(x, x, w, gate=x[:, :8])
    with pytest.raises(RuntimeError, match="gate must be"):
        ops.residual_norm(x.view(2, 2, 16), x.view(2, 2, 16), gate=x[:2].view(1, 2, 16))
    with pytest.raises(RuntimeError, match="32768"):
        ops.residual_norm(torch.zeros(1, 32776, dtype=F16).to(DEV), torch.zeros(1, 32776, dtype=F16).to(DEV))
    leaf = rnd((4, 16), 3).to(DEV).requires_grad_()
    y, _ = ops.residual_norm(leaf, x)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y, leaf, torch.ones(4, 16, dtype=F16).to(DEV), create_graph=True)


@pytest.mark.parametrize("shape", [(0, 4, 16), (3, 0, 16), (0, 16), (0, 0, 8)])
@pytest.mark.parametrize("gate", ["sample", "token"])
def test_residual_norm_empty_batch_with_a_gate_for_each_sample(shape, gate):
    t = norm_inputs(shape, F16, "layer", True, gate, 1)
    none = torch.zeros(shape, dtype=F16)
    got = run_norm(t, "layer", True, 1.0, 0.1, none, none)
    assert got["h"].shape == got["x"].shape == shape and got["gate"].shape == t["gate"].shape
    assert not got["weight"].any() and not got["gate"].any()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", [lambda x, y: ops.dropout(x, 0.1, 1), lambda x, y: ops.residual_norm(x, y)[1], lambda x, y: ops.residual_norm(y, x)[1],
                                  lambda x, y: ops.residual_norm(y, y, x[0])[1], lambda x, y: ops.residual_norm(y, y, gate=x)[1],
                                  lambda x, y: ops.linear_cross_entropy(x, y, TARGET.to(DEV)), lambda x, y: ops.linear_cross_entropy(y, x, TARGET.to(DEV)),
                                  lambda x, y: ops.linear_cross_entropy(y, y, TARGET.to(DEV), x[0, :6])])
def test_train_ops_refuse_forward_mode(call, grad):
    """A dual tensor is refused, whether it also requires a gradient or not: its
    tangent would be lost."""
    x, y = rnd((6, 16), 1).to(DEV).requires_grad_(grad), rnd((6, 16), 2).to(DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(dual, y)
    call(x, y)


TARGET = torch.arange(6)


@pytest.mark.parametrize("spoil,match", [(lambda v: v.cpu(), "expected"), (lambda v: v.to(F32) if v.dtype == F16 else v.to(F16), "expected"),
                                         (lambda v: v[:1], "expected")])
@pytest.mark.parametrize("call", ["norm", "loss"])
def test_train_ops_refuse_other_saved_tensors(call, spoil, match):
    """What saved-tensor hooks hand back is looked at before its pointer is used."""
    x = rnd((2, 3, 16), 1).to(DEV).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: spoil(v.detach())):
        if call == "norm":
            y = ops.residual_norm(x, x.detach(), rnd((16,), 2).to(DEV), post_norm=True, gate=rnd((2, 1, 16), 3).to(DEV))[1].float().sum()
        else:
            y = ops.linear_cross_entropy(x, rnd((9, 16), 4).to(DEV), torch.zeros(2, 3, dtype=torch.int64).to(DEV), rnd((9,), 5).to(DEV))
    with pytest.raises(RuntimeError, match=match):
        y.backward()


@pytest.mark.parametrize("kind,post,gate", [("layer", True, "sample"), ("rms", False, "none")])
def test_residual_norm_saved_tensors_come_back_strided_or_from_the_host(kind, post, gate):
    shape = (4, 19, 96)
    t = norm_inputs(shape, F16, kind, post, gate, 3)
    gx, gh = rnd(shape, 8), rnd(shape, 9)
    want = run_norm(t, kind, post, 1.0, 0.2, gx, gh)

    def strided(v):
        return v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() > 1 else v.clone()

    def off(v):
        b = torch.empty(v.numel() + 8, dtype=v.dtype, device=DEV)
        b[1:1 + v.numel()].copy_(v.reshape(-1))
        return b[1:1 + v.numel()].view(v.shape) if v.dtype == F16 else v

    for pack, unpack in ((lambda v: v.cpu(), lambda v: v.to(DEV)), (lambda v: v, strided), (lambda v: v, off)):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got = run_norm(t, kind, post, 1.0, 0.2, gx, gh)
        for k in want:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("call", ["norm with a channel gate", "norm with a sample gate", "norm with a token gate", "loss"])
def test_train_ops_form_the_gradients_that_are_asked_for(call):
    """autograd.grad for some of the inputs that require gradients: the others'
    are not even allocated, and those asked for are the same."""
    if call != "loss":
        t = norm_inputs((2, 512, 4096), F16, "layer", True, call.split()[3], 1)
        g = rnd((2, 512, 4096), 9).to(DEV)
        large = "f"
    else:
        t = {"x": rnd((8, 256), 1), "weight": rnd((60000, 256), 2, F16, 0.1), "bias": rnd((60000,), 3)}
        target, g = torch.arange(8).to(DEV), torch.tensor(64.0).to(DEV)
        large = "weight"

    def peak(names):
        dev = {k: v.to(DEV).requires_grad_() for k, v in t.items()}
        if call != "loss":
            y = ops.residual_norm(dev["x"], dev["f"], post_norm=True, p=0.1, seed=5, **{k: dev[k] for k in t if k not in ("x", "f")})[1]
        else:
            y = ops.linear_cross_entropy(dev["x"], dev["weight"], target, dev["bias"])
        kunlun.synchronize()
        kunlun.reset_peak_memory_stats()
        before = kunlun.memory_allocated()
        grads = torch.autograd.grad(y, [dev[k] for k in names], g)
        kunlun.synchronize()
        return kunlun.max_memory_allocated() - before, dict(zip(names, (v.cpu() for v in grads)))

    whole, every = peak(list(t))
    for names in [[k] for k in t if k != large] + [[k for k in t if k != large]]:
        part, some = peak(names)
        assert whole - part >= t[large].numel() * 2, names
        for k in names:
            assert torch.equal(some[k], every[k]), k


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(3, 7, 24), (2, 9, 96), (5, 31, 256), (3, 40, 1000), (2, 5, 4096), (2, 3, 9000), (1, 2, 20000)])
@pytest.mark.parametrize("kind,post,gate,p", [("layer", True, "sample", 0.1), ("rms", False, "none", 0.0), ("rms", True, "channel", 0.3), ("layer", False, "token", 0.0)])
def test_residual_norm_gradients_of_misaligned_tensors(shape, dtype, kind, post, gate, p):
    """Every tensor off a 16-byte boundary, each by an offset of its own, at widths
    that vectors would fit, against the 64-bit values; nothing beside a result is
    written."""
    t = norm_inputs(shape, dtype, kind, post, gate, sum(shape))
    gx, gh = rnd(shape, 8, dtype), rnd(shape, 9, dtype)
    hold = []

    def off(v, k):
        b = torch.full((v.numel() + 8,), 7.0, dtype=v.dtype, device="cuda")
        b[k:k + v.numel()] = v.reshape(-1).cuda()
        hold.append((b, k, v.numel()))
        return hold[-1][0][k:k + v.numel()].data_ptr()

    d = shape[-1]
    rows = t["x"].numel() // d
    step = 8 if dtype == F16 else 4  # elements of 16 bytes
    g = C.ResidualNormGradDesc()
    f = g.fwd
    f.dtype, f.norm, f.rows, f.cols, f.post_norm = int(dtype == F32), int(kind == "rms"), rows, d, int(post)
    f.residual_scale, f.eps, f.p, f.seed, f.offset = 0.75, 1e-5, p, 77, 5
    for i, k in enumerate(t):
        setattr(f, k, off(t[k], 1 + i % (step - 1)))
    f.gate_rows = t["gate"].numel() // d if "gate" in t else 0
    inputs = len(hold)
    names = ["x_new", "h"] + list(t)
    where = {}
    for i, k in enumerate(names):
        like = t[k] if k in t else t["x"]
        where[k] = (len(hold), like.shape)
        at = off(torch.zeros_like(like), 1 + (2 * i + 1) % (step - 1))
        if k in ("x_new", "h"):
            setattr(f, k, at)
        else:
            setattr(g, "d" + k, at)
    g.grad_x_new, g.grad_h = off(gx, 3), off(gh, 2)
    stats = torch.zeros(rows, 4, device="cuda")
    f.stats = stats.data_ptr()
    L = C.lib()
    size = L.tk_residual_norm_backward_workspace_size(C.ctypes.byref(g))
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    C.check(L.tk_residual_norm(C.ctypes.byref(f), None), "tk_residual_norm")
    C.check(L.tk_residual_norm_backward(C.ctypes.byref(g), ws.data_ptr(), size, None), "tk_residual_norm_backward")
    torch.cuda.synchronize()
    want = R.residual_norm64(t["x"], t["f"], t.get("weight"), t.get("bias"), post, t.get("post_weight"), t.get("post_bias"), t.get("gate"),
                             kind == "rms", 0.75, 1e-5, R.keep_mask(shape, p, 77, 5) if p > 0 else None, p, gx, gh)
    for k, (i, s) in where.items():
        b, at, n = hold[i]
        value, bound = want[k]
        got = b.cpu()
        R.assert_within(got[at:at + n].view(s), value.reshape(s), bound.expand_as(value).reshape(s), k)
        assert (got[:at] == 7).all() and (got[at + n:] == 7).all(), k
    assert inputs == len(t)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", [(3, 37, 768), (1, 3000, 256), (4, 500, 1000), (7, 33, 1151), (2, 1500, 4096), (16, 301, 136), (600, 5, 200)])
@pytest.mark.parametrize("kind,post,gate,p", [("layer", False, "none", 0.0), ("layer", True, "channel", 0.1), ("rms", True, "sample", 0.0), ("rms", False, "token", 0.1)])
def test_residual_norm_gradients_within_tight_bounds(shape, dtype, kind, post, gate, p):
    """Bounds that an x_new rounded to binary16, or a missing or wrong term, does
    not meet (test_train_ops_cpu.py): element by element and in norm."""
    t = norm_inputs(shape, dtype, kind, post, gate, sum(shape))
    gx, gh = rnd(shape, 8, dtype), rnd(shape, 9, dtype)
    got = run_norm(t, kind, post, 1.25, p, gx, gh)
    rows = t["x"].numel() // shape[-1]
    want = R.residual_norm64(t["x"], t["f"], t.get("weight"), t.get("bias"), post, t.get("post_weight"), t.get("post_bias"), t.get("gate"),
                             kind == "rms", 1.25, 1e-5, R.keep_mask(shape, p, 77, 5) if p > 0 else None, p, gx, gh,
                             chain=R.column_chain(rows, shape[0] if gate == "sample" else None))
    for k, v in got.items():
        value, bound = want[k]
        R.assert_within(v, value.reshape(v.shape), bound.expand_as(value).reshape(v.shape), f"{k} {shape} {dtype} {kind}")
        assert R.norm_error(v, value.reshape(v.shape)) <= R.NORM_ERROR[dtype], k


def test_train_ops_captured_with_their_backward_passes():
    """Two steps captured through the public calls, forward and backward, replayed
    in turn on new values in the same inputs, against ordinary calls."""
    def values(seed):
        return [rnd((4, 16, 64), seed), rnd((4, 16, 64), seed + 1), rnd((64,), seed + 2, F16, 0.1, 1.0), rnd((1000, 64), seed + 3, F16, 0.3)]

    def step(x, f, w, head, target, offset):
        y, h = ops.residual_norm(x, f, w, post_norm=True, p=0.1, seed=3, offset=offset)
        loss = ops.linear_cross_entropy(ops.dropout(h, 0.1, 5, offset), head, target)
        return [y.detach(), loss.detach()] + list(torch.autograd.grad([y, loss], [x, f, w, head], [torch.ones_like(y), one]))

    one = torch.tensor(64.0).to(DEV)
    target = torch.randint(-1, 1000, (4, 16), generator=torch.Generator().manual_seed(2))
    target = torch.where(target < 0, -100, target).to(DEV)
    s = kunlun.Stream()
    graphs = []
    for k in range(2):
        leaves = [v.to(DEV).requires_grad_() for v in values(10 * k)]
        kunlun.synchronize()
        with kunlun.stream(s):
            step(*leaves, target, k)
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(s.stream_id)):
                out = step(*leaves, target, k)
        graphs.append((graph, leaves, out))
    torch.cuda.synchronize()
    for seed in (100, 200):
        for k, (graph, leaves, out) in enumerate(graphs):
            with torch.no_grad():
                for leaf, v in zip(leaves, values(seed + 50 * k)):
                    leaf.copy_(v.to(DEV))
        kunlun.synchronize()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for k, (_, leaves, out) in enumerate(graphs):
            want = step(*[v.to(DEV).requires_grad_() for v in values(seed + 50 * k)], target, k)
            for a, b in zip(out, want):
                assert torch.equal(a.cpu(), b.cpu())
