"""The linear cross entropy against its 64-bit definition on the same rounded
inputs (tests/_train_helpers.py derives the bounds), its gradients, masks and
refusals, and the training operators in one step."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

torch_kunlun = pytest.importorskip("torch_kunlun")
kunlun = torch_kunlun.kunlun
from tests import _train_helpers as R  # noqa: E402
from torch_kunlun_b200 import _capi, ops  # noqa: E402

DEV = "kunlun"
F16, F32 = torch.float16, torch.float32


def rnd(shape, seed, dtype=F16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def ce_inputs(n, d, v, dtype, bias, ignored=0, seed=0):
    g = torch.Generator().manual_seed(seed + 50)
    t = {"x": rnd((n, d), seed, dtype), "weight": rnd((v, d), seed + 1, dtype, 2.0 / d ** 0.5)}
    if bias:
        t["bias"] = rnd((v,), seed + 2, dtype, 0.3)
    target = torch.randint(0, v, (n,), generator=g)
    target[torch.randperm(n, generator=g)[:ignored]] = -100
    return t, target


def run_ce(t, target, reduction, grad=None, ignore=-100, wanted=("x", "weight", "bias")):
    dev = {k: v.to(DEV).requires_grad_(grad is not None and k in wanted) for k, v in t.items()}
    loss = ops.linear_cross_entropy(dev["x"], dev["weight"], target.to(DEV), dev.get("bias"), ignore, reduction)
    out = {"loss": loss}
    if grad is not None:
        names = [k for k in t if k in wanted]
        out.update(zip(names, torch.autograd.grad(loss, [dev[k] for k in names], grad.to(DEV))))
    assert _capi.device_error(0) == 0
    return {k: v.detach().cpu() for k, v in out.items()}


def check_ce(t, target, reduction, grad=None, ignore=-100, wanted=("x", "weight", "bias")):
    got = run_ce(t, target, reduction, grad, ignore, wanted)
    cu = {k: v.cuda() for k, v in t.items()}
    want = R.linear_ce64(cu["x"], cu["weight"], target.cuda(), cu.get("bias"), ignore, reduction,
                         None if grad is None else grad.cuda())
    for k, v in got.items():
        value, bound = want[k]
        R.assert_within(v, value.cpu(), bound.cpu(), f"{k} {tuple(t['x'].shape)} {tuple(t['weight'].shape)} {t['x'].dtype} {reduction}")
    return got


def loss_grad(n, reduction, seed=0):
    if reduction == "none":
        return torch.randn(n, generator=torch.Generator().manual_seed(seed + 7))
    return torch.tensor(256.0 if reduction == "mean" else 0.75)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,d,v", [(1, 1, 1), (1, 8, 2), (3, 7, 5), (5, 64, 257), (16, 16, 128), (128, 256, 256), (130, 128, 300), (129, 768, 1000),
                                   (257, 100, 1031), (300, 72, 5000), (64, 1024, 10007), (500, 31, 77), (5000, 96, 40), (1000, 264, 2560)])
@pytest.mark.parametrize("reduction,bias", [("mean", False), ("none", True)])
def test_linear_ce(n, d, v, dtype, reduction, bias):
    t, target = ce_inputs(n, d, v, dtype, bias, seed=n + d + v)
    check_ce(t, target, reduction, loss_grad(n, reduction))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,ignored", [(1, 1), (40, 39), (300, 0), (300, 172), (300, 300), (2000, 1700)])
def test_linear_ce_ignored_rows(n, ignored, dtype):
    for reduction in ("none", "sum"):
        t, target = ce_inputs(n, 80, 700, dtype, True, ignored, seed=n + ignored)
        got = check_ce(t, target, reduction, loss_grad(n, reduction))
        if reduction == "none":
            assert not got["loss"][target == -100].any()
        assert not got["x"][target == -100].any()


def test_linear_ce_without_any_target():
    t, _ = ce_inputs(9, 16, 30, F16, True)
    target = torch.full((9,), -100)
    got = run_ce(t, target, "mean", torch.tensor(1.0))
    assert torch.isnan(got["loss"])
    assert not got["x"].any() and not got["weight"].any() and not got["bias"].any()
    assert run_ce(t, target, "sum")["loss"] == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_ce_non_finite_ignored_rows_do_not_matter(dtype):
    t, target = ce_inputs(150, 96, 500, dtype, False, 40, seed=3)
    clean = run_ce(t, target, "mean", torch.tensor(64.0))
    off = (target == -100).nonzero()[:, 0]
    t["x"][off[0]] = float("nan")
    t["x"][off[1]] = float("inf")
    t["x"][off[2]] = torch.finfo(dtype).min
    again = run_ce(t, target, "mean", torch.tensor(64.0))
    for k in clean:
        assert torch.equal(clean[k], again[k]), k


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_ce_non_finite_row_stays_in_its_row(dtype):
    t, target = ce_inputs(140, 64, 300, dtype, False, seed=4)
    t["x"][17, 3] = float("nan")
    got = run_ce(t, target, "none", loss_grad(140, "none"))
    assert torch.isnan(got["loss"][17]) and torch.isnan(got["x"][17]).all()
    rest = torch.arange(140) != 17
    assert torch.isfinite(got["loss"][rest]).all() and torch.isfinite(got["x"][rest]).all()


def test_linear_ce_target_out_of_range_is_nan():
    t, target = ce_inputs(20, 32, 100, F16, False, seed=5)
    target[4], target[11] = 100, -1
    got = run_ce(t, target, "none", torch.ones(20))
    bad = torch.zeros(20, dtype=torch.bool)
    bad[[4, 11]] = True
    assert torch.isnan(got["loss"][bad]).all() and torch.isfinite(got["loss"][~bad]).all()
    assert torch.isnan(got["x"][bad]).all() and torch.isfinite(got["x"][~bad]).all()


def test_linear_ce_bias_of_minus_infinity_removes_a_word():
    t, target = ce_inputs(30, 48, 300, F16, True, seed=6)
    target[target == 299] = 0
    target[target == 5] = 1
    t["bias"][5] = t["bias"][299] = float("-inf")
    got = run_ce(t, target, "none")
    keep = [i for i in range(300) if i not in (5, 299)]
    z = t["x"].double() @ t["weight"].double().T + t["bias"].double()
    want = torch.logsumexp(z[:, keep], 1) - z.gather(1, target[:, None])[:, 0]
    assert torch.allclose(got["loss"].double(), want, atol=2e-5, rtol=0)  # 2^-20 + (48/16 + 16) 2^-23 of |z| terms below 8


def test_linear_ce_large_logits_do_not_overflow():
    # a bare exponential of these logits overflows binary32
    t, target = ce_inputs(60, 64, 400, F32, False, seed=8)
    t["weight"] *= 100
    check_ce(t, target, "mean", torch.tensor(1.0))


@pytest.mark.parametrize("scale_x,scale_w", [(1e-8, 1e4), (1e6, 1e-5), (1e-20, 1e20)])
def test_linear_ce_fp32_magnitudes(scale_x, scale_w):
    t, target = ce_inputs(70, 120, 500, F32, False, seed=9)
    t["x"] *= scale_x
    t["weight"] *= scale_w
    check_ce(t, target, "mean", torch.tensor(1.0))


def test_linear_ce_other_ignore_index_and_leading_dimensions():
    t, target = ce_inputs(24, 40, 90, F16, False, seed=10)
    target[::3] = 0
    check_ce(t, target, "mean", torch.tensor(32.0), ignore=0)
    x3 = t["x"].view(2, 3, 4, 40).to(DEV)
    loss = ops.linear_cross_entropy(x3, t["weight"].to(DEV), target.view(2, 3, 4).to(DEV), reduction="none")
    assert loss.shape == (2, 3, 4) and loss.dtype == F32
    flat = run_ce(t, target, "none")["loss"]
    assert torch.equal(loss.cpu().view(-1), flat)


def test_linear_ce_single_row_without_leading_dimensions():
    t, target = ce_inputs(1, 40, 90, F16, True, seed=2)
    x = t["x"][0].to(DEV).requires_grad_()
    loss = ops.linear_cross_entropy(x, t["weight"].to(DEV), target[0].to(DEV), t["bias"].to(DEV), reduction="none")
    assert loss.shape == ()
    loss.backward()
    want = R.linear_ce64(t["x"], t["weight"], target, t["bias"], reduction="none", grad=torch.ones(1))
    R.assert_within(loss.detach().cpu()[None], *want["loss"], "loss")
    R.assert_within(x.grad.cpu()[None], *want["x"], "x")


def test_linear_ce_replayed_from_a_graph():
    """The C entries captured into a CUDA graph and replayed on new values in the
    same memory, twice, against ordinary calls."""
    n, d, v = 300, 96, 1000
    t, target = ce_inputs(n, d, v, F16, True, 40, seed=31)
    cu = {k: u.cuda() for k, u in t.items()}
    tg, g, loss = target.cuda(), torch.tensor([512.0], device="cuda"), torch.zeros(1, device="cuda")
    out = {k: torch.empty_like(u) for k, u in cu.items()}
    L, desc = _capi.lib(), _capi.LinearCeGradDesc()
    f = desc.fwd
    f.dtype, f.rows, f.cols, f.vocab, f.ignore_index, f.reduction = 0, n, d, v, -100, 1
    f.x, f.weight, f.bias, f.target, f.loss = cu["x"].data_ptr(), cu["weight"].data_ptr(), cu["bias"].data_ptr(), tg.data_ptr(), loss.data_ptr()
    desc.grad_loss, desc.dx, desc.dweight, desc.dbias = g.data_ptr(), out["x"].data_ptr(), out["weight"].data_ptr(), out["bias"].data_ptr()

    def room(size):
        b = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
        return b, (b.data_ptr() + 1023) // 1024 * 1024

    keep = [room(L.tk_linear_ce_state_size(ctypes.byref(f)))]
    f.state = keep[0][1]
    sizes = L.tk_linear_ce_workspace_size(ctypes.byref(f)), L.tk_linear_ce_backward_workspace_size(ctypes.byref(desc))
    keep += [room(s) for s in sizes]

    def call(stream):
        _capi.check(L.tk_linear_ce(ctypes.byref(f), keep[1][1], sizes[0], stream), "tk_linear_ce")
        _capi.check(L.tk_linear_ce_backward(ctypes.byref(desc), keep[2][1], sizes[1], stream), "tk_linear_ce_backward")

    call(None)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call(s.cuda_stream)
    for seed in (32, 33):
        t2, target2 = ce_inputs(n, d, v, F16, True, 10 * (seed - 30), seed=seed)
        for k in cu:
            cu[k].copy_(t2[k])
        tg.copy_(target2)
        graph.replay()
        torch.cuda.synchronize()
        plain = run_ce(t2, target2, "mean", torch.tensor(512.0))
        assert torch.equal(loss.cpu()[0], plain["loss"])
        for k in cu:
            assert torch.equal(out[k].cpu(), plain[k]), k


def test_linear_ce_strided_and_misaligned_inputs():
    t, target = ce_inputs(50, 64, 200, F16, True, seed=11)
    plain = run_ce(t, target, "none")["loss"]
    xt = t["x"].t().contiguous().to(DEV).t()
    w = torch.empty(200 * 64 + 1, dtype=F16, device=DEV)
    w[1:].copy_(t["weight"].view(-1).to(DEV))
    b = torch.empty(201, dtype=F16, device=DEV)
    b[1:].copy_(t["bias"].to(DEV))
    got = ops.linear_cross_entropy(xt, w[1:].view(200, 64), target.to(DEV), b[1:], reduction="none").cpu()
    assert torch.equal(got, plain)


@pytest.mark.parametrize("n,d,v,ignored", [(2100, 512, 2300, 0), (2500, 1000, 2100, 900), (2050, 2048, 5003, 0), (4000, 1024, 2048, 3990)])
def test_linear_ce_many_tiles(n, d, v, ignored):
    # more tiles than pairs of SMs, and few, split along K
    t, target = ce_inputs(n, d, v, F16, True, ignored, seed=n)
    check_ce(t, target, "mean", torch.tensor(4096.0))


@pytest.mark.parametrize("dtype,n,d,v", [(F16, 16384, 64, 20003), (F16, 14000, 512, 20003), (F32, 9000, 40, 20003)])
def test_linear_ce_several_pieces_of_the_vocabulary(dtype, n, d, v):
    # dz of all columns is larger than one piece
    t, target = ce_inputs(n, d, v, dtype, True, n // 3, seed=12)
    check_ce(t, target, "mean", torch.tensor(4096.0))


@pytest.mark.parametrize("wanted", [("x",), ("weight",), ("bias",), ("x", "bias")])
def test_linear_ce_some_gradients(wanted):
    t, target = ce_inputs(90, 56, 310, F16, True, 8, seed=13)
    check_ce(t, target, "mean", torch.tensor(128.0), wanted=wanted)


def test_linear_ce_extreme_row_gradients():
    # one row's gradient far above the others', a zero one, and none at all
    t, target = ce_inputs(64, 72, 200, F16, False, seed=14)
    g = torch.ones(64)
    g[3], g[4] = 1000.0, 0.0
    got = check_ce(t, target, "none", g)
    assert not got["x"][4].any()
    zero = run_ce(t, target, "none", torch.zeros(64))
    assert not zero["x"].any() and not zero["weight"].any()


def test_linear_ce_empty_batch():
    t = {"x": torch.zeros(0, 16, dtype=F16), "weight": rnd((9, 16), 1), "bias": rnd((9,), 2)}
    target = torch.zeros(0, dtype=torch.int64)
    assert run_ce(t, target, "none")["loss"].shape == (0,)
    assert run_ce(t, target, "sum")["loss"] == 0 and torch.isnan(run_ce(t, target, "mean")["loss"])
    got = run_ce(t, target, "sum", torch.tensor(1.0))
    assert got["x"].shape == (0, 16) and not got["weight"].any() and not got["bias"].any()


def test_linear_ce_gradient_against_differences():
    t, target = ce_inputs(20, 24, 60, F32, True, 3, seed=15)
    got = run_ce(t, target, "mean", torch.tensor(1.0))
    wide = {k: v.double() for k, v in t.items()}

    def value(u):
        z = u["x"] @ u["weight"].T + u["bias"]
        return float(F.cross_entropy(z, target))

    for k in t:
        v = torch.randn(t[k].shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
        step = 1e-5
        slope = (value({**wide, k: wide[k] + step * v}) - value({**wide, k: wide[k] - step * v})) / (2 * step)
        # truncation step^2 and cancellation 2^-52 / step are far below 2^-18 of
        # the gradient's terms, its binary32 error
        assert abs(float((got[k].double() * v).sum()) - slope) <= 2.0 ** -18 * float((got[k].double() * v).abs().sum()) + 1e-8, k


def test_linear_ce_is_deterministic_on_streams_and_with_reused_memory():
    t, target = ce_inputs(700, 200, 3000, F16, True, 90, seed=16)
    g = torch.tensor(512.0)
    first = run_ce(t, target, "mean", g)
    s = kunlun.Stream()
    for _ in range(3):
        with kunlun.stream(s):
            junk = torch.empty(64 << 20, dtype=F16, device=DEV).fill_(float("nan"))  # what the workspace may hold
            del junk
            again = run_ce(t, target, "mean", g)
        s.synchronize()
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_linear_ce_backward_twice():
    t, target = ce_inputs(100, 64, 300, F16, False, seed=17)
    x = t["x"].to(DEV).requires_grad_()
    loss = ops.linear_cross_entropy(x, t["weight"].to(DEV), target.to(DEV))
    one, = torch.autograd.grad(loss, x, torch.tensor(2.0).to(DEV), retain_graph=True)
    two, = torch.autograd.grad(loss, x, torch.tensor(4.0).to(DEV))
    want = R.linear_ce64(t["x"], t["weight"], target, grad=torch.tensor(2.0))["x"]
    R.assert_within(one.cpu(), *want, "first")
    R.assert_within(two.cpu(), *R.linear_ce64(t["x"], t["weight"], target, grad=torch.tensor(4.0))["x"], "second")


def test_linear_ce_refusals():
    t, target = ce_inputs(6, 16, 40, F16, True)
    x, w, b, y = t["x"].to(DEV), t["weight"].to(DEV), t["bias"].to(DEV), target.to(DEV)
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(x, w, y, reduction="max")
    for bad in (lambda: ops.linear_cross_entropy(x, w[:, :8], y), lambda: ops.linear_cross_entropy(x, w.float(), y),
                lambda: ops.linear_cross_entropy(x, w, y[:4]), lambda: ops.linear_cross_entropy(x, w, target),
                lambda: ops.linear_cross_entropy(x, w, y.to(torch.int32)), lambda: ops.linear_cross_entropy(x, w, y, b[:3]),
                lambda: ops.linear_cross_entropy(t["x"], t["weight"], target),
                lambda: ops.linear_cross_entropy(x, w, y, b.cpu())):
        with pytest.raises(RuntimeError, match="linear_cross_entropy"):
            bad()
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(ops.linear_cross_entropy(leaf, w, y), leaf, create_graph=True)


def test_training_operators_in_one_step():
    """Two blocks of linear - relu - linear under residual norms with dropout,
    then the loss: every operator's results and gradients checked against its
    64-bit form on the values and gradients it met in the step."""
    n, d, v, hid = 96, 128, 500, 256
    names = [("w1", (hid, d)), ("w2", (d, hid)), ("g", (d,)), ("b", (d,)), ("pg", (d,)), ("pb", (d,)), ("gate", (d,))]
    params = [{k: (rnd(s, 10 * i + j, F16, 1 / s[-1] ** 0.5 if len(s) == 2 else 0.1) + (0 if len(s) == 2 or k in ("b", "pb") else 1)).to(F16)
               for j, (k, s) in enumerate(names)} for i in range(2)]
    dev = [{k: t.to(DEV).requires_grad_() for k, t in p.items()} for p in params]
    x0 = rnd((n, d), 77)
    head, target = rnd((v, d), 78, F16, 0.1), torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(3))
    target[::7] = -100
    hd = head.to(DEV).requires_grad_()
    x = x0.to(DEV).requires_grad_()
    h, steps = x, []
    for i, p in enumerate(dev):
        f = F.linear(torch.relu(F.linear(h, p["w1"])), p["w2"])
        x_new, h = ops.residual_norm(x, f, p["g"], p["b"], post_norm=True, post_weight=p["pg"], post_bias=p["pb"], gate=p["gate"], p=0.1, seed=42, offset=i)
        for t in (x, f, x_new, h):
            t.retain_grad()
        steps.append((x, f, x_new, h))
        x = x_new
    y = ops.dropout(h, 0.2, 42, 9)
    y.retain_grad()
    loss = ops.linear_cross_entropy(y, hd, target.to(DEV))
    loss.backward(torch.tensor(1024.0).to(DEV))
    cpu = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    want = R.linear_ce64(cpu(y), head, target, grad=torch.tensor(1024.0))
    R.assert_within(cpu(loss), *want["loss"], "loss")
    R.assert_within(cpu(y.grad), *want["x"], "dy")
    R.assert_within(cpu(hd.grad), *want["weight"], "dhead")
    keep = R.keep_mask(h.shape, 0.2, 42, 9)
    last = torch.where(keep, cpu(y.grad).float() * torch.tensor(1.25), 0.0).to(F16)
    assert torch.equal(cpu(h.grad), last)
    for i in (1, 0):
        xi, fi, xn, hi = steps[i]
        p = params[i]
        gx = cpu(xn.grad) if i == 0 else None
        got = R.residual_norm64(cpu(xi), cpu(fi), p["g"], p["b"], True, p["pg"], p["pb"], p["gate"], False, 1.0, 1e-5,
                                R.keep_mask(xi.shape, 0.1, 42, i), 0.1, gx, cpu(hi.grad))
        R.assert_within(cpu(xn), *got["x_new"], f"x_new {i}")
        R.assert_within(cpu(hi), *got["h"], f"h {i}")
        R.assert_within(cpu(fi.grad), *got["f"], f"df {i}")
        for k, name in (("g", "weight"), ("b", "bias"), ("pg", "post_weight"), ("pb", "post_bias"), ("gate", "gate")):
            R.assert_within(cpu(dev[i][k].grad), *got[name], f"{name} {i}")
        assert torch.isfinite(cpu(dev[i]["w1"].grad)).all() and cpu(dev[i]["w1"].grad).any()


def off_boundary(t):
    """A copy whose data start 2 (fp16) or 4 (fp32) bytes off a 16-byte boundary."""
    b = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    v = b[1:].view(t.shape)
    v.copy_(t)
    assert v.data_ptr() % 16 == t.element_size()
    return v


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("before", ["on", "off"])
@pytest.mark.parametrize("after", ["on", "off"])
def test_linear_ce_saved_tensors_come_back_at_another_address(before, after, bias):
    """Saved-tensor hooks (offloading, packing) hand the weight back in other
    memory: on a 16-byte boundary or off it, whatever it was in the forward pass."""
    t, target = ce_inputs(300, 96, 1000, F16, bias, 30, seed=21)
    want = run_ce(t, target, "mean", torch.tensor(512.0))
    dev = {k: v.to(DEV) for k, v in t.items()}
    if before == "off":
        dev["weight"] = off_boundary(dev["weight"])
    dev = {k: v.requires_grad_() for k, v in dev.items()}
    move = off_boundary if after == "off" else torch.clone
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.detach(), lambda v: move(v) if v.dtype == F16 else v):
        loss = ops.linear_cross_entropy(dev["x"], dev["weight"], target.to(DEV), dev.get("bias"))
    grads = torch.autograd.grad(loss, list(dev.values()), torch.tensor(512.0).to(DEV))
    assert torch.equal(loss.detach().cpu(), want["loss"])
    for k, g in zip(dev, grads):
        assert torch.equal(g.cpu(), want[k]), k


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 65), (F32, 64)])
def test_linear_ce_saved_on_the_host(dtype, d):
    t, target = ce_inputs(40, d, 300, dtype, True, 5, seed=22)
    want = run_ce(t, target, "sum", torch.tensor(1.0))
    dev = {k: v.to(DEV).requires_grad_() for k, v in t.items()}
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.to(DEV)):
        loss = ops.linear_cross_entropy(dev["x"], dev["weight"], target.to(DEV), dev["bias"], reduction="sum")
    grads = torch.autograd.grad(loss, list(dev.values()))
    for k, g in zip(dev, grads):
        assert torch.equal(g.cpu(), want[k]), k


@pytest.mark.parametrize("dtype,low,high", [(F16, -4, 4), (F32, -12, 3)])
def test_linear_ce_each_row_has_its_own_gradient(dtype, low, high):
    """Gradients of the rows over many decades: every row of dx is as exact,
    relative to its own gradient, as with all gradients 1, and is the same
    whatever the other rows' gradients are."""
    n, d, v = 64, 72, 5000
    t, target = ce_inputs(n, d, v, dtype, True, 6, seed=41)
    g = (10.0 ** torch.linspace(low, high, n, dtype=torch.float64)).float()
    g[1::2] *= -1
    g[7] = 0
    got = check_ce(t, target, "none", g)
    value, bound = R.linear_ce64(t["x"], t["weight"], target, t["bias"], reduction="none", grad=torch.ones(n))["x"]
    own = g.double()[:, None]
    # linear in g_i: the error of a gradient of 1, times |g_i|, and the result's own rounding
    R.assert_within(got["x"], own * value, own.abs() * bound + R.ulp(own * value, dtype), "x")
    other = g.clone()
    other[::3] = 1.0
    again = run_ce(t, target, "none", other)
    same = torch.ones(n, dtype=torch.bool)
    same[::3] = False
    assert torch.equal(got["x"][same], again["x"][same])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_ce_subnormal_and_far_row_gradients(dtype):
    # a row far below the others adds nothing to dW that its rounding shows; alone it is all of it
    n, d, v = 40, 64, 300
    t, target = ce_inputs(n, d, v, dtype, True, seed=42)
    g = torch.full((n,), 2.0 ** -140)
    got = run_ce(t, target, "none", g)
    assert all(torch.isfinite(got[k]).all() for k in got)
    t["x"][3] *= 2.0 ** -9
    for big in (1.0, 2.0 ** -20):
        g = torch.full((n,), 2.0 ** -24 * big)
        g[3] = 512 * big
        check_ce(t, target, "none", g)
        g[3] = 0
        g[4] = -big
        check_ce(t, target, "none", g)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_ce_non_finite_row_gradients_stay_in_their_rows(dtype):
    n = 70
    t, target = ce_inputs(n, 96, 400, dtype, True, 8, seed=43)
    live = (target != -100).nonzero()[:, 0]
    g = loss_grad(n, "none")
    bad = torch.zeros(n, dtype=torch.bool)
    bad[live[[5, 9]]] = True
    g[bad] = 0.0
    clean = run_ce(t, target, "none", g)
    for values in ([float("nan"), 1.0], [float("inf"), 1.0], [float("nan"), float("-inf")]):
        g[bad] = torch.tensor(values)
        got = run_ce(t, target, "none", g)
        assert torch.equal(got["loss"], clean["loss"])
        assert torch.equal(got["x"][~bad], clean["x"][~bad])
        assert not torch.isfinite(got["x"][live[5]]).any()
        assert not torch.isfinite(got["weight"]).any() and not torch.isfinite(got["bias"]).any()


def test_linear_ce_row_gradients_over_several_pieces():
    t, target = ce_inputs(14000, 72, 20003, F16, True, 14000 // 3, seed=44)
    check_ce(t, target, "none", loss_grad(14000, "none") * 64)


@pytest.mark.parametrize("d", [1024, 1000, 1001])
def test_linear_ce_holds_its_input_once(d):
    # from forward to backward: the state, which has x's rows, and not x besides
    t, target = ce_inputs(4096, d, 300, F16, False, 500, seed=51)
    w, tg = t["weight"].to(DEV).requires_grad_(), target.to(DEV)
    kunlun.synchronize()
    before = kunlun.memory_allocated()
    loss = ops.linear_cross_entropy(t["x"].to(DEV), w, tg)
    kunlun.synchronize()
    f = _capi.LinearCeDesc()
    f.dtype, f.rows, f.cols, f.vocab, f.reduction = 0, 4096, d, 300, 1
    assert kunlun.memory_allocated() - before <= _capi.lib().tk_linear_ce_state_size(ctypes.byref(f)) + (1 << 20)
    got, = torch.autograd.grad(loss, w, torch.tensor(64.0).to(DEV))
    assert torch.equal(got.cpu(), run_ce(t, target, "mean", torch.tensor(64.0))["weight"])


def test_linear_ce_input_changed_after_the_forward_pass():
    t, target = ce_inputs(50, 64, 200, F16, True, 5, seed=52)
    want = run_ce(t, target, "mean", torch.tensor(64.0))
    dev = {k: v.to(DEV).requires_grad_(k != "x") for k, v in t.items()}
    loss = ops.linear_cross_entropy(dev["x"], dev["weight"], target.to(DEV), dev["bias"])
    dev["x"].zero_()
    got = torch.autograd.grad(loss, [dev["weight"], dev["bias"]], torch.tensor(64.0).to(DEV))
    assert torch.equal(got[0].cpu(), want["weight"]) and torch.equal(got[1].cpu(), want["bias"])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,v", [(64, 300), (512, 1000), (768, 5003), (2048, 700)])
def test_linear_ce_of_rows_whose_target_dominates(dtype, d, v):
    """Target logits of 5 to 500 far above the others: no loss is negative, and a
    small one is as exact as its logits' differences, whatever their size."""
    n = 200
    t, target = ce_inputs(n, d, v, dtype, True, seed=d + v)
    w = t["weight"].double()[target]
    size = 10.0 ** torch.linspace(0.7, 2.7, n, dtype=torch.float64)
    t["x"] = (size[:, None] * w / w.square().sum(1, keepdim=True)).to(dtype)
    X, W = t["x"].double(), t["weight"].double()
    z = X @ W.T + t["bias"].double()
    hit = z.gather(1, target[:, None])
    want = torch.log1p((z - hit).exp().scatter(1, target[:, None], 0.0).sum(1))
    assert (want < 1e-6).sum() > 20 and (want > 1e-3).any()
    # a logit's error: each step of 16 (three products for fp32) cut to binary32, the planes' 2^-20, the bias
    mag = X.abs() @ W.abs().T + t["bias"].double().abs()
    e = ((d * (1 if dtype == F16 else 3) / 16 + 16) * 2.0 ** -23 + (0 if dtype == F16 else 2.0 ** -20)) * mag
    e = e.amax(1) + e.gather(1, target[:, None])[:, 0]
    # the others' exponentials move by the differences' errors, and 2^-18 for exponentials and logarithm; the sum, the
    # target's 1 among its terms, is rounded at each of 32 additions in a row and then 32 + v / 2048 joins: a half
    # step, 2^-24, each, whatever the loss
    for reduction in ("none", "sum"):
        got = run_ce(t, target, reduction)["loss"]
        assert (got >= 0).all()
        value, bound = (want, want * (torch.expm1(e) + 2.0 ** -18) + (64 + v / 2048) * 2.0 ** -24)
        if reduction == "sum":
            value, bound = value.sum(), bound.sum()
        R.assert_within(got, value, bound, f"loss {reduction}")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_ce_of_one_word_is_zero(dtype):
    t, target = ce_inputs(300, 72, 1, dtype, True, seed=3)
    t["x"] *= 50
    got = run_ce(t, target, "none", torch.ones(300))
    assert not got["loss"].any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d,v", [(64, 300), (768, 5003), (1032, 300), (1500, 777), (4096, 700)])
def test_linear_ce_gradient_of_rows_whose_target_dominates(dtype, d, v):
    """The softmax of the backward pass is that of the forward pass's logits: where
    the target has all of it, its entry of dz is zero up to logsumexp's rounding,
    however large the logits."""
    n = 100
    t, target = ce_inputs(n, d, v, dtype, False, seed=d + v)
    w = t["weight"].double()[target]
    size = 10.0 ** torch.linspace(1.7, 2.7, n, dtype=torch.float64)
    t["x"] = (size[:, None] * w / w.square().sum(1, keepdim=True)).to(dtype)
    X, W = t["x"].double(), t["weight"].double()
    z = X @ W.T
    lse = torch.logsumexp(z, 1)
    dz = (z - lse[:, None]).exp()
    hit = z.gather(1, target[:, None])
    rest = (z - hit).exp().scatter(1, target[:, None], 0.0).sum(1, keepdim=True)
    dz.scatter_(1, target[:, None], -rest / (1 + rest))
    others = dz.scatter(1, target[:, None], 0.0).abs()
    assert (others < 1e-6).all()
    # the target's entry: logsumexp / ln 2 and its difference from the logit are rounded (a half step, 2^-24, each) and
    # held to the sum's 64 + v / 2048 half steps, the exponential to 2^-22; the others' are below 1e-6 and 1 % exact
    e_hit = 2.0 ** -23 * (lse.abs() / 0.6931 + 64 + v / 2048) + 2.0 ** -22
    e_dz = (0.01 * others + 2.0 ** -39).scatter(1, target[:, None], e_hit[:, None])
    value = dz @ W
    bound = e_dz @ W.abs() + (d + v) * 2.0 ** -23 * (dz.abs() @ W.abs()) + R.ulp(value, dtype)
    got = run_ce(t, target, "sum", torch.tensor(1.0), wanted=("x",))["x"]
    R.assert_within(got, value, bound, "x")


@pytest.mark.parametrize("dtype,size", [(F16, 2.0 ** 13), (F32, 2.0 ** 40), (F32, 2.0 ** 100)])
def test_linear_ce_a_far_larger_row_leaves_the_others_alone(dtype, size):
    """The losses and gradients of rows do not depend on another row's size, as
    padding that the caller weighs with zero may have any."""
    n = 60
    t, target = ce_inputs(n, 72, 500, dtype, True, 5, seed=61)
    at = int((target != -100).nonzero()[3])
    rest = torch.arange(n) != at
    g = loss_grad(n, "none")
    g[at] = 0
    t["x"][at] = t["x"][at].clamp(-1, 1)
    want = run_ce(t, target, "none", g)
    t["x"][at] *= size
    got = run_ce(t, target, "none", g)
    assert torch.equal(got["loss"][rest], want["loss"][rest]) and torch.equal(got["x"][rest], want["x"][rest])
    assert torch.equal(got["weight"], want["weight"]) and torch.equal(got["bias"], want["bias"])
    t["x"][at] = torch.finfo(dtype).min
    got = run_ce(t, target, "none", g)
    assert torch.equal(got["loss"][rest], want["loss"][rest]) and torch.equal(got["x"][rest], want["x"][rest])


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_linear_ce_fp32_rows_of_many_sizes(reduction):
    n = 90
    t, target = ce_inputs(n, 100, 400, F32, True, 7, seed=62)
    t["x"] *= (2.0 ** torch.linspace(-100, 4, n))[:, None]
    t["x"][5] = 0
    check_ce(t, target, reduction, loss_grad(n, reduction))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,d,v,reduction", [(50, 64, 200, "none"), (300, 96, 1000, "mean"), (70, 100, 333, "sum"), (16384, 64, 20003, "mean")])
def test_linear_ce_gradients_of_misaligned_tensors(n, d, v, reduction, dtype):
    """Every tensor, results among them, off a 16-byte boundary and at offsets of
    its own, over one and several pieces of the vocabulary: the aligned call's bits."""
    t, target = ce_inputs(n, d, v, dtype, True, n // 9, seed=n + d)
    g = loss_grad(n, reduction).reshape(-1)
    want = run_ce(t, target, reduction, g if reduction == "none" else g[0])
    L, desc, hold = _capi.lib(), _capi.LinearCeGradDesc(), []

    def off(v, k):
        b = torch.full((v.numel() + 8,), 7.0 if v.is_floating_point() else 7, dtype=v.dtype, device="cuda")
        b[k:k + v.numel()] = v.reshape(-1).cuda()
        hold.append(b)
        return b[k:k + v.numel()].view(v.shape)

    def room(size):
        b = torch.full((size + 1024,), 255, dtype=torch.uint8, device="cuda")
        hold.append(b)
        return (b.data_ptr() + 1023) // 1024 * 1024

    f = desc.fwd
    f.dtype, f.rows, f.cols, f.vocab, f.ignore_index, f.reduction = int(dtype == F32), n, d, v, -100, ["none", "mean", "sum"].index(reduction)
    ins = {"x": off(t["x"], 1), "weight": off(t["weight"], 3), "bias": off(t["bias"], 1)}
    loss, gl, tg = off(torch.zeros(n if reduction == "none" else 1), 1), off(g, 1), off(target, 1)
    outs = {k: off(torch.zeros_like(t[k]), i + 1) for i, k in enumerate(t)}
    f.x, f.weight, f.bias, f.target, f.loss = (u.data_ptr() for u in (ins["x"], ins["weight"], ins["bias"], tg, loss))
    assert all(u.data_ptr() % 16 for u in (*ins.values(), *outs.values(), loss, gl, tg))
    desc.grad_loss, desc.dx, desc.dweight, desc.dbias = gl.data_ptr(), outs["x"].data_ptr(), outs["weight"].data_ptr(), outs["bias"].data_ptr()
    f.state = room(L.tk_linear_ce_state_size(ctypes.byref(f)))
    sizes = L.tk_linear_ce_workspace_size(ctypes.byref(f)), L.tk_linear_ce_backward_workspace_size(ctypes.byref(desc))
    torch.cuda.synchronize()
    _capi.check(L.tk_linear_ce(ctypes.byref(f), room(sizes[0]), sizes[0], None), "tk_linear_ce")
    _capi.check(L.tk_linear_ce_backward(ctypes.byref(desc), room(sizes[1]), sizes[1], None), "tk_linear_ce_backward")
    torch.cuda.synchronize()
    assert torch.equal(loss.cpu(), want["loss"].reshape(-1))
    for i, k in enumerate(t):
        assert torch.equal(outs[k].cpu(), want[k]), k
        rim = outs[k].numel() + i + 1
        whole = torch.as_strided(outs[k], (outs[k].numel() + 8,), (1,), 0).cpu()
        assert (whole[:i + 1] == 7).all() and (whole[rim:] == 7).all(), k  # nothing beside the result is written
