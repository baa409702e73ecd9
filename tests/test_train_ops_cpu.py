"""What needs no GPU of the training operators: the generator's published
vectors, the 64-bit references against torch's autograd, and the argument
checks that come before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from tests import _train_helpers as R
from torch_kunlun_b200 import _capi as C


def test_philox_known_answers():
    # the published test vectors of Philox4x32-10: counter, key -> words
    def block(counter, key):
        lo = counter[0] | counter[1] << 32
        c = [counter[0], counter[1], counter[2], counter[3]]
        k = [key[0], key[1]]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c, lo
    assert block([0] * 4, [0] * 2)[0] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert block([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2)[0] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert block([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0])[0] == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    words = R.philox_words(8, 0x299F31D0A4093822, 0x0370734413198A2E)
    for i in range(2):
        assert list(words[4 * i:4 * i + 4]) == block([i, 0, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0])[0]
    assert words.dtype == np.uint64


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("post", [False, True])
def test_residual_norm_reference_matches_autograd(rms, post):
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float32)  # noqa: E731
    x, f, w, b, gate = n(2, 5, 12), n(2, 5, 12), n(12), n(12), n(2, 1, 12)
    pw, pb = (n(12), n(12)) if post else (None, None)
    gx, gh, keep = n(2, 5, 12), n(2, 5, 12), torch.rand(2, 5, 12, generator=g) > 0.3
    got = R.residual_norm64(x, f, w, b, post, pw, pb, gate, rms, 0.7, 1e-5, keep, 0.3, gx, gh)
    leaves = {k: v.double().requires_grad_() for k, v in dict(x=x, f=f, weight=w, bias=b, post_weight=pw, post_bias=pb, gate=gate).items() if v is not None}

    def norm(v, w, b):
        m = 0 if rms else v.mean(-1, keepdim=True)
        return (v - m) / ((v - m).square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    u = norm(leaves["f"], leaves["post_weight"], leaves["post_bias"]) if post else leaves["f"]
    x_new = 0.7 * leaves["x"] + leaves["gate"] * u * keep.double() / 0.7
    h = norm(x_new, leaves["weight"], leaves["bias"])
    grads = torch.autograd.grad([x_new, h], list(leaves.values()), [gx.double(), gh.double()])
    for k, v in {"x_new": x_new, "h": h, **dict(zip(leaves, grads))}.items():
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-10), k


def test_dropout_refuses_bad_arguments_before_the_device():
    L = C.lib()
    assert L.tk_dropout(5, 16, 16, 4, 0.1, 1, 0, None) == 1
    assert L.tk_dropout(0, 16, 16, -1, 0.1, 1, 0, None) == 1
    assert L.tk_dropout(0, None, 16, 4, 0.1, 1, 0, None) == 1
    for p in (-0.5, 1.5, float("nan")):
        assert L.tk_dropout(0, 16, 16, 4, p, 1, 0, None) == 1
        assert b"[0, 1]" in L.tk_last_error_string()
    assert L.tk_dropout(0, None, None, 0, 0.1, 1, 0, None) == 0  # nothing to do


def _norm_desc(**kw):
    d = C.ResidualNormDesc()
    d.dtype, d.norm, d.rows, d.cols, d.residual_scale, d.eps = 0, 0, 4, 16, 1.0, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("fields,status", [
    (dict(dtype=7), 1), (dict(norm=2), 1), (dict(rows=-1), 1), (dict(cols=0), 1), (dict(cols=32769), 2),
    (dict(p=1.5), 1), (dict(p=float("nan")), 1), (dict(post_weight=16), 1), (dict(gate=16, gate_rows=3), 1),
    (dict(gate=16, gate_rows=0), 1), (dict(rows=1 << 62), 1), (dict(), 1)])  # the last: NULL tensors
def test_residual_norm_refuses_bad_arguments_before_the_device(fields, status):
    L = C.lib()
    d = _norm_desc(**fields)
    assert L.tk_residual_norm(ctypes.byref(d), None) == status
    g = C.ResidualNormGradDesc()
    g.fwd = d
    assert L.tk_residual_norm_backward(ctypes.byref(g), None, 0, None) == status
    if fields:
        assert L.tk_residual_norm_backward_workspace_size(ctypes.byref(g)) == 0
    assert L.tk_residual_norm(None, None) == 1 and L.tk_residual_norm_backward(None, None, 0, None) == 1


def test_residual_norm_backward_needs_its_inputs():
    L = C.lib()
    g = C.ResidualNormGradDesc()
    g.fwd = _norm_desc(x=16, f=16, stats=16)
    assert L.tk_residual_norm_backward(ctypes.byref(g), None, 0, None) == 1
    assert b"no incoming gradient" in L.tk_last_error_string()
    g.grad_h = 16
    for field in ("dpost_weight", "dpost_bias", "dgate"):
        setattr(g, field, 16)
        assert L.tk_residual_norm_backward(ctypes.byref(g), None, 0, None) == 1, field
        setattr(g, field, None)
    for field, bad in (("f", None), ("x", None), ("stats", 8)):
        kept = getattr(g.fwd, field)
        setattr(g.fwd, field, bad)
        assert L.tk_residual_norm_backward(ctypes.byref(g), None, 0, None) == 1
        assert b"are needed" in L.tk_last_error_string()
        setattr(g.fwd, field, kept)
    assert L.tk_residual_norm(ctypes.byref(_norm_desc(rows=0)), None) == 0


@pytest.mark.parametrize("rows,units", [(1, 1), (5, 3), (148, 148), (1000, 296), (16384, 296), (97, 96)])
def test_row_ranges_partition_and_unit_of_inverts(rows, units):
    # unit_begin / unit_of of residual_norm.cu
    begin = [u * rows // units for u in range(units + 1)]
    assert begin[0] == 0 and begin[-1] == rows and all(a < b for a, b in zip(begin, begin[1:]))
    for r in range(rows):
        u = ((r + 1) * units - 1) // rows
        assert begin[u] <= r < begin[u + 1]


@pytest.mark.parametrize("rows,units,gate_rows", [(12, 5, 3), (4001 * 3, 296, 3), (811 * 13, 148, 811), (96, 7, 96 // 2), (300, 13, 1)])
def test_gate_segments_reach_the_column_kernel_once(rows, units, gate_rows):
    """Every gate row is finished exactly once: by the unit that holds it whole,
    or by the item of the first unit boundary inside it, over the slots its
    units wrote."""
    period = rows // gate_rows
    begin = [u * rows // units for u in range(units + 1)]
    unit_of = lambda r: ((r + 1) * units - 1) // rows  # noqa: E731
    written, finished = {}, {}
    for u in range(units):
        lo = begin[u]
        while lo < begin[u + 1]:
            row = lo // period
            hi = min(begin[u + 1], (row + 1) * period)
            if lo == row * period and hi == (row + 1) * period:
                finished[row] = finished.get(row, 0) + 1
            else:
                slot = 2 * u + (0 if lo == begin[u] else 1)
                assert slot not in written
                written[slot] = (row, hi - lo)
            lo = hi
    for u in range(1, units):
        row = begin[u] // period
        if begin[u] % period == 0 or unit_of(row * period) != u - 1:
            continue
        last = unit_of((row + 1) * period - 1)
        covered = 0
        for v in range(u - 1, last + 1):
            got_row, n = written.pop(2 * v + (0 if begin[v] // period == row else 1))
            assert got_row == row
            covered += n
        assert covered == period
        finished[row] = finished.get(row, 0) + 1
    assert not written and finished == {r: 1 for r in range(gate_rows)}


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_linear_ce_reference_matches_torch(reduction):
    g = torch.Generator().manual_seed(5)
    x, w, b = (torch.randn(s, generator=g) for s in ((11, 6), (17, 6), (17,)))
    target = torch.randint(0, 17, (11,), generator=g)
    target[[2, 7]] = -100
    up = torch.randn(11, generator=g) if reduction == "none" else torch.tensor(3.0)
    got = R.linear_ce64(x, w, target, b, reduction=reduction, grad=up)
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    loss = torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].T + leaves[2], target, reduction=reduction)
    grads = torch.autograd.grad(loss, leaves, up.double())
    for k, v in zip(("loss", "x", "weight", "bias"), (loss, *grads)):
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-10), k


def _ce_desc(**kw):
    d = C.LinearCeDesc()
    d.dtype, d.rows, d.cols, d.vocab, d.reduction, d.ignore_index, d.loss = 0, 4, 16, 32, 1, -100, 16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("fields,status", [
    (dict(dtype=3), 1), (dict(reduction=5), 1), (dict(rows=-1), 1), (dict(cols=0), 1), (dict(vocab=0), 1),
    (dict(vocab=1 << 31), 2), (dict(rows=1 << 40), 2), (dict(rows=1 << 30, vocab=1 << 20), 2), (dict(cols=1 << 30, vocab=1 << 20), 2)])
def test_linear_ce_refuses_bad_arguments_before_the_device(fields, status):
    L = C.lib()
    d = _ce_desc(**fields)
    g = C.LinearCeGradDesc()
    g.fwd = d
    assert L.tk_linear_ce_workspace_size(ctypes.byref(d)) == 0 and L.tk_linear_ce_state_size(ctypes.byref(d)) == 0
    assert L.tk_linear_ce_backward_workspace_size(ctypes.byref(g)) == 0
    assert L.tk_linear_ce(ctypes.byref(d), None, 0, None) == status
    assert L.tk_linear_ce_backward(ctypes.byref(g), None, 0, None) == status


def test_linear_ce_needs_pointers_and_workspace():
    L = C.lib()
    assert L.tk_linear_ce(None, None, 0, None) == 1 and L.tk_linear_ce_backward(None, None, 0, None) == 1
    d = _ce_desc()
    assert L.tk_linear_ce(ctypes.byref(d), None, 0, None) == 1  # NULL tensors
    d.x = d.weight = d.target = 1024  # never dereferenced: the workspace check fails first
    assert L.tk_linear_ce(ctypes.byref(d), None, 0, None) == 4
    need = L.tk_linear_ce_workspace_size(ctypes.byref(d))
    assert L.tk_linear_ce(ctypes.byref(d), 512, need, None) == 4  # not 1024-byte aligned
    assert L.tk_linear_ce(ctypes.byref(d), 1024, need - 1, None) == 4
    g = C.LinearCeGradDesc()
    g.fwd = d
    assert L.tk_linear_ce_backward(ctypes.byref(g), None, 0, None) == 1  # no state
    g.fwd.state, g.grad_loss = 1024, 1024
    assert L.tk_linear_ce_backward(ctypes.byref(g), None, 0, None) == 4
    g.dbias = 1024
    assert L.tk_linear_ce_backward(ctypes.byref(g), None, 0, None) == 1 and b"bias" in L.tk_last_error_string()


@pytest.mark.parametrize("dtype,rows,vocab", [(0, 1, 1), (0, 8192, 65536), (0, 16384, 30011), (1, 9000, 20003), (0, 200000, 140000), (1, 1 << 20, 300)])
def test_linear_ce_workspace_is_bounded_by_its_pieces(dtype, rows, vocab):
    """dz is held one piece at a time: at most 512 MiB, or one 256-column tile."""
    L = C.lib()
    g = C.LinearCeGradDesc()
    g.fwd = _ce_desc(dtype=dtype, rows=rows, vocab=vocab, cols=64, weight=1024)
    pad = (rows + 255) // 256 * 256
    planes = 1 + dtype
    packed = planes * pad * 64 * 2 + (planes * vocab * 64 * 2 if dtype else 0)
    dz = max(512 << 20, pad * 2 * planes * 256)
    acc = pad * 64 * 4
    split = 2 * 148 * 128 * 256 * 4
    assert L.tk_linear_ce_backward_workspace_size(ctypes.byref(g)) <= packed + dz + acc + split + 4 * pad + 8192


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("cols", [96, 97])
def test_linear_ce_state_size_does_not_depend_on_addresses(dtype, cols):
    # the backward pass may see the weight at another address, and a caller may ask before it has one
    L = C.lib()
    size = lambda **kw: L.tk_linear_ce_state_size(ctypes.byref(_ce_desc(dtype=dtype, rows=300, cols=cols, vocab=1000, **kw)))  # noqa: E731
    sizes = {size(weight=w, bias=b) for w in (None, 1024, 1026, 1032) for b in (None, 1024)}
    assert len(sizes) == 1 and sizes.pop() > 0


def test_linear_ce_workspaces_have_room_for_a_weight_off_the_boundary():
    L = C.lib()
    g = C.LinearCeGradDesc()
    sizes = []
    for weight in (1024, 1026):
        g.fwd = _ce_desc(rows=300, cols=96, vocab=1000, weight=weight)
        sizes.append((L.tk_linear_ce_workspace_size(ctypes.byref(g.fwd)), L.tk_linear_ce_backward_workspace_size(ctypes.byref(g))))
    packed = 1000 * 96 * 2
    assert all(off >= on + packed for on, off in zip(*sizes))


@pytest.mark.parametrize("gate_rows", [0, 1, 5])
def test_residual_norm_without_rows_takes_any_gate(gate_rows):
    L = C.lib()
    d = _norm_desc(rows=0, gate=1024, gate_rows=gate_rows)
    assert L.tk_residual_norm(ctypes.byref(d), None) == 0
    g = C.ResidualNormGradDesc()
    g.fwd = d
    assert L.tk_residual_norm_backward_workspace_size(ctypes.byref(g)) > 0
    assert L.tk_residual_norm_backward(ctypes.byref(g), None, 0, None) == 0
    assert L.tk_residual_norm(ctypes.byref(_norm_desc(rows=0, gate=1024, gate_rows=-1)), None) == 1


def _norm_gradients(t, gx, gh, keep, p, rms, mistake=None):
    """The residual norm's results from its formulas in binary64, rounded once;
    `mistake` leaves one thing out or takes it wrong."""
    d = {k: v.double() for k, v in t.items()}
    gx, gh = gx.double(), gh.double()
    mean = (lambda v: 0.0) if rms else (lambda v: v.mean(-1, keepdim=True))

    def norm(v):
        r = ((v - mean(v)).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        return (v - mean(v)) * r, r

    def back(n, r, g):
        a = 0.0 if mistake == "mean" else mean(g)
        return r * (g - a - (0.0 if mistake == "product mean" else n * (g * n).mean(-1, keepdim=True)))

    drop = keep.double() / (1 - p)
    q, rq = norm(d["f"])
    u = drop * (q * d["post_weight"] + d["post_bias"])
    x_new = d["x"] + d["gate"] * u
    if mistake == "rounded":
        x_new = x_new.to(t["x"].dtype).double()
    n, r = norm(x_new)
    g = gx + back(n, r, gh * (1.0 if mistake == "weight" else d["weight"]))
    gu = g * (1.0 if mistake == "gate" else d["gate"]) * (1.0 if mistake == "mask" else drop)
    rows = (0, 1)
    out = {"x": g, "weight": (gh * n).sum(rows), "bias": gh.sum(rows), "gate": (g * u).sum(rows),
           "post_weight": (gu * (q if mistake != "row" else q * (torch.arange(q.shape[1]) > 0)[:, None])).sum(rows), "post_bias": gu.sum(rows),
           "f": back(q, rq, gu * (1.0 if mistake == "post weight" else d["post_weight"]))}
    return {k: v.to(t["x"].dtype) for k, v in out.items()}


@pytest.mark.parametrize("shape", [(3, 37, 768), (1, 3000, 256)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rms", [False, True])
def test_residual_norm_bounds_tell_mistakes(shape, dtype, rms):
    """The bounds for the unrounded x_new admit the formulas' rounded values and
    none of these mistakes."""
    g = torch.Generator().manual_seed(12)
    n = lambda s, scale=1.0, mean=0.0: (torch.randn(s, generator=g) * scale + mean).to(dtype)  # noqa: E731
    d = shape[-1]
    t = {"x": n(shape, 1.0, 0.5), "f": n(shape, 0.7), "weight": n(d, 0.1, 1.0), "bias": n(d, 0.1), "post_weight": n(d, 0.1, 1.0),
         "post_bias": n(d, 0.1), "gate": n(d, 0.3, 0.5)}
    gx, gh, keep = n(shape), n(shape), torch.rand(shape, generator=g) > 0.1
    rows = shape[0] * shape[1]
    want = R.residual_norm64(t["x"], t["f"], t["weight"], t["bias"], True, t["post_weight"], t["post_bias"], t["gate"], rms, 1.0, 1e-5,
                             keep, 0.1, gx, gh, chain=R.column_chain(rows))

    def beyond(mistake):
        got = _norm_gradients(t, gx, gh, keep, 0.1, rms, mistake)
        off = set()
        for k, v in got.items():
            value, bound = want[k]
            if ((v.double() - value).abs() > bound.expand_as(value)).any() or R.norm_error(v, value) > R.NORM_ERROR[dtype]:
                off.add(k)
        return off

    assert not beyond(None)
    expected = {"product mean": {"x", "f", "gate"}, "weight": {"x", "f"}, "gate": {"f", "post_weight", "post_bias"},
                "mask": {"f", "post_weight", "post_bias"}, "post weight": {"f"}, "row": {"post_weight"}}
    if not rms:
        expected["mean"] = {"x", "f"}
    for mistake, outputs in expected.items():
        assert outputs <= beyond(mistake), mistake


def test_residual_norm_bounds_tell_a_rounded_x_new():
    """Gradients from x_new rounded to binary16, without a norm behind the block:
    admitted by the wide bounds, beyond the tight ones."""
    g = torch.Generator().manual_seed(12)
    shape = (3, 37, 768)
    n = lambda s, scale=1.0, mean=0.0: (torch.randn(s, generator=g) * scale + mean).half()  # noqa: E731
    x, f, w, gx, gh = n(shape, 1.0, 0.5), n(shape, 0.7), n(768, 0.1, 1.0), n(shape), n(shape)
    tight = R.residual_norm64(x, f, w, gx=gx, gh=gh, chain=R.column_chain(111))["weight"]
    wide = R.residual_norm64(x, f, w, gx=gx, gh=gh)["weight"]

    def weight_gradient(x_new):
        c = x_new - x_new.mean(-1, keepdim=True)
        return (gh.double() * c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).sum((0, 1)).half()

    x_new = x.double() + f.double()
    off = lambda got, want: int(((got.double() - want[0]).abs() > want[1]).sum())  # noqa: E731
    assert off(weight_gradient(x_new), tight) == 0
    rounded = weight_gradient(x_new.half().double())
    assert off(rounded, wide) == 0 and off(rounded, tight) > 4
