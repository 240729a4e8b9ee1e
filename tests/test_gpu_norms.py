"""rms_norm and residual_norm on the GPU against float64, with the bounds of norm_reference.py.

Widths that use every row layout (parts of a warp, a block, several channels per thread), odd and
misaligned ones, no rows, one row, strided views; every mix of stream and update types; gates per
channel, per row and broadcast; scales; gradients against the formula and against differences;
another stream, a captured and replayed graph, equal results run to run.
"""
from __future__ import annotations

import itertools

import pytest
import torch

import norm_reference as ref
from gpa_b200 import _lib, residual_norm, rms_norm

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


WIDTHS = [1, 7, 8, 31, 40, 64, 100, 128, 250, 256, 257, 264, 1000, 1001, 1024, 2049, 2560, 4099, 8192,
          8200, 9001, 16383, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
def test_rms_norm_matches_float64(width, dtype, out_dtype):
    g = _gen(width)
    rows = 2 if width > 4000 else 37
    x = _randn(g, (rows, width), dtype, 2.0).requires_grad_()
    w = (1 + 0.2 * _randn(g, (width,))).requires_grad_()
    dy = _randn(g, (rows, width), out_dtype)
    y = rms_norm(x, w, EPS, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    ref.check("y", y, ref.plain_forward(x, w, EPS, out_dtype))
    with torch.no_grad():
        assert torch.equal(rms_norm(x, w, EPS, out_dtype=out_dtype), y)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = ref.plain_backward(x, w, EPS, dy)
    assert dx.dtype == dtype and dw.dtype == F32
    ref.check("dx", dx, want["dx"])
    ref.check("dweight", dw, want["dweight"])


def _inputs(seed, shape, stream, update, out, post, gate, scale):
    g = _gen(seed)
    width = shape[-1]
    t = {"residual": _randn(g, shape, stream, 2.0), "update": _randn(g, shape, update, 0.7),
         "weight": 1 + 0.2 * _randn(g, (width,)),
         "post_weight": 1 + 0.2 * _randn(g, (width,)) if post else None,
         "gate": None if gate is None else _randn(g, gate, update, 1.5),
         "scale": 0.3 * _randn(g, (width,)) if scale == "vector" else None}
    const = 0.25 if scale == "number" else 1.0
    return t, const, _randn(g, shape, stream, 0.5), _randn(g, shape, out, 0.5)


def _check_case(t, const, ds, dn, out, stream_grad=True, normed_grad=True):
    for x in t.values():
        if x is not None:
            x.requires_grad_()
    scale = t["scale"] if t["scale"] is not None else (const if const != 1.0 else None)
    h, n = residual_norm(t["residual"], t["update"], t["weight"], EPS, post_weight=t["post_weight"],
                         gate=t["gate"], scale=scale, out_dtype=out)
    assert h.dtype == t["residual"].dtype and n.dtype == out
    rest = (t["post_weight"], t["gate"], t["scale"], const, EPS)
    ref.check("stream", h, ref.stream_of(t["residual"], t["update"], *rest))
    ref.check("normed", n, ref.plain_forward(h, t["weight"], EPS, out))
    names = [k for k, x in t.items() if x is not None]
    outs = [o for o, k in ((h, stream_grad), (n, normed_grad)) if k]
    ups = [o for o, k in ((ds, stream_grad), (dn, normed_grad)) if k]
    if not normed_grad:
        names.remove("weight")
    grads = dict(zip(names, torch.autograd.grad(outs, [t[k] for k in names], ups)))
    want = ref.backward(h, t["update"], t["weight"], *rest[:3], const, EPS, ds if stream_grad else None,
                        dn if normed_grad else None)
    for k, x in grads.items():
        assert x.dtype == t[k].dtype and x.shape == t[k].shape
        ref.check("d" + k, x, want["d" + k])


MIXES = list(itertools.product([False, True], [None, "row", "full"], [None, "vector", "number"]))


@pytest.mark.parametrize("post,gate,scale", MIXES)
@pytest.mark.parametrize("width", [48, 1001, 1024])
def test_residual_norm_parts(width, post, gate, scale):
    shape = (3, 11, width)
    gs = {None: None, "row": (3, 11, 1), "full": shape}[gate]
    t, const, ds, dn = _inputs(width + 7 * post, shape, F32, BF16, BF16, post, gs, scale)
    _check_case(t, const, ds, dn, BF16)


@pytest.mark.parametrize("stream,update,out", list(itertools.product([F32, BF16, F16], repeat=3)))
def test_residual_norm_types(stream, update, out):
    shape = (2, 5, 264)
    t, const, ds, dn = _inputs(5, shape, stream, update, out, True, shape, "vector")
    _check_case(t, const, ds, dn, out)


@pytest.mark.parametrize("width", WIDTHS)
def test_residual_norm_widths(width):
    shape = (3, width)
    t, const, ds, dn = _inputs(width, shape, F32, BF16, BF16, True, shape, "vector")
    _check_case(t, const, ds, dn, BF16)


@pytest.mark.parametrize("rows", [1, 2, 1185, 20011])
@pytest.mark.parametrize("width", [24, 512])
def test_residual_norm_rows(rows, width):
    t, const, ds, dn = _inputs(rows, (rows, width), BF16, BF16, BF16, True, (rows, 1), "vector")
    _check_case(t, const, ds, dn, BF16)


@pytest.mark.parametrize("stream_grad,normed_grad", [(True, False), (False, True)])
def test_one_output_without_gradient(stream_grad, normed_grad):
    t, const, ds, dn = _inputs(3, (4, 9, 136), F32, F32, F32, True, (4, 9, 136), "vector")
    _check_case(t, const, ds, dn, F32, stream_grad, normed_grad)


def test_broadcast_gate_and_scalar_tensor_scale_get_summed_gradients():
    g = _gen(1)
    h, y = _randn(g, (3, 5, 64)), _randn(g, (3, 5, 64))
    w = 1 + 0.1 * _randn(g, (64,))
    gate = _randn(g, (3, 1, 64)).requires_grad_()
    scale = torch.tensor(0.4, device="cuda", requires_grad=True)
    up = _randn(g, (3, 5, 64))
    s, n = residual_norm(h, y, w, EPS, gate=gate, scale=scale)
    dg, dc = torch.autograd.grad((s, n), (gate, scale), (up, up))
    full, vec = gate.detach().expand(3, 5, 64).contiguous().requires_grad_(), torch.full((64,), 0.4, device="cuda")
    vec.requires_grad_()
    s2, n2 = residual_norm(h, y, w, EPS, gate=full, scale=vec)
    dg2, dc2 = torch.autograd.grad((s2, n2), (full, vec), (up, up))
    assert torch.equal(s, s2) and torch.equal(n, n2)
    # 5 and 64 terms summed in fp32: one rounding of the running sum for each
    assert (dg - dg2.sum(1, keepdim=True)).abs().max() <= 5 * ref.U * dg2.abs().sum(1).max()
    assert dc.shape == () and (dc - dc2.sum()).abs() <= 64 * ref.U * dc2.abs().sum()


def test_strided_views_are_read_in_place_and_copies_agree():
    g = _gen(2)
    joint = _randn(g, (2, 7, 6 * 32), BF16)
    w = 1 + 0.1 * _randn(g, (32,))
    x = joint[..., :4 * 32].unflatten(-1, (4, 32))
    assert torch.equal(rms_norm(x, w), rms_norm(x.contiguous(), w))
    odd = joint[..., 3:3 + 4 * 32].unflatten(-1, (4, 32))  # rows off the 16-byte boundary
    a, b = rms_norm(odd, w), rms_norm(odd.contiguous(), w)
    ref.check("odd", a, ref.plain_forward(odd, w, 1e-6, BF16))
    ref.check("odd", b, ref.plain_forward(odd, w, 1e-6, BF16))
    t = _randn(g, (5, 3, 4, 40)).permute(2, 0, 1, 3)  # three strides: copied
    wt = 1 + 0.1 * _randn(g, (40,))
    ref.check("permuted", rms_norm(t, wt), ref.plain_forward(t, wt, 1e-6, F32))
    col = _randn(g, (9, 48)).T  # no unit stride
    wc = 1 + 0.1 * _randn(g, (9,))
    ref.check("transposed", rms_norm(col, wc), ref.plain_forward(col, wc, 1e-6, F32))
    big, small = _randn(g, (6, 10, 64)), _randn(g, (1, 10, 64)).expand(6, 10, 64)
    s, n = residual_norm(big[:, ::2], small[:, 1::2], 1 + 0.1 * _randn(g, (64,)))
    assert torch.equal(s, big[:, ::2] + small[:, 1::2])
    x = joint.detach().requires_grad_()
    y = rms_norm(x[..., :128].unflatten(-1, (4, 32)), w)
    up = _randn(g, y.shape, BF16)
    (dx,) = torch.autograd.grad(y, x, up)
    want = ref.plain_backward(joint[..., :128].unflatten(-1, (4, 32)), w, 1e-6, up)
    ref.check("dx", dx[..., :128].unflatten(-1, (4, 32)), want["dx"])
    assert not dx[..., 128:].any()


def test_no_rows_and_vectors():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 4, 16, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    assert y.shape == x.shape
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and not dw.any()
    s, n = residual_norm(x, x.detach(), w, gate=torch.empty(0, 4, 1, device="cuda"))
    (dw,) = torch.autograd.grad((s, n), (w,), (torch.empty_like(s), torch.empty_like(n)))
    assert not dw.any()
    v = torch.randn(16, device="cuda")
    ref.check("vector", rms_norm(v, w), ref.plain_forward(v, w, 1e-6, F32))
    s, n = residual_norm(v, v, w)
    assert torch.equal(s, v + v)


def test_zero_rows_infinities_and_nan_stay_in_their_rows():
    x = torch.randn(4, 64, device="cuda")
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    w = torch.ones(64, device="cuda")
    y = rms_norm(x, w)
    assert not y[0].any() and y[1].isnan().any() and y[2].isnan().all() and y[3].isfinite().all()
    s, n = residual_norm(x, torch.zeros_like(x), w)
    assert n[3].isfinite().all() and not n[0].any()


def test_16_bit_weights_get_16_bit_gradients():
    g = _gen(4)
    x, w = _randn(g, (6, 72), BF16).requires_grad_(), (1 + 0.1 * _randn(g, (72,))).bfloat16().requires_grad_()
    y = rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    want = ref.plain_backward(x, w, 1e-6, torch.ones_like(y))
    value, bound = want["dweight"]
    assert dw.dtype == BF16
    ref.check("dweight", dw, (value, bound + ref.HALF[BF16] * (value.abs() + bound)))


def _scalar(h, n, up_h, up_n):
    return float((h.double() * up_h).sum() + (n.double() * up_n).sum())


def test_gradients_against_differences():
    g = _gen(6)
    shape = (2, 3, 40)
    t, _, _, _ = _inputs(9, shape, F32, F32, F32, True, shape, "vector")
    up_h, up_n = _randn(g, shape).double(), _randn(g, shape).double()

    def value(p, double):
        if double:
            p = {k: x.detach().double().cpu() for k, x in p.items()}
            u = p["update"] / ref.rms(p["update"], EPS) * p["post_weight"]
            h = p["residual"] + p["scale"] * torch.sigmoid(p["gate"]) * u
            return _scalar(h, h / ref.rms(h, EPS) * p["weight"], up_h.cpu(), up_n.cpu())
        h, n = residual_norm(p["residual"], p["update"], p["weight"], EPS, post_weight=p["post_weight"],
                             gate=p["gate"], scale=p["scale"])
        return _scalar(h, n, up_h, up_n)

    for x in t.values():
        x.requires_grad_()
    h, n = residual_norm(t["residual"], t["update"], t["weight"], EPS, post_weight=t["post_weight"],
                         gate=t["gate"], scale=t["scale"])
    grads = dict(zip(t, torch.autograd.grad((h, n), list(t.values()), (up_h.float(), up_n.float()))))
    # the difference quotient of the kernel: its outputs carry K U each, divided by the step;
    # the float64 quotients at two steps say how far a quotient is from the derivative
    noise = 2 * ref.K * ref.U * float((h.double().abs() * up_h.abs()).sum() + (n.double().abs() * up_n.abs()).sum())
    for k in t:
        d = _randn(g, t[k].shape)
        base = {j: x.detach() for j, x in t.items()}

        def quotient(step, double):
            a, b = ({**base, k: base[k] + s * step * d} for s in (1, -1))
            return (value(a, double) - value(b, double)) / (2 * step)

        step = 2.0 ** -6
        q64, half64 = quotient(step, True), quotient(step / 2, True)
        along = float((grads[k].double() * d.double()).sum())
        # inputs base + step * d are rounded to fp32: a change of U |x| in each, times the gradient
        moved = float((grads[k].double().abs() * (base[k].abs() + step * d.abs()).double()).sum()) * ref.U / step
        assert abs(quotient(step, False) - q64) <= noise / step + 2 * moved, k
        assert abs(along - half64) <= abs(q64 - half64) + 1e-9 * abs(q64) + moved + noise, k


def test_other_stream_and_repeated_runs_agree():
    t, const, ds, dn = _inputs(8, (7, 33, 320), F32, BF16, BF16, True, (7, 33, 320), "vector")
    for x in t.values():
        x.requires_grad_()

    def step():
        h, n = residual_norm(t["residual"], t["update"], t["weight"], EPS, post_weight=t["post_weight"],
                             gate=t["gate"], scale=t["scale"], out_dtype=BF16)
        return (h, n, *torch.autograd.grad((h, n), list(t.values()), (ds, dn)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_captured_step_replays_on_new_values():
    t, const, ds, dn = _inputs(8, (5, 96), F32, BF16, BF16, True, (5, 96), "vector")
    new, _, _, _ = _inputs(9, (5, 96), F32, BF16, BF16, True, (5, 96), "vector")
    for x in t.values():
        x.requires_grad_()

    def step(p):
        h, n = residual_norm(p["residual"], p["update"], p["weight"], EPS, post_weight=p["post_weight"],
                             gate=p["gate"], scale=p["scale"], out_dtype=BF16)
        return (h.detach(), n.detach(), *torch.autograd.grad((h, n), list(p.values()), (ds, dn)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(t)
    with torch.no_grad():
        for k, x in t.items():
            x.copy_(new[k])
    graph.replay()
    want = step({k: x.detach().requires_grad_() for k, x in new.items()})
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_launches_are_counted():
    n = _lib.launch_count()
    rms_norm(torch.ones(2, 8, device="cuda"), torch.ones(8, device="cuda"))
    assert _lib.launch_count() == n + 1


def test_second_derivatives_are_refused():
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(rms_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


def test_one_tensor_in_two_places_gets_both_gradients():
    g = _gen(20)
    x, w = _randn(g, (5, 72)).requires_grad_(), (1 + 0.1 * _randn(g, (72,))).requires_grad_()
    up = _randn(g, (5, 72))
    s, n = residual_norm(x, x, w, EPS, post_weight=w)
    dx, dw = torch.autograd.grad((s, n), (x, w), (up, up))
    a, b, u, v = (t.detach().clone().requires_grad_() for t in (x, x, w, w))
    parts = torch.autograd.grad(residual_norm(a, b, u, EPS, post_weight=v), (a, b, u, v), (up, up))
    assert torch.equal(dx, parts[0] + parts[1]) and torch.equal(dw, parts[2] + parts[3])


def test_offsets_beyond_32_bits():
    """2^31 values and more: the last rows equal those of a call with these rows alone."""
    rows, width = (1 << 21) + 3, 1024
    x = torch.empty(rows, width, device="cuda", dtype=BF16)
    x[-5:] = _randn(_gen(21), (5, width), BF16)
    x[:-5] = 1
    w = 1 + 0.1 * _randn(_gen(22), (width,))
    assert torch.equal(rms_norm(x, w)[-5:], rms_norm(x[-5:].clone(), w))
    leaf = x.requires_grad_()
    y = rms_norm(leaf, w)
    up = torch.zeros_like(y)
    up[-5:] = x[-5:].detach()
    (dx,) = torch.autograd.grad(y, leaf, up)
    small = x[-5:].detach().clone().requires_grad_()
    (ds,) = torch.autograd.grad(rms_norm(small, w), small, up[-5:])
    assert torch.equal(dx[-5:], ds) and not dx[:-5].any()


def test_tensors_that_move_between_forward_and_backward():
    """As sharded parameters do: the values come back at another address before the backward."""
    g = _gen(30)
    x, w = _randn(g, (6, 80)).requires_grad_(), (1 + 0.1 * _randn(g, (80,))).requires_grad_()
    up = _randn(g, (6, 80))
    want = torch.autograd.grad(rms_norm(x, w), (x, w), up)
    y = rms_norm(x, w)
    s, n = residual_norm(x, x.detach().clone(), w, post_weight=w)  # not the memory spoilt below
    old = x.data, w.data
    with torch.no_grad():
        x.data, w.data = old[0].clone(), old[1].clone()
        for t in old:
            t.fill_(float("nan"))
    for a, b in zip(want, torch.autograd.grad(y, (x, w), up)):
        assert torch.equal(a, b)
    (dw,) = torch.autograd.grad(n, (w,), up)
    assert dw.isfinite().all()


def test_gates_at_the_ends_of_their_range():
    """Closed, open and saturated gates: 0, 1 and the values between, and no NaN from infinities."""
    a = torch.tensor([-float("inf"), -1e30, -200., -88., -87.5, -86., -20., -1., -0., 1e-30, 1., 20., 86., 200.,
                      1e30, float("inf")], device="cuda")
    width = 64
    g = _gen(31)
    h, u = _randn(g, (16, width)), _randn(g, (16, width))
    w = torch.ones(width, device="cuda")
    for gate in (a[:, None].contiguous(), a[:, None].expand(16, width).contiguous()):
        gate.requires_grad_()
        s, n = residual_norm(h, u, w, EPS, gate=gate)
        ref.check("stream", s, ref.stream_of(h, u, None, gate, None, 1.0, EPS))
        assert torch.equal(s[0], h[0]) and torch.equal(s[-1], h[-1] + u[-1])
        (da,) = torch.autograd.grad((s, n), (gate,), (u, u))
        assert da.isfinite().all() and not da[:3].any() and not da[-3:].any()
    nan = torch.full((16, 1), float("nan"), device="cuda")
    assert residual_norm(h, u, w, EPS, gate=nan)[0].isnan().all()


def test_saved_tensors_that_come_back_with_other_strides():
    """Kept on the host between forward and backward, strided inputs come back dense.  The gate then
    starts on 16 bytes, which it does not in place: other sums, the same bounds."""
    g = _gen(32)
    joint, wide = _randn(g, (3, 50, 96), BF16), _randn(g, (3, 50, 200), BF16)
    x, gate = (t.detach().requires_grad_() for t in (joint[..., 16:48], wide[..., 100:132]))
    h, w = _randn(g, (3, 50, 32)), (1 + 0.1 * _randn(g, (32,))).requires_grad_()
    up, upn = _randn(g, (3, 50, 32)), _randn(g, (3, 50, 32), BF16)

    post = w.detach().clone().requires_grad_()

    def step():
        s, n = residual_norm(h, x, w, EPS, gate=gate, post_weight=post)
        y = rms_norm(x, w)
        return s, torch.autograd.grad((s, n), (x, gate, w, post), (up, upn)), torch.autograd.grad(y, (x, w), upn)

    with torch.autograd.graph.save_on_cpu():
        s, parts, plain = step()
    want = ref.backward(s, x, w, post, gate, None, 1.0, EPS, up, upn)
    for name, t in zip(("update", "gate", "weight", "post_weight"), parts):
        ref.check("d" + name, t, want["d" + name])
    for a, b in zip(step()[2], plain):
        assert torch.equal(a, b)


@pytest.mark.parametrize("parts", [False, True])
@pytest.mark.parametrize("width", [24, 64, 1001, 1024, 8200])
def test_infinities_stay_out_of_the_gradient_of_the_stream_alone(width, parts):
    """Only the stream has a gradient: it is the residual's, also in rows that overflowed."""
    g = _gen(33)
    h, u, up = _randn(g, (6, width)), _randn(g, (6, width)), _randn(g, (6, width))
    h[1, 3], h[2, 5] = float("inf"), float("nan")
    h.requires_grad_()
    u.requires_grad_()
    w = torch.ones(width, device="cuda", requires_grad=True)
    s, n = residual_norm(h, u, w, EPS, scale=torch.full((width,), 0.5, device="cuda") if parts else 0.5)
    dh, du = torch.autograd.grad(s, (h, u), up)
    assert torch.equal(dh, up) and torch.equal(du, 0.5 * up)


@pytest.mark.parametrize("width", [40, 1001, 1024])
def test_fp32_gates_near_zero_keep_their_gradients_digits(width):
    """Gates of e^-1 to e^-60, whose gradients shrink with them.  The exponential is within 4 U, the
    reciprocal, the products and 1 - s add 10 U to a gradient of every channel; a row's gate adds
    up positive terms, in at most 26 additions (see norm_reference)."""
    g = _gen(34)
    h, u, up = (_randn(g, (12, width)) for _ in range(3))
    up = up.abs() * u.sign()
    w = torch.ones(width, device="cuda")
    for shape, room in (((12, width), 16), ((12, 1), 16 + 26)):
        a = (-1 - 59 * torch.rand(shape, generator=g)).cuda().requires_grad_()
        s, n = residual_norm(h, u, w, EPS, gate=a)
        (da,) = torch.autograd.grad(s, a, up)
        gate = torch.sigmoid(a.detach().double())
        want = up.double() * u.double() * gate * (1 - gate)
        if shape[1] == 1:
            want = want.sum(-1, keepdim=True)
        assert ((da.double() - want).abs() <= room * ref.U * want.abs()).all(), shape


OTHER_TYPES_FIRST = """
import sys, torch
from gpa_b200 import residual_norm
def step(stream, update, gate, out, width):
    g = torch.Generator().manual_seed(width)
    h, u, a = (torch.randn(4000, width, generator=g).to(t).cuda().requires_grad_() for t in (stream, update, gate))
    w, p, c = ((1 + 0.1 * torch.randn(width, generator=g)).cuda().requires_grad_() for _ in range(3))
    s, n = residual_norm(h, u, w, post_weight=p, gate=a, scale=c, out_dtype=out)
    return torch.autograd.grad((s, n), (w, p, c), (torch.ones_like(s), torch.ones_like(n)))
F, B, H = torch.float32, torch.bfloat16, torch.float16
for width in (384, 768, 1280, 1792, 2560, 4096):
    if sys.argv[1] == "first":
        step(H, H, H, H, width)
    torch.save(step(F, F, B, F, width), f"{sys.argv[2]}/{sys.argv[1]}{width}.pt")
"""


def test_column_sums_do_not_depend_on_earlier_calls(tmp_path):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for order in ("first", "alone"):
        r = subprocess.run([sys.executable, "-c", OTHER_TYPES_FIRST, order, str(tmp_path)], cwd=root,
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
    for width in (384, 768, 1280, 1792, 2560, 4096):
        a, b = (torch.load(f"{tmp_path}/{order}{width}.pt") for order in ("first", "alone"))
        assert all(torch.equal(x, y) for x, y in zip(a, b)), width


@pytest.mark.parametrize("stream,update", [(F32, BF16), (F16, F16)])
@pytest.mark.parametrize("width", WIDTHS)
def test_residual_norm_widths_without_parts(width, stream, update):
    shape = (3, width)
    t, const, ds, dn = _inputs(width, shape, stream, update, update, False, None, "number")
    _check_case(t, const, ds, dn, update)
