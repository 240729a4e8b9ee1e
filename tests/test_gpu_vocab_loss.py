"""linear_cross_entropy on the GPU against float64 on the CPU.

Bounds (U = 2^-24, fp32's rounding; HALF[t] half a step of type t).  A logit is a sum of D exact
products (16-bit inputs; each rounded once more for fp32 ones) whose additions lose at most 2 U of
the running magnitude each, whether they round or truncate: Ez = 2 (D + 2) U sum |x| |w|.  The
loss takes two logits and an exp / log of relative error below 64 U.  A gradient of a logit is
P = exp(z - lse) - [v = y]: its exp part is off by that relative error plus 2 max Ez, and P is
rounded once to the input's type when that has 16 bits.  Each row's own gradient (reduction "none")
multiplies dx in fp32, and the rows that dW takes, rounded to their type.  The products with P then add
2 (n + 2) U sum |P| |w| over their n terms, and the result is rounded once.
"""
from __future__ import annotations

import math

import pytest
import torch

from gpa_b200 import _lib, linear_cross_entropy
from norm_reference import HALF, TINY, U

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(seed, lead, width, vocab, dtype, masked=0.0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*lead, width, generator=g).to(dtype).cuda()
    w = (torch.randn(vocab, width, generator=g) * spread / width ** .5).to(dtype).cuda()
    y = torch.randint(0, vocab, lead, generator=g)
    if masked:
        y[torch.rand(lead, generator=g) < masked] = -100
    return x, w, y.cuda()


def _reference(x, w, y, up, reduction):
    """({name: (value, bound)}) in float64 on the CPU; `up` is the gradient of the loss."""
    dtype, shape = x.dtype, x.shape
    x, w, y = x.detach().double().cpu().flatten(0, -2), w.detach().double().cpu(), y.cpu().flatten()
    keep = y != -100
    xk, yk = x[keep], y[keep]
    n, v, d = xk.shape[0], w.shape[0], w.shape[1]
    z = xk @ w.T
    ez = 2 * (d + 2) * U * (xk.abs() @ w.abs().T)
    worst = ez.amax(-1, keepdim=True) if n else torch.zeros(0, 1, dtype=torch.float64)
    lse = torch.logsumexp(z, -1, keepdim=True)
    picked = z.gather(-1, yk[:, None])
    loss = (lse - picked)[:, 0]
    e_loss = (2 * worst + 64 * U + 4 * U * (lse.abs() + picked.abs()))[:, 0]
    out = {}
    if reduction == "none":
        full, bound = torch.zeros(len(y), dtype=torch.float64), torch.zeros(len(y), dtype=torch.float64)
        full[keep], bound[keep] = loss, e_loss + U * loss.abs()
        out["loss"] = (full, bound)
        g = up.double().cpu().flatten()[keep][:, None]
    else:
        k = max(n, 1) if reduction == "mean" else 1
        out["loss"] = (loss.sum() / k, (e_loss.sum() + 4 * U * loss.abs().sum()) / k)
        g = torch.full((n, 1), float(up) / k, dtype=torch.float64)
    soft = (z - lse).exp()
    hot = torch.zeros_like(z).scatter_(-1, yk[:, None], 1.0)
    ep = soft * (2 * worst + 64 * U) + U * (soft + hot)
    p = soft - hot
    if dtype != F32:
        # rounded once to the type: fp16 underflows at 2^-25 of the scale 2^14 that keeps small
        # probabilities in range
        ep = ep + HALF[dtype] * (p.abs() + ep) + (2.0 ** -39 if dtype == F16 else 0.0)
    p, ep = p * g, ep * g.abs() * (1 + 4 * U)
    dx, ex = p @ w, ep @ w.abs() + 2 * (v + 2) * U * (p.abs() @ w.abs())
    dw, ew = p.T @ xk, ep.T @ xk.abs() + 2 * (n + 2) * U * (p.abs().T @ xk.abs())
    if dtype != F32 and reduction == "none" and n:
        # dW takes the rows times their own gradients, rounded once more (fp16: as shares of the
        # largest gradient, which may fall below its normal range)
        ew = ew + HALF[dtype] * (p.abs().T @ xk.abs()) + TINY[dtype] * g.abs().max() * (soft + hot).sum(0)[:, None]
    fx, fe = torch.zeros_like(x), torch.zeros_like(x)
    fx[keep], fe[keep] = dx, ex + (HALF[dtype] + 4 * U) * (dx.abs() + ex) + TINY[dtype]
    out["dhidden"] = (fx.view(shape), fe.view(shape))
    out["dweight"] = (dw, ew + (HALF[dtype] + 4 * U) * (dw.abs() + ew) + TINY[dtype])
    return out


def _check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu().view(value.shape)
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), bad.numel(),
                           float(((got - value).abs() / bound.clamp_min(1e-300)).max()))


def _run(x, w, y, reduction, seed=0):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction=reduction)
    assert loss.dtype == F32 and loss.shape == (y.shape if reduction == "none" else ())
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, y, reduction=reduction), loss)
    g = torch.Generator().manual_seed(seed + 99)
    up = torch.randn(loss.shape, generator=g).cuda()
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    return loss, dx, dw, up


def _case(seed, lead, width, vocab, dtype, reduction, masked=0.0):
    x, w, y = _inputs(seed, lead, width, vocab, dtype, masked)
    loss, dx, dw, up = _run(x, w, y, reduction, seed)
    want = _reference(x, w, y, up, reduction)
    _check("loss", loss, want["loss"])
    _check("dhidden", dx, want["dhidden"])
    _check("dweight", dw, want["dweight"])


DTYPES = [BF16, F16, F32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead,width,vocab", [
    ((1,), 64, 256), ((1,), 1, 1), ((3, 5), 8, 7), ((2, 130), 128, 500), ((257,), 64, 257), ((255,), 192, 511),
    ((256,), 256, 512), ((3, 171), 72, 1003), ((700,), 40, 300), ((64,), 520, 2000), ((5,), 1000, 1500),
    ((2, 33), 61, 129), ((130,), 1024, 300), ((2, 3, 50), 320, 777), ((1300,), 96, 96), ((40,), 2050, 700),
])
def test_sizes(dtype, lead, width, vocab):
    _case(width + vocab, lead, width, vocab, dtype, "mean")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("masked", [0.0, 0.3, 0.97])
@pytest.mark.parametrize("lead", [(4, 150), (3, 40), (2, 13)])  # the three forms of the products
def test_reductions_and_masks(dtype, reduction, masked, lead):
    _case(11, lead, 136, 900, dtype, reduction, masked)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 127, 128, 129, 256, 257])
def test_rows_round_the_tiles(dtype, rows):
    _case(rows, (rows,), 200, 1290, dtype, "mean")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_labelled_token_and_no_token(dtype, reduction):
    x, w, y = _inputs(3, (2, 9), 64, 300, dtype)
    y.fill_(-100)
    loss, dx, dw, _ = _run(x, w, y, reduction)
    assert not loss.any() and not dx.any() and not dw.any()
    loss, dx, dw, _ = _run(x[:, :0], w, y[:, :0], reduction)
    assert not loss.any() and dx.shape == (2, 0, 64) and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_tokens_are_not_read(dtype):
    x, w, y = _inputs(5, (3, 100), 128, 400, dtype, 0.4)
    want = _run(x, w, y, "mean")
    dirty = x.clone()
    dirty[y == -100] = float("nan")
    got = _run(dirty, w, y, "mean")
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_ignore_index_may_be_a_token():
    x, w, y = _inputs(6, (50,), 64, 100, BF16)
    y[::3] = 7
    other = torch.where(y == 7, -100, y)
    a = linear_cross_entropy(x, w, y, ignore_index=7)
    assert torch.equal(a, linear_cross_entropy(x, w, other))
    assert torch.equal(a, linear_cross_entropy(x, w, other.int()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_label_outside_the_vocabulary_gives_nan_there(dtype):
    x, w, y = _inputs(7, (20,), 64, 100, dtype)
    y[4], y[9] = 100, -3
    loss = linear_cross_entropy(x, w, y, reduction="none")
    assert loss[4].isnan() and loss[9].isnan() and int(loss.isnan().sum()) == 2
    xr = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(linear_cross_entropy(xr, w, y, reduction="sum"), xr)
    rows = dx.isnan().any(-1)
    assert rows[4] and rows[9] and int(rows.sum()) == 2


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_logits(dtype):
    """Logits of +-200 and rows whose probability sits on one entry: finite, and within bounds."""
    x, w, y = _inputs(8, (60,), 64, 513, dtype, spread=60.0)
    loss, dx, dw, up = _run(x, w, y, "none")
    assert loss.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()
    _check("loss", loss, _reference(x, w, y, up, "none")["loss"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_in_one_token_stays_in_its_loss(dtype):
    x, w, y = _inputs(9, (6,), 64, 300, dtype)
    x[2, 5] = float("nan")
    loss = linear_cross_entropy(x, w, y, reduction="none")
    assert loss[2].isnan() and int(loss.isnan().sum()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_inputs(dtype):
    x, w, y = _inputs(10, (3, 40), 96, 333, dtype, 0.2)
    want = _run(x, w, y, "mean")
    wide = torch.zeros(3, 41, 107, device="cuda", dtype=dtype)
    wide[:, :40, 3:99] = x
    tall = torch.zeros(333, 107, device="cuda", dtype=dtype)
    tall[:, 5:101] = w
    strided = (wide[:, :40, 3:99], tall[:, 5:101])
    assert not strided[0].is_contiguous()
    for a, b in zip(want, _run(*strided, y, "mean")):
        assert torch.equal(a, b)
    flipped = w.T.contiguous().T  # no unit stride along the channels
    for a, b in zip(want, _run(x.transpose(0, 1).contiguous().transpose(0, 1), flipped, y, "mean")):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_one_gradient_is_wanted(dtype):
    x, w, y = _inputs(12, (70,), 64, 600, dtype)
    _, dx, dw, _ = _run(x, w, y, "sum")
    up = torch.randn((), generator=torch.Generator().manual_seed(99)).cuda()
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xr, w, y, reduction="sum"), xr, up)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, wr, y, reduction="sum"), wr, up)[0], dw)


def test_many_rows_and_a_large_vocabulary_in_pieces():
    """More rows than one piece of the vocabulary holds: the pieces' gradients add up.  The plain
    form in fp32 on the GPU stands in for float64 here, at bf16's rounding of P and the result."""
    x, w, y = _inputs(13, (2, 4100), 128, 70001, BF16, 0.1)
    loss, dx, dw, up = _run(x, w, y, "mean")
    x, w = x.float().flatten(0, 1), w.float()
    keep = y.flatten() != -100
    z = x @ w.T
    lse = torch.logsumexp(z, -1, keepdim=True)
    at = y.flatten().clamp_min(0)[:, None]
    ref = ((lse - z.gather(-1, at))[:, 0] * keep).sum() / keep.sum()
    assert abs(float(loss - ref)) <= 1e-5 * float(ref)
    z = (z - lse).exp_()
    z.scatter_add_(-1, at, torch.full_like(lse, -1.0))
    z *= (keep.float() / keep.sum())[:, None] * up
    rx, rw = z @ w, z.T @ x
    # two roundings of relative size 2^-8 at most: norm-wise below the sum of both
    assert float((dx.float().flatten(0, 1) - rx).norm() / rx.norm()) <= 2 * HALF[BF16]
    assert float((dw.float() - rw).norm() / rw.norm()) <= 2 * HALF[BF16]


def test_gradient_against_differences():
    """Along random directions in fp32; the float64 quotients at two steps bound the curvature."""
    x, w, y = _inputs(14, (30,), 24, 90, F32, 0.2)
    loss, dx, dw, _ = _run(x, w, y, "mean")
    one = torch.ones((), device="cuda")
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(linear_cross_entropy(xr, wr, y), (xr, wr), one)
    g = torch.Generator().manual_seed(1)
    ex, ew = torch.randn(x.shape, generator=g).cuda(), torch.randn(w.shape, generator=g).cuda()

    def quotient(h, double):
        vals = []
        for s in (1, -1):
            a, b = x + s * h * ex, w + s * h * ew
            if double:
                vals.append(torch.nn.functional.cross_entropy(a.double() @ b.double().T, y))
            else:
                vals.append(linear_cross_entropy(a, b, y).double())
        return float(vals[0] - vals[1]) / (2 * h)

    h = 2.0 ** -6
    q, half = quotient(h, True), quotient(h / 2, True)
    along = float((dx * ex).double().sum() + (dw * ew).double().sum())
    noise = float(_reference(x, w, y, one, "mean")["loss"][1]) * 2
    assert abs(quotient(h, False) - q) <= noise / h
    # inputs x + h e are rounded to fp32 in both quotients: U (|x| + h |e|) times the gradient
    moved = U / h * float((dx.abs() * (x.abs() + ex.abs())).sum() + (dw.abs() * (w.abs() + ew.abs())).sum())
    assert abs(along - half) <= abs(q - half) + 2 * moved + 1e-6 * abs(q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_stream_repeats_and_replays(dtype):
    x, w, y = _inputs(15, (2, 200), 192, 1100, dtype, 0.1)
    x2, w2, y2 = _inputs(16, (2, 200), 192, 1100, dtype, 0.5)
    want, want2 = _run(x, w, y, "mean"), _run(x2, w2, y2, "mean")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(x, w, y, "mean")
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    sx, sw, sy, up = x.clone().requires_grad_(), w.clone().requires_grad_(), y.clone(), want[3]

    def step():
        loss = linear_cross_entropy(sx, sw, sy)
        return (loss.detach(), *torch.autograd.grad(loss, (sx, sw), up))

    graphs = []
    for _ in range(2):  # two graphs of the same step: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for values, ref in (((x2, w2, y2), want2), ((x, w, y), want)):
        with torch.no_grad():
            for s, v in zip((sx, sw, sy), values):
                s.copy_(v)
        for graph, _ in graphs:
            graph.replay()
        for _, got in graphs:
            for a, b in zip(got, ref):
                assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    x, w, y = _inputs(17, (9,), 32, 50, F32)
    x.requires_grad_()
    (g,) = torch.autograd.grad(linear_cross_entropy(x, w, y), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


@pytest.mark.parametrize("lead", [(300,), (20,)])
def test_two_streams_at_once(lead):
    cases = [_inputs(30 + i, lead, 256, 5000, BF16, 0.1) for i in range(2)]
    want = [_run(*c, "mean") for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                x, w = (t.detach().requires_grad_() for t in c[:2])
                loss = linear_cross_entropy(x, w, c[2])
                got[i].append((loss.detach(), *torch.autograd.grad(loss, (x, w), want[i][3])))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """More than 2^31 values of hidden, and of the weight: the tokens and entries at the far end."""
    n, d, v = (1 << 21) + 70, 1024, 300
    x = torch.zeros(n, d, device="cuda", dtype=BF16)
    xs, w, ys = _inputs(40, (70,), d, v, BF16)
    x[-70:] = xs
    y = torch.full((n,), -100, device="cuda")
    y[-70:] = ys
    y[0] = 1
    loss = linear_cross_entropy(x, w, y, reduction="none")
    want = linear_cross_entropy(xs, w, ys, reduction="none")
    # the same logits through differently cut sums: two fp32 results of the same exact value
    bound = 2 * _reference(xs, w, ys, torch.zeros(70), "none")["loss"][1]
    assert ((loss[-70:] - want).abs().double().cpu() <= bound).all() and not loss[1:-70].any()
    del x
    v = (1 << 21) + 300
    w = torch.zeros(v, d, device="cuda", dtype=BF16)
    xs, end, ys = _inputs(41, (9,), d, 300, BF16)
    w[-300:] = end
    wr = w.requires_grad_()
    ys = ys + (v - 300)
    loss = linear_cross_entropy(xs, wr, ys, reduction="none")
    z = xs.double() @ end.detach().double().T
    z = torch.cat((z, z.new_zeros(9, 1)), 1)  # every other entry has the logit 0
    z[:, -1] += torch.log(torch.tensor(float(v - 300), dtype=torch.float64))
    ref = torch.nn.functional.cross_entropy(z, ys - (v - 300), reduction="none")
    ez = 2 * (d + 2) * U * (xs.double().abs() @ end.double().abs().T).amax(-1)
    # beside the logits' errors: 2^21 equal terms, each within 64 U, added in any order
    assert ((loss.double() - ref).abs() <= 2 * ez + 200 * U + 8 * U * ref.abs()).all()
    (dw,) = torch.autograd.grad(loss.sum(), wr)
    p = torch.softmax(z, -1)[:, :300] - torch.nn.functional.one_hot(ys - (v - 300), 300)
    want = p.T @ xs.double()
    off = HALF[BF16] * (p.abs().T @ xs.double().abs()) * 1.1 + HALF[BF16] * want.abs()
    assert ((dw[-300:].double() - want).abs() <= off).all()


FIRST_CALL_IN_A_CAPTURE = """
import torch
from gpa_b200 import linear_cross_entropy, residual_norm
g = torch.Generator().manual_seed(0)
x = torch.randn(300, 128, generator=g).bfloat16().cuda().requires_grad_()
h = torch.randn(300, 128, generator=g).cuda().requires_grad_()
w = torch.randn(700, 128, generator=g).bfloat16().cuda().requires_grad_()
n = torch.ones(128, device="cuda", requires_grad=True)
y = torch.randint(0, 700, (300,), generator=g).cuda()
def step():
    s, m = residual_norm(h, x, n)
    loss = linear_cross_entropy(m, w, y) + s.float().mean()
    return (loss.detach(), *torch.autograd.grad(loss, (x, h, w, n)))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
for a, b in zip(got, step()):
    assert torch.equal(a, b)
print("captured")
"""


def test_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], cwd=root, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_no_tensor_core_kernel_timed_out():
    assert _lib.device_status() == 0


def _spoil(nbytes):
    """Memory that the next allocations get, filled with NaN."""
    torch.cuda.empty_cache()
    for size in nbytes:
        torch.full((max(1, size // 4),), float("nan"), device="cuda")
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,labelled,width,vocab", [
    (16, 16, 1024, 7000), (100, 100, 640, 8000), (200, 200, 384, 28996), (16, 16, 256, 6200), (100, 90, 512, 28996),
    (512, 512, 512, 7000), (768, 768, 512, 7000), (4096, 200, 1024, 7000),
])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_nothing_of_the_scratch_reaches_the_gradients(rows, labelled, width, vocab, dtype, reduction):
    """Vocabularies that end in the last tile's first blocks of 64: the parts of dhidden that are
    added up are all written.  The workspaces come from memory full of NaN."""
    x, w, y = _inputs(rows + vocab, (rows,), width, vocab, dtype)
    y[torch.randperm(rows, generator=torch.Generator().manual_seed(1)).cuda()[labelled:]] = -100
    xr, wr = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(xr, wr, y, reduction=reduction)
    up = torch.randn(loss.shape, generator=torch.Generator().manual_seed(2)).cuda()
    _spoil([1 << 30])
    dx, dw = torch.autograd.grad(loss, (xr, wr), up)
    want = _reference(x, w, y, up, reduction)
    _check("dhidden", dx, want["dhidden"])
    _check("dweight", dw, want["dweight"])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead", [(40,), (300,)])
def test_saved_tensors_that_come_back_with_other_strides(lead, dtype):
    """Kept on the host between forward and backward, a strided weight comes back dense."""
    x, w, y = _inputs(18, lead, 64, 700, dtype)
    wide = torch.zeros(700, 208, device="cuda", dtype=dtype)
    wide[:, 16:80] = w
    want = _run(x, w, y, "none")
    with torch.autograd.graph.save_on_cpu():
        got = _run(x, wide[:, 16:80], y, "none")
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_no_token_and_a_frozen_weight(dtype, reduction):
    x, w, y = _inputs(19, (0,), 64, 300, dtype)
    x.requires_grad_()
    loss = linear_cross_entropy(x, w, y, reduction=reduction)
    (dx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
    assert dx.shape == (0, 64) and dx.dtype == dtype


@pytest.mark.parametrize("dtype,rows", [(F16, 8193), (F16, 1 << 18), (BF16, 65537), (BF16, 1 << 20), (F32, 1 << 18)])
@pytest.mark.parametrize("width,vocab", [(64, 64), (40, 300)])
def test_weight_gradient_over_very_many_rows(dtype, rows, width, vocab):
    """Sums of one sign over the rows: entry 0 is nobody's label.  P is off by the logits' error and
    half a step of its type, dW is rounded once more; in between an accumulator loses at most 2^-23
    of itself with each 16 rows, over 8192 of them at a time (fp16; fp32 less), and these are added
    with at most one rounding each: 2^-14 + rows / 8192 U.  bf16 adds 65536 at a time: 2^-11."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = (0.5 + torch.rand(rows, width, generator=g, device="cuda")).to(dtype)
    w = (torch.randn(vocab, width, generator=g, device="cuda") * 0.05).to(dtype).requires_grad_()
    y = torch.randint(1, vocab, (rows,), generator=g, device="cuda")
    (dw,) = torch.autograd.grad(linear_cross_entropy(x, w, y), w)
    wd = w.detach().double()
    want, size, worst = torch.zeros_like(wd), torch.zeros_like(wd), 0.0
    for i in range(0, rows, 1 << 16):
        xd, yd = x[i:i + (1 << 16)].double(), y[i:i + (1 << 16), None]
        worst = max(worst, 2 * (width + 2) * U * float((xd @ wd.abs().T).amax()))
        p = torch.softmax(xd @ wd.T, -1)
        full = p.scatter_add(1, yd, torch.ones_like(yd, dtype=torch.float64))  # softmax + onehot
        want += (p.scatter_add(1, yd, -torch.ones_like(yd, dtype=torch.float64))).T @ xd / rows
        size += full.T @ xd / rows
    kept = 0.0 if dtype == F32 else 2.0 ** -14 if dtype == F16 else 2.0 ** -11
    off = 2 * worst + 64 * U + HALF[dtype] + kept + (rows / 8192 + 4) * U + (1024 * U if dtype == F32 else 0.0)
    bound = off * size + HALF[dtype] * want.abs() + TINY[dtype]
    assert ((dw.double() - want).abs() <= bound).all(), float(((dw.double() - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,width", [(20, 64), (100, 64), (300, 64), (300, 1500), (20, 1500)])
@pytest.mark.parametrize("big", [300.0, 1000.0, 3000.0, 20000.0])
def test_a_token_that_has_all_the_probability(dtype, rows, width, big):
    """One entry's logit is big x for 0.3 < x < 1, every other one 0: the loss is 0 and so are the
    gradients.  An exp2 of a value near 0 and its correction are within 4 U of 1 each, their
    product, the sum of one term, its log and reciprocal within 8 more: 16 U of a probability.  The
    2999 entries of logit 0 have at most e^(-0.3 big) each, 2.5e-36 in all at 300: fp32 holds that."""
    g = torch.Generator().manual_seed(int(big))
    x = torch.zeros(rows, width)
    x[:, 0] = 0.3 + 0.7 * torch.rand(rows, generator=g)
    w = torch.randn(3000, width, generator=g) * 0.5
    w[:, 0] = 0
    w[1234] = 0
    w[1234, 0] = big
    x, w, y = x.to(dtype).cuda(), w.to(dtype).cuda(), torch.full((rows,), 1234).cuda()
    for label, expected in ((1234, 0.0), (77, 1.0)):
        y.fill_(label)
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = linear_cross_entropy(xr, wr, y, reduction="none")
        want = x[:, 0].double() * w[1234, 0].double() * expected
        assert ((loss.double() - want).abs() <= 16 * U + 2 * U * want).all()
        dx, dw = torch.autograd.grad(loss.sum(), (xr, wr))
        # of each row: (P - hot) w over the two entries that matter
        p = expected * (w[1234].double() - w[label].double())
        off = (16 * U + HALF[dtype]) * expected + 16 * U
        assert ((dx.double() - p).abs() <= off * (w[1234].abs() + w[label].abs()).double() +
                HALF[dtype] * p.abs() + TINY[dtype] + 3000 * math.exp(-0.3 * big) * w.abs().double().amax()).all()
        total = x.double().abs().sum(0)
        assert (dw[1234].double().abs() <= expected * total * (1 + 1e-2) + 16 * U * total + TINY[dtype]).all()


@pytest.mark.parametrize("rows,width,vocab", [
    (1, 1, 1), (1, 4, 5), (7, 3, 63), (8, 128, 64), (8, 6144, 700), (8, 6200, 300), (9, 130, 65), (9, 3100, 500),
    (16, 1001, 5003), (16, 3200, 129), (17, 1500, 1187), (17, 1700, 300), (31, 64, 4800), (32, 2900, 333),
    (32, 3200, 333), (32, 127, 9999), (12, 3700, 300), (32, 1792, 400), (32, 1793, 400), (8, 7168, 200), (8, 7200, 200),
])
@pytest.mark.parametrize("masked", [0.0, 0.5])
def test_few_fp32_rows(rows, width, vocab, masked):
    """Rows of one block and of two, what fits shared memory and what does not, sizes off every unit."""
    _case(rows + width, (rows,), width, vocab, F32, "mean", masked)


def test_few_fp32_rows_of_strided_and_spoilt_tensors():
    x, w, y = _inputs(50, (3, 9), 96, 777, F32, 0.3)
    want = _run(x, w, y, "none")
    wide, tall = (torch.full(shape, float("nan"), device="cuda") for shape in ((3, 11, 107), (777, 131)))
    wide[:, 1:10, 3:99], tall[:, 7:103] = x, w  # neither starts on 16 bytes; NaN all round
    for a, b in zip(want, _run(wide[:, 1:10, 3:99], tall[:, 7:103], y, "none")):
        assert torch.equal(a, b)
    dirty = x.clone()
    dirty[y == -100] = float("inf")
    for a, b in zip(want, _run(dirty, w, y, "none")):
        assert torch.equal(a, b)
    broken = w.clone()
    broken[5, 3] = float("nan")
    loss = linear_cross_entropy(x, broken, y, reduction="none")
    assert (loss.isnan() == (y != -100)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead", [(20,), (60,), (300,)])
def test_gradients_of_extreme_logits(lead, dtype):
    """Some entries have no probability above 2^-126 in any row: exp2 and the tensor cores' sums hold
    no smaller numbers, so each P may be off by that much, beside the bounds of other logits."""
    x, w, y = _inputs(8, lead, 64, 513, dtype, spread=60.0)
    loss, dx, dw, up = _run(x, w, y, "none")
    want = _reference(x, w, y, up, "none")
    xd, wd, g = x.double().cpu(), w.double().cpu(), up.double().cpu()[:, None].abs()
    (vx, bx), (vw, bw) = want["dhidden"], want["dweight"]
    _check("dhidden", dx, (vx, bx + 2.0 ** -126 * g * wd.abs().sum(0)))
    _check("dweight", dw, (vw, bw + 2.0 ** -126 * (g * xd.abs()).sum(0)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead", [(5,), (20,), (100,), (300,)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_captured_steps_of_every_form_replay(lead, dtype, reduction):
    """Each form of the products, captured and replayed on new values, equals eager calls."""
    x, w, y = _inputs(60, lead, 72, 700, dtype, 0.2)
    other = _inputs(61, lead, 72, 700, dtype, 0.5)
    up = torch.randn(lead if reduction == "none" else (), generator=torch.Generator().manual_seed(1)).cuda()

    def step(x, w, y):
        loss = linear_cross_entropy(x, w, y, reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), up))

    held = x.clone().requires_grad_(), w.clone().requires_grad_(), y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for values in (other, (x, w, y)):
        with torch.no_grad():
            for a, b in zip(held, values):
                a.copy_(b)
        graph.replay()
        want = step(*(t.clone().requires_grad_() for t in values[:2]), values[2])
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_very_many_rows_without_labels(dtype):
    n = (1 << 16) + 300
    x, w, y = _inputs(62, (n,), 24, 90, dtype)
    keep = torch.randperm(n, generator=torch.Generator().manual_seed(2))[:200].cuda()
    few = torch.full_like(y, -100)
    few[keep] = y[keep]
    loss, dx, dw, up = _run(x, w, few, "mean")
    order = few != -100
    _, sx, sw, _ = _run(x[order], w, few[order], "mean")
    assert torch.equal(dw, sw) and torch.equal(dx[order], sx) and not dx[~order].any()
    loss, dx, dw, up = _run(x, w, torch.full_like(y, -100), "mean")
    assert not loss and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [10, 50, 150])
def test_weight_gradient_of_odd_rows_in_turns(rows, dtype):
    """dW of rows that are no multiple of 8 channels passes through padded ones, 512 MB at a time: the
    same values as of rows that are padded with zeros to begin with, which stay where they are."""
    x, w, y = _inputs(rows, (rows,), 4001, 70001, dtype, 0.2)
    loss, dx, dw, _ = _run(x, w, y, "mean")
    wide = [torch.nn.functional.pad(t, (0, 7)) for t in (x, w)]
    got = _run(*wide, y, "mean")
    assert torch.equal(loss, got[0]) and torch.equal(dx, got[1][:, :-7]) and torch.equal(dw, got[2][:, :-7])
    assert not got[1][:, -7:].any() and not got[2][:, -7:].any()
