"""group_norm_act on the GPU against the definition in 64 bits.

Bounds, with h = 2^-24, counted operation by operation (mean and rstd are fp64 in the kernel):
  xhat: the difference (two operations), rstd, the product: 4 h |xhat|;   z = xhat gamma + beta: err_z = h (6 |gamma xhat| + |z|)
  act: its largest slope (1.13) times err_z, and 12 h (|z| + |y|) of its own evaluation (exp, erf, a division; 1 + erf cancels)
  dz = dy act'(z): |dy| (12 h (1 + |z|) + 1.6 err_z)      (the second derivatives stay below 1.6 in magnitude; none and ReLU: 0)
  sums: of products good to 8 h, at most 300 additions one after the other in fp32 (a thread's rows, the tree)
  dx = rstd (gamma dz - s1 - xhat s2): the parts' errors and 8 h of each part
and half a step of the type the result is stored in."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
ACTS = [None, "relu", "silu", "gelu"]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def act64(z, act):
    """(y, dy/dz) in 64 bits."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def stored(err, want, dtype):
    return err + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (want.abs() + err) + (2.0 ** -25 if dtype == torch.float16 else 0))


def reference(x, groups, weight, bias, eps, act, dy=None):
    """{name: (value, bound)} in 64 bits; x, dy [n, c, *]."""
    n, c = x.shape[:2]
    one = torch.ones(c, dtype=torch.float64, device=x.device)
    gamma, beta = (weight.double() if weight is not None else one)[:, None], (bias.double() if bias is not None else 0 * one)[:, None]
    v = x.double().reshape(n, groups, -1)
    mean = v.mean(2, keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(2, keepdim=True) + eps)
    xhat = ((v - mean) * rstd).reshape(n, c, -1)
    z = xhat * gamma + beta
    y, slope = act64(z, act)
    err_z = H * (6 * (gamma * xhat).abs() + z.abs())
    err_y = 1.13 * err_z + (0 if act in (None, "relu") else 12 * H * (z.abs() + y.abs()))
    out = {"y": (y, stored(err_y, y, x.dtype))}
    if dy is None:
        return out
    d = dy.double().reshape(n, c, -1)
    dz = d * slope
    err_dz = 0 * dz if act in (None, "relu") else d.abs() * (12 * H * (1 + z.abs()) + 1.6 * err_z)
    add = 300 * H
    err_b = err_dz.sum((0, 2)) + add * dz.abs().sum((0, 2))
    err_w = (err_dz * xhat.abs()).sum((0, 2)) + (add + 8 * H) * (dz * xhat).abs().sum((0, 2))
    wt = weight.dtype if weight is not None else torch.float32
    out["dbias"] = (dz.sum((0, 2)), stored(err_b, dz.sum((0, 2)), wt))
    out["dweight"] = ((dz * xhat).sum((0, 2)), stored(err_w, (dz * xhat).sum((0, 2)), wt))
    g = lambda t: t.reshape(n, groups, -1).mean(2, keepdim=True)
    up = lambda t: t.expand(n, groups, v.shape[2]).reshape(n, c, -1)
    dh = gamma * dz
    s1, s2 = up(g(dh)), up(g(dh * xhat))
    e1 = up(g(gamma.abs() * err_dz)) + add * up(g(dh.abs()))
    e2 = up(g(gamma.abs() * err_dz * xhat.abs())) + (add + 8 * H) * up(g((dh * xhat).abs()))
    r = up(rstd)
    dx = r * (dh - s1 - xhat * s2)
    err = r * (gamma.abs() * err_dz + e1 + xhat.abs() * e2 + 8 * H * (dh.abs() + s1.abs() + 2 * (xhat * s2).abs()))
    out["dx"] = (dx, stored(err, dx, x.dtype))
    return out


def channels_last(t):
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def make(dev, shape, dtype, seed=0, offset=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = shape[1]
    view = (1, c) + (1,) * (len(shape) - 2)
    x = torch.randn(shape, generator=gen, device=dev) * 1.5 + offset * torch.randn(c, generator=gen, device=dev).view(view)
    dy = torch.randn(shape, generator=gen, device=dev)
    w, b = 1 + 0.3 * torch.randn(c, generator=gen, device=dev), 0.3 * torch.randn(c, generator=gen, device=dev)
    return channels_last(x.to(dtype)), channels_last(dy.to(dtype)), w, b


def check(got, want, label=""):
    value, bound = want
    err = (got.detach().double().reshape(value.shape) - value).abs()
    fine, worst = bool(got.isfinite().all()), float((err / bound.clamp(min=1e-300)).max())
    assert fine and worst <= 1.0, (label, worst)


def run_both(x, groups, w, b, act, dy, eps=1e-5):
    from geomae_amd import ops
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps, act)
    have = [t for t in leaves if t is not None]
    grads = dict(zip([k for k, t in zip(("dx", "dweight", "dbias"), leaves) if t is not None], torch.autograd.grad(y, have, dy)))
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(x, groups, w, b, eps, act), y)
    return {"y": y, **grads}


SHAPES = [((1, 1, 1, 1), 1), ((2, 6, 1, 1), 3), ((1, 32, 1), 32), ((3, 32, 2), 1), ((2, 37, 5, 7), 1), ((2, 38, 5, 7), 19),
          ((3, 90, 11, 13), 9), ((2, 128, 33, 17), 32), ((1, 256, 64), 8), ((4, 256, 7, 9), 32), ((1, 2056, 3, 5), 8),
          ((2, 1030, 2, 2), 5), ((70, 24), 3), ((300, 8, 3), 2), ((5000, 16), 4), ((2, 64, 3, 4, 5), 16), ((2, 1024, 6), 1024),
          ((1, 16, 90, 101), 2), ((1, 8, 257, 129), 1), ((1, 3, 100, 100), 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=[f"{'x'.join(map(str, s))}g{g}" for s, g in SHAPES])
def test_matches_the_definition(dev, shape, groups, dtype):
    x, dy, w, b = make(dev, shape, dtype)
    for act in ACTS:
        want = reference(x, groups, w, b, 1e-5, act, dy)
        got = run_both(x, groups, w, b, act, dy)
        for k in want:
            check(got[k], want[k], (act, k))
        assert got["y"].dtype == dtype and got["y"].stride() == x.stride() or 1 in shape


def test_gradient_is_the_difference_quotient(dev):
    """d loss along a direction, by central differences of the 64-bit definition, against the kernel's dx, dweight, dbias."""
    x, dy, w, b = make(dev, (2, 24, 6, 5), torch.float32)
    gen = torch.Generator(device=dev).manual_seed(9)
    for act in (None, "silu", "gelu"):
        got = run_both(x, 4, w, b, act, dy)
        for k, base in (("dx", x), ("dweight", w), ("dbias", b)):
            v = torch.randn(base.shape, generator=gen, device=dev).double()

            def loss(t):
                a = {"dx": x.double(), "dweight": w.double(), "dbias": b.double()}
                a[k] = base.double() + t * v
                return (reference(a["dx"], 4, a["dweight"], a["dbias"], 1e-5, act)["y"][0] * dy.double().reshape(2, 24, -1)).sum()
            slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
            mine = (got[k].double() * v).sum()
            # the quotient's own error is of second order (1e-8 of the third derivative, some hundred terms of order 10)
            assert abs(float(mine - slope)) <= 1e-5 * float((got[k].double() * v).abs().sum()) + 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_large_mean_and_no_variance(dev, dtype):
    """A mean a thousand times the spread; groups whose elements are all equal (rstd = 1 / sqrt(eps))."""
    x, dy, w, b = make(dev, (2, 16, 20, 20), torch.float32)
    x = channels_last((x + 1000.0).to(dtype))
    for act in ACTS:
        want = reference(x, 4, w, b, 1e-5, act, dy.to(dtype))
        got = run_both(x, 4, w, b, act, dy.to(dtype))
        for k in want:
            check(got[k], want[k], (act, k))
    flat = channels_last(torch.full((2, 16, 5, 5), 3.25, device=dev, dtype=dtype))
    got = run_both(flat, 4, w, b, None, channels_last(dy[:, :, :5, :5].to(dtype)))
    check(got["y"], reference(flat, 4, w, b, 1e-5, None)["y"])
    assert got["dx"].isfinite().all()


def test_relu_border_is_decided_in_64_bits(dev):
    """2 x 10^7 elements: every element's mask in dx is the definition's (an fp32 z would miss a few)."""
    x, dy, w, b = make(dev, (2, 128, 280, 280), torch.float32, seed=3)
    w[5], w[6] = 0.0, -0.7
    got = run_both(x, 32, w, b, "relu", dy)
    want = reference(x, 32, w, b, 1e-5, "relu", dy)
    for k in want:
        check(got[k], want[k], k)


def test_parameters_none_frozen_and_16_bit(dev):
    from geomae_amd import ops
    x, dy, w, b = make(dev, (2, 24, 9, 7), torch.bfloat16)
    for ww, bb in ((None, None), (w, None), (w.bfloat16(), b.bfloat16()), (w.half(), b.half())):
        for act in ("relu", "gelu"):
            want, got = reference(x, 6, ww, bb, 1e-5, act, dy), run_both(x, 6, ww, bb, act, dy)
            for k in got:
                check(got[k], want[k], (act, k))
                assert k in ("y", "dx") or got[k].dtype == ww.dtype
    xl = x.detach().requires_grad_()
    y = ops.group_norm_act(xl, 6, w, b.requires_grad_(), activation="silu")     # the weight is frozen
    y.backward(dy)
    assert w.grad is None and xl.grad is not None and b.grad is not None
    x2 = x.detach()                                                        # only a parameter wants a gradient
    ops.group_norm_act(x2, 6, w.requires_grad_(), None, activation="silu").backward(dy)
    check(w.grad, reference(x, 6, w, None, 1e-5, "silu", dy)["dweight"])


def test_any_alignment_and_gradient_layout(dev):
    """x at an odd element of its storage; dy contiguous instead of channels-last, and expanded."""
    for dtype in (torch.float32, torch.bfloat16):
        x, dy, w, b = make(dev, (2, 24, 9, 7), dtype)
        buf = torch.empty(x.numel() + 3, dtype=dtype, device=dev)
        xo = buf[1:1 + x.numel()].view(2, 9, 7, 24).movedim(-1, 1)
        xo.copy_(x)
        want = reference(x, 6, w, b, 1e-5, "silu", dy)
        got = run_both(xo, 6, w, b, "silu", dy.contiguous())
        for k in want:
            check(got[k], want[k], k)
    ones = torch.ones((), device=dev).expand(2, 24, 9, 7)
    x, _, w, b = make(dev, (2, 24, 9, 7), torch.float32)
    got, want = run_both(x, 6, w, b, "silu", ones), reference(x, 6, w, b, 1e-5, "silu", ones)
    for k in want:
        check(got[k], want[k], k)


def test_streamed_past_the_caches_at_any_alignment(dev):
    """Over 64 MB (the form that loads and stores past the caches), x at an odd element, rows that end inside a tile of loads."""
    for dtype, shape, groups in ((torch.bfloat16, (1, 72, 701, 701), 9), (torch.float32, (1, 36, 701, 701), 6), (torch.float16, (2, 30, 801, 801), 3)):
        n, c, h, w = shape
        _, _, wt, b = make(dev, (1, c, 1, 1), torch.float32)
        buf = torch.randn(n * c * h * w + 3, device=dev).to(dtype)
        gbuf = torch.randn(n * c * h * w + 1, device=dev).to(dtype)
        x, dy = buf[3:].view(n, h, w, c).movedim(-1, 1), gbuf[1:].view(n, h, w, c).movedim(-1, 1)
        want, got = reference(x, groups, wt, b, 1e-5, "gelu", dy), run_both(x, groups, wt, b, "gelu", dy)
        for k in want:
            check(got[k], want[k], (dtype, k))


def test_no_second_derivative(dev):
    from geomae_amd import ops
    x, dy, w, b = make(dev, (2, 24, 9, 7), torch.float32)
    x = x.detach().requires_grad_()
    dx, = torch.autograd.grad(ops.group_norm_act(x, 6, w, b, activation="silu"), x, dy, create_graph=True)
    check(dx, reference(x.detach(), 6, w, b, 1e-5, "silu", dy)["dx"])
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.sum().backward()


def test_input_changed_before_the_backward_pass_is_noticed(dev):
    from geomae_amd import ops
    x, dy, w, b = make(dev, (2, 24, 9, 7), torch.float32)
    w.requires_grad_()
    y = ops.group_norm_act(x, 6, w, b, activation="silu")
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_empty_batches(dev):
    from geomae_amd import ops
    w, b = torch.ones(8, device=dev, requires_grad=True), torch.zeros(8, device=dev, requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = channels_last(torch.zeros(shape, device=dev)).requires_grad_()
        y = ops.group_norm_act(x, 2, w, b, activation="relu")
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(shape, device=dev))
        assert dx.shape == shape and not dw.any() and not db.any()


def test_nonfinite_values_stay_in_their_group(dev):
    from geomae_amd import ops
    x, _, w, b = make(dev, (3, 24, 9, 7), torch.float32)
    for bad in (float("nan"), float("inf")):
        z = x.clone(memory_format=torch.preserve_format)
        z[1, 5, 2, 3] = bad                                                 # sample 1, group 1
        y = ops.group_norm_act(z, 6, w, b, activation="silu")
        clean = ops.group_norm_act(x, 6, w, b, activation="silu")
        hit = torch.zeros(3, 24, dtype=torch.bool, device=dev)
        hit[1, 4:8] = True
        assert torch.equal(y[~hit], clean[~hit]) and not y[1, 5, 2, 3].isfinite()


def test_results_repeat_bit_for_bit_and_on_other_streams(dev):
    x, dy, w, b = make(dev, (4, 128, 50, 50), torch.float32)
    x2, dy2, w2, b2 = make(dev, (2, 256, 25, 25), torch.bfloat16, seed=1)
    first, second = run_both(x, 32, w, b, "gelu", dy), run_both(x2, 8, w2, b2, "relu", dy2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, args in zip(streams, ((x, 32, w, b, "gelu", dy), (x2, 8, w2, b2, "relu", dy2))):
            with torch.cuda.stream(st):
                got.append(run_both(*args))
        torch.cuda.synchronize()
        for want, g in zip((first, second), got):
            assert all(torch.equal(want[k], g[k]) for k in want)


def test_captured_passes(dev):
    """Forward and backward of two sizes in two captured graphs, replayed in turn with eager work between, on new inputs."""
    from geomae_amd import ops
    sets = []
    for shape, groups, act in (((4, 128, 40, 40), 32, "relu"), ((100, 16, 3), 4, "gelu")):
        x, dy, w, b = make(dev, shape, torch.float32)
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation=act), leaves, dy)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], activation=act)
            grads = torch.autograd.grad(y, leaves, dy)
        y = y.detach()
        sets.append((shape, groups, act, leaves, dy, graph, y, grads))
    for r in range(4):
        for i, (shape, groups, act, leaves, dy, graph, y, grads) in enumerate(sets):
            x, d, w, b = make(dev, shape, torch.float32, seed=10 + 2 * r + i)
            with torch.no_grad():
                for t, v in zip((*leaves, dy), (x, w, b, d)):
                    t.copy_(v)
            graph.replay()
        for shape, groups, act, leaves, dy, graph, y, grads in sets:
            want = run_both(leaves[0].detach(), groups, leaves[1].detach(), leaves[2].detach(), act, dy)
            assert torch.equal(want["y"], y)
            assert all(torch.equal(want[k], g) for k, g in zip(("dx", "dweight", "dbias"), grads))


def test_offsets_past_32_bits(dev):
    """Two samples of 1.1 x 2^31 elements: the second, whose elements all lie past 2^31, is what it is alone."""
    from geomae_amd import ops
    rows = 295_280_000
    x = torch.empty(2, rows, 8, dtype=torch.bfloat16, device=dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    for i in range(2):
        for k in range(0, rows, 1 << 25):
            part = x[i, k:k + (1 << 25)]
            part.copy_(torch.randn(part.shape, generator=gen, device=dev, dtype=torch.bfloat16))
    w, b = torch.ones(8, device=dev), torch.zeros(8, device=dev)
    x = x.movedim(-1, 1)
    y = ops.group_norm_act(x, 2, w, b, activation="relu")
    alone = ops.group_norm_act(x[1:], 2, w, b, activation="relu")
    # (two samples share the launch's workgroups, one has them alone: the sums are cut elsewhere, fp64 keeps that below a rounding
    # of the result for all but a few elements)
    differ = (y[1:] != alone).sum()
    assert int(differ) <= 1e-6 * rows * 8 and torch.allclose(y[1, :, -1000:].float(), alone[0, :, -1000:].float(), rtol=2 ** -7)


def test_module_and_refusals(dev):
    from geomae_amd import ops
    from geomae_amd.norm import GroupNormAct
    x = torch.randn(2, 8, 5, 6, device=dev, requires_grad=True)             # contiguous: the module copies it
    m = GroupNormAct(8, 4, activation="silu").to(dev)
    y = m(x)
    assert y.is_contiguous(memory_format=torch.channels_last)
    check(y, reference(x.detach(), 4, m.weight, m.bias, 1e-5, "silu")["y"])
    y.sum().backward()
    assert x.grad.shape == x.shape and m.weight.grad is not None
    cl = channels_last(x.detach())
    for args, match in (((x.detach(), 4), "channels-last"), ((cl.double(), 4), "float32"), ((cl, 3), "divide"), ((cl, 0), "divide"),
                        ((cl[:, :, ::2], 4), "channels-last"), ((torch.zeros(8, device=dev), 2), r"\[N, C"),
                        ((cl, 4, torch.ones(7, device=dev)), "weight must be"), ((cl, 4, torch.ones(8)), "weight must be a CUDA"),
                        ((cl, 4, None, torch.ones(8, device=dev)), "needs a weight"),
                        ((cl, 4, torch.ones(8, device=dev), torch.ones(8, device=dev).half()), "one dtype"),
                        ((cl, 4, None, None, -1.0), "eps"), ((cl, 4, None, None, 1e-5, "tanh"), "activation")):
        with pytest.raises(RuntimeError, match=match):
            ops.group_norm_act(*args)
    from geomae_amd._lib import GeomaeLibraryError
    with pytest.raises(GeomaeLibraryError, match="at most 1024"):
        ops.group_norm_act(torch.zeros(1, 2048, device=dev), 2048)


def test_capture_beside_a_graph_of_eager_work_is_refused(dev):
    """A backward pass in a capture, while eager work on the default stream holds the gradient of the same weight, is an error
    that leaves the process and the stream usable; once that work is released the capture succeeds."""
    from geomae_amd import _lib, ops
    on_default = _lib.host().accumulates_on_default_stream
    x, dy, w, b = make(dev, (2, 16, 8, 8), torch.float32)
    w, b = w.requires_grad_(), b.requires_grad_()
    side = torch.cuda.Stream()
    assert not on_default(w)
    held = ops.group_norm_act(x, 4, w, b)
    assert on_default(w) and on_default(b) and not on_default(x) and not on_default(held)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph, stream=side):
            torch.autograd.grad(ops.group_norm_act(x, 4, w, b), (w, b), dy)
    del held, graph
    assert not on_default(w) and not on_default(b)
    with torch.cuda.stream(side):
        y = ops.group_norm_act(x, 4, w, b)
        assert not on_default(w)
        torch.autograd.grad(y, (w, b), dy)
        del y
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(ops.group_norm_act(x, 4, w, b), (w, b), dy)
    for _ in range(2):
        graph.replay()
        want = torch.autograd.grad(ops.group_norm_act(x, 4, w, b), (w, b), dy)
        assert all(torch.equal(a, c) for a, c in zip(want, got))


WORKGROUPS = [((1, 24, 40, 40), 1), ((2, 12, 30, 30), 1), ((2, 180, 9, 9), 1), ((2, 360, 9, 9), 1), ((2, 2056, 3), 1), ((1, 4096, 2), 1),
              ((1, 4092, 2), 1), ((3, 20, 53, 50), 2), ((1, 20, 53, 50), 2), ((2, 64, 50, 52), 16), ((2, 64, 52, 51), 16), ((65, 6, 30), 2),
              ((1, 64, 40, 40), 1), ((2, 32, 28, 28), 1), ((10, 64, 52, 52), 32), ((1, 1 << 20, 5), 1024), ((1, (1 << 20) + 1, 3), 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,groups", WORKGROUPS, ids=[f"{'x'.join(map(str, s))}g{g}" for s, g in WORKGROUPS])
def test_columns_and_rows_of_a_workgroup(dev, shape, groups, dtype):
    """Columns that a wave does not hold whole rows of, few and many rows of them, more than half of the threads as columns, and
    numbers of rows on both sides of the backward pass's choice of form; gamma negative and zero in places."""
    x, dy, w, b = make(dev, shape, dtype, seed=5)
    w[::3] *= -1
    w[1::7] = 0
    for act in ACTS:
        want = reference(x, groups, w, b, 1e-5, act, dy)
        got = run_both(x, groups, w, b, act, dy)
        for k in want:
            check(got[k], want[k], (act, k))


def test_gradient_sums_do_not_lose_what_is_small(dev):
    """Many samples, so that a workgroup has all rows of one: 1 and then 999 times half a unit of its last place.  Added one after the other
    in fp32 they vanish (3e-5 of the sum); at most 300 additions in a row lose 300 h."""
    n, rows, c = 1024, 1000, 131
    x = torch.randn(n, rows, c, device=dev).movedim(-1, 1)
    dy = torch.full((n, rows, c), 2.0 ** -25, device=dev)
    dy[:, 0] = 1.0
    w, b = torch.ones(c, device=dev), torch.zeros(c, device=dev)
    got = run_both(x, 1, w, b, None, dy.movedim(-1, 1))
    want = n * (1 + 999 * 2.0 ** -25)
    assert float((got["dbias"].double() / want - 1).abs().max()) <= 300 * H


@pytest.mark.parametrize("shape", [(2, 16, 20, 20), (1, 16, 120, 120)], ids=["one launch", "three launches"])
@pytest.mark.parametrize("mean", [2.0 ** 14, 2.0 ** 17, 2.0 ** 20])
def test_a_mean_far_from_the_spread(dev, shape, mean):
    """fp32 holds a spread of 1 beside 2^20 to four bits behind the point; the variance is that of what it holds, to the bounds of any other
    input.  Also with the far element in the first place, which the sums are taken against, and in the last."""
    x, dy, w, b = make(dev, shape, torch.float32)
    far = channels_last(x + mean)
    first, last = x.clone(memory_format=torch.preserve_format), x.clone(memory_format=torch.preserve_format)
    first[:, ::4, 0, 0] = mean
    last[:, 3::4, -1, -1] = -mean
    for t in (far, first, last):
        for act in (None, "relu"):
            want, got = reference(t, 4, w, b, 1e-5, act, dy), run_both(t, 4, w, b, act, dy)
            for k in want:
                check(got[k], want[k], (act, k))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_keep_fp32s_digits(dev, act):
    """fp32 over |z| up to 11, at the rounding of each operation and not of the activation's largest value.  The bound is the slope's share of
    z's own 7 h |z| and the activation's operations (ulp = 2 h):
      silu: z log2(e) rounds twice, of which the power makes 2 |z| h; exponential 2 h, sum h, reciprocal 2 h, product h: (6 + 2 |z|) h |y|
      gelu: |z| density R: the exponent z^2 / 2 rounds three times: 1.5 z^2 h; exponential 2 h, two products 2 h; R = 1/2 - u Q, fit 1.1 h,
            u and Q 6 h of up to 1/2, h / 2 of its own, and R (1 + |z|) is never below 0.4: 9 (1 + |z|) h; the last sum h |y|
    In the 2-norm over z < -1, where the slope is small: no worse than the same in elementary fp32 operations and 2 h of z."""
    rows, c = 64, 1024
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(rows, c, generator=gen, device=dev)
    for scale in (1.0, 3.0):
        w, b = torch.full((c,), scale, device=dev), torch.zeros(c, device=dev)
        z = reference(x, 1, w, b, 1e-5, None)["y"][0].reshape(rows, c)
        dy = torch.zeros(rows, c, device=dev)
        dy[:, ::37] = 1.0                                                   # (dx of these is their slope's, less two small means)
        got = run_both(x, 1, w, b, act, dy)
        y, slope = act64(z, act)
        err_z = H * (6 * z.abs() + z.abs())
        a = z.abs()
        if act == "gelu":
            tail = 0.5 * torch.erfc(a / math.sqrt(2))
            own = H * (y.abs() + a * tail * (6 + 1.5 * z * z + 9 * (1 + a)))
        else:
            own = H * y.abs() * (6 + 2 * a)
        err = (got["y"].double() - y).abs()
        assert float((err / (slope.abs() * err_z + err_z ** 2 + own)).max()) <= 1.0, (scale, act)
        zf = z.float()
        if act == "gelu":
            plain = zf * (0.5 * (1 + torch.erf(zf * math.sqrt(0.5))))
        else:
            plain = zf / (1 + torch.exp(-zf))
        low = z < -1
        own_norm, plain_norm = (float((e[low] ** 2).sum().sqrt()) for e in (got["y"].double() - y, plain.double() - act64(zf.double(), act)[0]))
        assert own_norm <= plain_norm + 2 * H * float((z * slope)[low].norm()), (scale, act, own_norm, plain_norm)
        check(got["dx"], reference(x, 1, w, b, 1e-5, act, dy)["dx"])


def test_entry_point_without_rows_zeroes_the_weights_gradients(dev):
    from geomae_amd import _lib
    lib, stream = _lib.load(), torch.cuda.current_stream(dev).cuda_stream
    for n, rows in ((0, 10), (3, 0)):
        for k, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16)):
            for which in ((1, 1), (1, 0), (0, 1)):
                grads = [torch.full((600,), 5.0, device=dev, dtype=dtype) for _ in range(2)]
                ptrs = [t.data_ptr() if w else None for t, w in zip(grads, which)]
                assert lib.geomae_group_norm_backward(None, None, 0, n, rows, 600, 2, None, None, k, 0, None, None, *ptrs, None, 0, stream) == 0
                torch.cuda.synchronize()
                assert all(not t.any() if w else (t == 5.0).all() for t, w in zip(grads, which))


def test_one_and_two_channels_a_thread_past_the_caches(dev):
    """Over 64 MB in groups whose channels divide by 2 or not at all: accesses of one and two elements that leave the caches."""
    for dtype, c, groups in ((torch.float32, 33, 3), (torch.float32, 42, 7), (torch.bfloat16, 70, 7), (torch.float16, 66, 6)):
        x, dy, w, b = make(dev, (1, c, 701, 701), dtype)
        assert x.numel() * x.element_size() > 64e6 and (c // groups) % 4
        want, got = reference(x, groups, w, b, 1e-5, "silu", dy), run_both(x, groups, w, b, "silu", dy)
        for k in want:
            check(got[k], want[k], (dtype, k))


def test_definition_is_torchs():
    """The 64-bit definition above against torch's group norm and activations, gradients included, on the CPU."""
    import torch.nn.functional as F
    gen = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(3, 24, 5, 7, generator=gen, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(24, generator=gen, dtype=torch.float64) for _ in range(2))
    for act, f in ((None, lambda z: z), ("relu", F.relu), ("silu", F.silu), ("gelu", F.gelu)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = f(F.group_norm(leaves[0], 6, leaves[1], leaves[2], 1e-3))
        theirs = dict(zip(("y", "dx", "dweight", "dbias"), (y, *torch.autograd.grad(y, leaves, dy))))
        mine = reference(x, 6, w, b, 1e-3, act, dy)
        for k, t in theirs.items():
            assert torch.allclose(mine[k][0].reshape(t.shape), t.detach(), rtol=1e-11, atol=1e-12), (act, k)
