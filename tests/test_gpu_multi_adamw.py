"""MultiTensorAdamW on the GPU against the definition in 64 bits (adamw_definition.py).

Bounds, with h = 2^-24 (half a step of fp32), counted operation by operation:
  m' = m + w (x - m), x = g coef:        h (|m'| + 5 w (|g| + |m|))       [x, w, the difference, the product; the sum]
  v' = v b2 + (1 - b2) x x:              7 h v'                           [all terms positive; b2, 1 - b2, 3 products, x twice; the sum]
  update u = lr/bc1 m' / (r/bc + eps):   12 h |u| + |u| err(m')/|m'|      [r: 4, two divisions, bc, eps, the step size, the product]
  p' = p (1 - lr wd) - u:                3 h |p| + h |p'| + err(u)        and half a step of the parameter's own type if that is 16 bits
An 8-bit moment is the definition's code unless the position is nearer to the draw's border than the moment's own fp32 error
(in steps); then its neighbour will do."""
import gc

import adamw_definition as D
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
LR, BETAS, EPS, WD = 1e-3, (0.9, 0.999), 1e-8, 0.05


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def new(params, **kw):
    from geomae_amd.optim import MultiTensorAdamW
    return MultiTensorAdamW(params, **{**dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD), **kw})


def f64(t):
    return t.detach().double().cpu().numpy()


def in_memory_order(t):
    """The elements of a dense tensor as they lie in memory."""
    return t.detach().as_strided((t.numel(),), (1,)) if t.numel() else t.detach().reshape(-1)


def snapshot(opt, p):
    """(p or its master, m, v, step) in 64 bits, in memory order."""
    st = opt.state[p]
    m, v = in_memory_order(st["exp_avg"]), in_memory_order(st["exp_avg_sq"])
    if opt.state_bits == 8:
        e = [st[k].cpu().numpy() for k in ("exp_avg_exponent", "exp_avg_sq_exponent")]
        m, v = D.decode(m.cpu().numpy(), e[0], D.SIGNED), D.decode(v.cpu().numpy(), e[1], D.ROOT) ** 2
    else:
        m, v = f64(m), f64(v)
    return f64(in_memory_order(st.get("master", p))), m, v, int(st["step"])


def check(opt, p, before, g, index, coef=1.0, lr=LR, wd=WD, coef_err=H):
    """p and its state after a step from `before` with gradient g (memory order, 64 bits)."""
    p0, m0, v0, s0 = before
    assert int(opt.state[p]["step"]) == s0 + 1
    want_p, want_m, want_v = D.step(p0, g, m0, v0, s0 + 1, lr, BETAS, EPS, wd, coef)
    got_p, got_m, got_v, _ = snapshot(opt, p)
    w = 1 - BETAS[0]
    err_m = H * (np.abs(want_m) + 5 * w * (np.abs(g * coef) + np.abs(m0))) + w * coef_err * np.abs(g * coef) + 2.0 ** -149
    # squares below the smallest normal number round to multiples of 2^-149
    err_v = 7 * H * want_v + 2 * coef_err * want_v + 3 * 2.0 ** -149
    bc1, bc2 = 1 - BETAS[0] ** (s0 + 1), 1 - BETAS[1] ** (s0 + 1)
    den = np.sqrt(want_v) / np.sqrt(bc2) + EPS
    err_r = np.minimum(err_v / np.maximum(2 * np.sqrt(want_v), 1e-300), np.sqrt(err_v))
    u = lr / bc1 * want_m / den
    err_u = 12 * H * np.abs(u) + lr / bc1 * err_m / den + np.abs(u) * err_r / np.sqrt(bc2) / den * 1.01
    err_p = 3 * H * np.abs(p0) + H * np.abs(want_p) + err_u
    if opt.state[p].get("master") is None and p.dtype != torch.float32:
        err_p = err_p + (torch.finfo(p.dtype).eps / 2) * (np.abs(want_p) + err_p) + (2.0 ** -25 if p.dtype == torch.float16 else 0)
    assert (np.abs(got_p - want_p) <= err_p).all(), float(np.max(np.abs(got_p - want_p) / err_p))
    if opt.state[p].get("master") is not None:
        assert torch.equal(opt.state[p]["master"].to(p.dtype), p.detach())
    if opt.state_bits == 32:
        assert (np.abs(got_m - want_m) <= err_m).all() and (np.abs(got_v - want_v) <= err_v).all()
        return
    um, ur = D.draws(opt.seed, index, s0 + 1, p.numel())
    want_r, got_r = np.sqrt(want_v), np.sqrt(got_v)
    for got, x, u16, table, err, digits in ((got_m, want_m, um, D.SIGNED, err_m, 3), (got_r, want_r, ur, D.ROOT, err_r + H * want_r, 4)):
        val, _, margin = D.encode(x, u16, table)
        width = 2.0 ** (digits + 1)                                    # a position is below 16 resp. 32 steps
        border = width * (err / np.maximum(np.abs(x), 1e-300) + 2 * H)
        off = got != val
        assert not (off & (margin > border)).any(), (table is D.ROOT, int(off.sum()))
        assert (np.abs(got - val)[off] <= 2.0 ** -digits * np.maximum(np.abs(got), np.abs(val))[off] * 1.0001 + 2.0 ** -120).all()
        # the border is met by chance only: its width times a draw's density, and five standard errors
        assert off.sum() <= 5 + 2 * np.minimum(border, 1).sum() + 5 * np.sqrt(2 * np.minimum(border, 1).sum())


SIZES = [1, 2, 3, 31, 32, 33, 63, 64, 255, 1023, 4095, 4096, 4097, 10_007]


def make(dev, dtype, sizes=SIZES, seed=0, gap=1):
    """Parameters as views into one buffer with gaps, so that most are not aligned to 4 elements; gradients likewise."""
    gen = torch.Generator().manual_seed(seed)
    total = sum(s + gap for s in sizes) + 1
    buf = torch.randn(total, generator=gen).mul_(0.1).to(dtype).to(dev)
    gbuf = (torch.randn(total, generator=gen) * torch.exp(2 * torch.randn(total, generator=gen)) * 1e-3).to(dtype).to(dev)
    params, at = [], 1
    for s in sizes:
        p = torch.nn.Parameter(buf[at:at + s])
        p.grad = gbuf[at:at + s]
        params.append(p)
        at += s + gap
    return params, buf


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True),
                                          (torch.float16, False), (torch.float16, True)])
def test_steps_match_the_definition(dev, bits, dtype, master):
    params, buf = make(dev, dtype)
    opt = new(params, state_bits=bits, master_weights=master, seed=5)
    outside = torch.ones(buf.numel(), dtype=torch.bool)
    for p in params:
        o = (p.data_ptr() - buf.data_ptr()) // buf.element_size()
        outside[o:o + p.numel()] = False
    kept = buf.cpu()[outside]
    for _ in range(3):
        before = [snapshot(opt, p) for p in params]
        opt.step()
        for i, p in enumerate(params):
            check(opt, p, before[i], f64(p.grad), i)
    assert torch.equal(buf.cpu()[outside], kept)                       # what lies between the parameters is not touched


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("scale", [1.0, 0.125])
@pytest.mark.parametrize("max_norm", [0.05, 1e6])
def test_clipping_and_scaling(dev, bits, scale, max_norm):
    params, _ = make(dev, torch.float32)
    opt = new(params, state_bits=bits)
    as_tensor = torch.tensor(scale, device=dev)
    norm = scale * np.sqrt(sum((f64(p.grad) ** 2).sum() for p in params))
    for s in (scale, as_tensor):
        before = [snapshot(opt, p) for p in params]
        opt.step(max_norm=max_norm, grad_scale=s)
        assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm + 1e-12
        coef = scale * min(1.0, max_norm / (norm + 1e-6))
        for i, p in enumerate(params):
            check(opt, p, before[i], f64(p.grad), i, coef=coef, coef_err=6 * H)


def test_many_tensors_groups_and_missing_gradients(dev):
    """More tensors than a launch takes, more hyper-parameter sets than a launch takes, gradients missing in between; the mix of
    types in one optimizer."""
    sizes = [(7 * i) % 131 + 1 for i in range(600)]
    f32, _ = make(dev, torch.float32, sizes[:400])
    b16, _ = make(dev, torch.bfloat16, sizes[400:], seed=1)
    params = f32 + b16
    groups = [{"params": params[i::23], "lr": LR * (1 + i), "weight_decay": 0.01 * i} for i in range(23)]
    opt = new(groups, state_bits=8, master_weights=True)
    order = [p for g in groups for p in g["params"]]
    for i, p in enumerate(order):
        if i % 5 == 0:
            p.grad = None
    before = [snapshot(opt, p) for p in order]
    opt.step(max_norm=1e6)
    norm = np.sqrt(sum((f64(p.grad) ** 2).sum() for p in order if p.grad is not None))
    assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm
    i = 0
    for g in groups:
        for p in g["params"]:
            if p.grad is None:
                assert int(opt.state[p]["step"]) == 0
                assert all(np.array_equal(a, b) for a, b in zip(snapshot(opt, p)[:3], before[i][:3]))
            else:
                check(opt, p, before[i], f64(in_memory_order(p.grad)), i, lr=g["lr"], wd=g["weight_decay"])
            i += 1


def test_layouts(dev):
    """Channels-last and transposed parameters; gradients in another layout than their parameter's; a 0-d and an empty one."""
    torch.manual_seed(0)
    conv = torch.nn.Parameter(torch.randn(8, 5, 3, 3, device=dev).to(memory_format=torch.channels_last))
    conv.grad = torch.randn(8, 5, 3, 3, device=dev)
    lin = torch.nn.Parameter(torch.randn(7, 9, device=dev).t())
    lin.grad = torch.randn(9, 7, device=dev)
    scalar = torch.nn.Parameter(torch.randn((), device=dev))
    scalar.grad = torch.randn((), device=dev)
    empty = torch.nn.Parameter(torch.zeros(0, 4, device=dev))
    empty.grad = torch.zeros(0, 4, device=dev)
    strided = torch.nn.Parameter(torch.randn(6, 4, device=dev))
    strided.grad = torch.randn(6, 8, device=dev)[:, ::2]
    params = [conv, lin, scalar, empty, strided]
    for bits in (32, 8):
        opt = new(params, state_bits=bits)
        before = [snapshot(opt, p) for p in params]
        opt.step()
        for i, p in enumerate(params):
            if p.numel():
                g = torch.empty_strided(p.shape, p.stride(), device=dev).copy_(p.grad)
                check(opt, p, before[i], f64(in_memory_order(g)), i)
        assert opt.state[conv]["exp_avg"].stride() == conv.stride()


def test_matches_torch_adamw_and_takes_its_state(dev):
    """Ten steps beside torch.optim.AdamW on the same gradients, then a resumed run from ITS state_dict.  Per step the two
    differ by the two sides' own bounds; ten steps of at most lr each."""
    params, _ = make(dev, torch.float32)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = new(params), torch.optim.AdamW(twins, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, foreach=False)
    gen = torch.Generator(device=dev).manual_seed(3)
    for _ in range(10):
        for p, q in zip(params, twins):
            q.grad = torch.randn(p.shape, generator=gen, device=dev)
            p.grad = q.grad.clone()
        a.step()
        b.step()
    bound = lambda p: 10 * (2 * 4 * H * p.detach().abs().max() + 2 * 40 * H * LR * 4)
    for p, q in zip(params, twins):
        assert float((p - q).abs().max()) <= float(bound(p))
    c = new([torch.nn.Parameter(q.detach().clone()) for q in twins])
    c.load_state_dict(b.state_dict())
    again = c.param_groups[0]["params"]
    for q, r in zip(twins, again):
        r.grad = q.grad
    b.step()
    c.step()
    for q, r in zip(twins, again):
        assert float((r - q).abs().max()) <= float(bound(q)) / 10
        assert int(c.state[r]["step"]) == 11


@pytest.mark.parametrize("bits,master", [(32, False), (8, False), (8, True)])
def test_checkpoint_resumes_bit_for_bit(dev, bits, master, tmp_path):
    def run(opt, params, steps, seed):
        gen = torch.Generator(device=dev).manual_seed(seed)
        for _ in range(steps):
            for p in params:
                p.grad = torch.randn(p.shape, generator=gen, device=dev).to(p.dtype)
            opt.step(max_norm=1.0)
    dtype = torch.bfloat16 if master else torch.float32
    params, _ = make(dev, dtype)
    opt = new(params, state_bits=bits, master_weights=master, seed=9)
    run(opt, params, 3, 1)
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    run(opt, params, 3, 2)
    back = new(copies, state_bits=bits, master_weights=master, seed=0)
    back.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    run(back, copies, 3, 2)
    assert all(torch.equal(a, b) for a, b in zip(params, copies))
    with pytest.raises(ValueError, match="bits"):
        new(copies, state_bits=40 - bits).load_state_dict(opt.state_dict())
    flat = dict(zip(("exp_avg", "exp_avg_sq"), opt.moments())) if bits == 32 else {k: v for k, v in opt._arena.items() if k != "step"}
    third = new([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=bits, master_weights=master, seed=9)
    third.load_flat_state(flat, step=6)
    run(opt, params, 1, 4)
    run(third, third.param_groups[0]["params"], 1, 4)
    assert all(torch.equal(a, b) for a, b in zip(params, third.param_groups[0]["params"]))
    with pytest.raises(ValueError, match="flat state"):
        third.load_flat_state({}, step=0)


def test_moments_are_what_the_codes_stand_for(dev):
    """Every code under every exponent byte, to bf16 and back."""
    from geomae_amd.optim import MultiTensorAdamW
    p = torch.nn.Parameter(torch.zeros(256 * 239, device=dev))
    opt = MultiTensorAdamW([p], state_bits=8)
    codes = torch.arange(256, dtype=torch.uint8).repeat(239).to(dev)
    exps = torch.arange(16, 255, dtype=torch.uint8).repeat_interleave(8).to(dev)
    opt.load_flat_state({"exp_avg": codes, "exp_avg_exponent": exps, "exp_avg_sq": codes, "exp_avg_sq_exponent": exps}, step=1)
    m, r = opt.moments()
    for got, table in ((m, D.SIGNED), (r, D.ROOT)):
        want = D.decode(codes.cpu().numpy(), exps.cpu().numpy(), table)
        got = f64(got)
        fine = np.abs(want) >= 2.0 ** -126                               # (bf16's subnormal numbers have fewer digits)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[fine], want[fine])
        small = ~fine & ~np.isnan(want)
        assert (np.abs(got - want)[small] <= 2.0 ** -134).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_gradients(dev, bits):
    """skip_nonfinite leaves everything as it was; without it NaN and infinity stay in the elements that had them."""
    for bad in (float("nan"), float("inf"), -float("inf")):
        params, _ = make(dev, torch.float32, [100, 33])
        opt = new(params, state_bits=bits)
        opt.step()
        kept = [p.detach().clone() for p in params], [t.clone() for t in opt._arena.values()]
        g0 = params[0].grad.clone()
        params[0].grad = g0.clone()
        params[0].grad[17] = bad
        opt.step(skip_nonfinite=True)
        assert not torch.isfinite(opt.grad_norm)
        assert all(torch.equal(a, b) for a, b in zip(kept[0], params)) and all(torch.equal(a, b) for a, b in zip(kept[1], opt._arena.values()))
        before = [snapshot(opt, p) for p in params]
        opt.step()
        assert not torch.isfinite(params[0][17]) and torch.isfinite(params[0].detach()).sum() == 99
        m, v = opt.moments()
        assert not torch.isfinite(m[17]) and not torch.isfinite(v[17])
        assert torch.isfinite(m).sum() == m.numel() - 1 and torch.isfinite(v).sum() == v.numel() - 1
        check(opt, params[1], before[1], f64(params[1].grad), 1)
        opt.step()                                                     # and the next step spreads nothing
        assert torch.isfinite(params[0].detach()).sum() == 99


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_and_draws_on(dev, bits):
    """A captured step, replayed with eager steps of the same and of another optimizer in between, is the eager run; its lr is
    read at every replay."""
    lr = torch.tensor(LR, device=dev)
    params, _ = make(dev, torch.float32)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    others, _ = make(dev, torch.float32, [50, 4097], seed=2)
    for p, q in zip(params, twins):
        q.grad = p.grad.clone()
    a, b, c = new(params, state_bits=bits, lr=lr), new(twins, state_bits=bits, lr=lr.clone()), new(others, state_bits=bits)
    other_grads = [p.grad.clone() for p in others]
    a.step(max_norm=0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.step(max_norm=0.5)
    with torch.cuda.graph(second, stream=side):
        c.step(max_norm=0.5)
    b.step(max_norm=0.5)
    for r in range(4):
        lr.fill_(LR / (1 + r))
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        b.param_groups[0]["lr"].fill_(LR / (1 + r))
        b.step(max_norm=0.5)
        assert all(torch.equal(p, q) for p, q in zip(params, twins)), r
        assert float(a.grad_norm) == float(b.grad_norm)
        for p, g in zip(others, other_grads):                          # eager, other gradients' addresses
            p.grad = g * (r + 1)
        c.step()
    a.step(max_norm=0.5)
    b.step(max_norm=0.5)
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    # one eager step, four replays (capturing takes none), one eager step
    assert int(a.state[params[0]]["step"]) == 6 == int(a.state[params[-1]]["step"]) and torch.isfinite(others[1]).all()


def test_streams_and_moved_storage(dev):
    """Two optimizers on two streams at once; a parameter whose storage moved is found again."""
    sets = [make(dev, torch.float32, [200_000, 77, 4096], seed=s)[0] for s in (0, 1)]
    opts = [new(s, state_bits=8, seed=1) for s in sets]
    twins = [[torch.nn.Parameter(p.detach().clone()) for p in s] for s in sets]
    for s, t in zip(sets, twins):
        for p, q in zip(s, t):
            q.grad = p.grad
    plain = [new(t, state_bits=8, seed=1) for t in twins]
    streams = [torch.cuda.Stream() for _ in opts]
    torch.cuda.synchronize()
    for _ in range(5):
        for o, st in zip(opts, streams):
            with torch.cuda.stream(st):
                o.step(max_norm=1.0)
    torch.cuda.synchronize()
    for o in plain:
        for _ in range(5):
            o.step(max_norm=1.0)
    assert all(torch.equal(p, q) for s, t in zip(sets, twins) for p, q in zip(s, t))
    sets[0][1].data = sets[0][1].data.clone()
    opts[0].step(max_norm=1.0)
    plain[0].step(max_norm=1.0)
    assert all(torch.equal(p, q) for p, q in zip(sets[0], twins[0]))
    sets[0][1].data = torch.zeros(78, device=dev)
    sets[0][1].grad = None
    with pytest.raises(RuntimeError, match="changed its shape"):
        opts[0].step()


def test_add_param_group_keeps_the_old_state(dev):
    params, _ = make(dev, torch.float32)
    opt = new(params[:-2], state_bits=8)
    opt.step()
    held = [[t.clone() for t in opt.state[p].values()] for p in params[:-2]]
    opt.add_param_group({"params": params[-2:], "lr": 1e-2})
    assert all(torch.equal(a, b) for p, h in zip(params[:-2], held) for a, b in zip(opt.state[p].values(), h))
    before = [snapshot(opt, p) for p in params]
    opt.step()
    for i, p in enumerate(params):
        check(opt, p, before[i], f64(p.grad), i, lr=LR if i < len(params) - 2 else 1e-2)


def test_nothing_to_update(dev):
    """Only empty tensors, or no gradient anywhere: nothing moves, and the norm is 0."""
    empty = torch.nn.Parameter(torch.zeros(0, 3, device=dev))
    empty.grad = torch.zeros(0, 3, device=dev)
    full = torch.nn.Parameter(torch.ones(50, device=dev))
    for params in ([empty], [full], [empty, full]):
        opt = new(params, state_bits=8)
        opt.step()
        opt._norm_word.fill_(7.0)
        opt.step(max_norm=1.0)
        assert float(opt.grad_norm) == 0.0 and (full == 1.0).all() and not opt._arena["step"].any()


def test_state_that_is_partly_there_and_masters(dev):
    """A state_dict without some parameters' state: those begin anew.  A tensor lr stays the tensor it was.  Masters follow a
    parameter that somebody else wrote once they are told."""
    params, _ = make(dev, torch.bfloat16, [40, 33])
    lr = torch.tensor(1e-2, device=dev)
    opt = new(params, state_bits=8, master_weights=True, lr=lr)
    for _ in range(2):
        opt.step()
    sd = opt.state_dict()
    sd = {**sd, "state": {0: {k: v.clone() for k, v in sd["state"][0].items()}},
          "param_groups": [{**sd["param_groups"][0], "lr": torch.tensor(5e-3)}]}
    opt.step()
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] is lr and abs(float(lr) - 5e-3) < 1e-9
    a, b = (opt.state[p] for p in params)
    assert int(a["step"]) == 2 and int(b["step"]) == 0 and not b["exp_avg"].any() and not b["exp_avg_sq"].any()
    assert all(torch.equal(a[k], v) for k, v in sd["state"][0].items())
    with torch.no_grad():
        params[1].fill_(0.5)
    opt.sync_masters()
    assert (b["master"] == 0.5).all()
    before = [snapshot(opt, p) for p in params]
    opt.step()
    for i, p in enumerate(params):
        check(opt, p, before[i], f64(p.grad), i, lr=float(lr))


def test_a_refused_group_leaves_the_optimizer_as_it_was(dev):
    base = torch.zeros(96, device=dev)
    p, q = torch.nn.Parameter(base[:40]), torch.nn.Parameter(base[32:])
    opt = new([p])
    with pytest.raises(ValueError, match="share memory"):
        opt.add_param_group({"params": [q]})
    p.grad = torch.ones(40, device=dev)
    before = snapshot(opt, p)
    opt.step()
    check(opt, p, before, f64(p.grad), 0)


def test_offsets_past_32_bits(dev):
    """2^31 + 4133 elements (bf16, 8-bit moments): the last ones, which a 32-bit offset would miss, are updated."""
    n = 2 ** 31 + 4133
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    p.grad[-5000:] = 0.5
    opt = new([p], state_bits=8, lr=0.25, weight_decay=0.0)
    opt.step(max_norm=0.0, skip_nonfinite=True)
    # from zero moments u = lr * sign(g) to within the sum of eps and the roundings, and -0.25 is a bf16 number
    assert (p.detach()[-5000:] == -0.25).all() and not p.detach()[:-5000].any()
    assert abs(float(opt.grad_norm) - np.sqrt(5000) * 0.5) <= 1e-5


def test_refusals(dev):
    from geomae_amd.optim import MultiTensorAdamW
    base = torch.zeros(64, device=dev)
    P = torch.nn.Parameter
    with pytest.raises(RuntimeError, match="dense"):
        MultiTensorAdamW([P(torch.zeros(4, 6, device=dev)[:, :3])])
    with pytest.raises(RuntimeError, match="float32"):
        MultiTensorAdamW([P(torch.zeros(4, device=dev, dtype=torch.float64))])
    with pytest.raises(ValueError, match="share memory"):
        MultiTensorAdamW([P(base[:40]), P(base[32:])])
    p = P(base)
    with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning):
        MultiTensorAdamW([p, p])
    with pytest.raises(ValueError, match="lr must be one float32"):
        MultiTensorAdamW([p], lr=torch.tensor(0.1))
    opt = MultiTensorAdamW([p], state_bits=8)
    p.grad = torch.ones(64, device=dev)
    with pytest.raises(RuntimeError, match="grad_scale"):
        opt.step(grad_scale=torch.tensor(1.0))
    opt.param_groups[0]["betas"] = (0.9, 1.0)
    with pytest.raises(ValueError, match="betas"):
        opt.step()
    opt.param_groups[0]["betas"] = (0.9, 0.99)
    with pytest.raises(RuntimeError, match="master_weights"):
        opt.masters()
    assert not base.any()


def test_is_not_copied_and_steps_after_hooks(dev):
    import copy
    import pickle
    p = torch.nn.Parameter(torch.ones(40, device=dev))
    opt = new([p])
    for f in (copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            f(opt)
    seen = []
    opt.register_step_post_hook(lambda *a: seen.append(1))
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)

    def closure():
        opt.zero_grad()
        loss = (p ** 2).sum()
        loss.backward()
        return loss
    version = p._version
    assert float(opt.step(closure)) == 40.0 and seen == [1] and p._version > version
    sched.step()
    assert opt.param_groups[0]["lr"] == LR / 2
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):   # a step between forward and backward is noticed
        loss = (p ** 2).sum()
        opt.step()
        loss.backward()


def test_beta_zero_and_eps_zero(dev):
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 70, device=dev))
        p.grad = torch.linspace(1, 2, 70, device=dev)
        opt = new([p], betas=(0.0, 0.0), eps=0.0, weight_decay=0.0, state_bits=bits)
        start = f64(p)
        opt.step()
        # m = g, v = g g: the update is lr, within the 12 h of its operations, and p rounds once
        assert np.abs(f64(p) - (start - LR)).max() <= 12 * H * LR + H


def test_a_parameter_changed_where_it_lies_is_refused(dev):
    """The same address with another length, order or type: no step, nothing changed."""
    for change in (lambda t: t[:2], lambda t: t.t(), lambda t: t.reshape(-1)):
        p = torch.nn.Parameter(torch.randn(4, 6, device=dev))
        other = torch.nn.Parameter(torch.randn(5, device=dev))
        opt = new([other, p])
        before = other.detach().clone()
        p.data = change(p.data)
        p.grad, other.grad = torch.ones_like(p), torch.ones_like(other)
        with pytest.raises(RuntimeError, match="shape, layout"):
            opt.step()
        assert torch.equal(other, before) and int(opt.state[other]["step"]) == 0
    opt = new([other])
    other.grad = torch.ones_like(other)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            opt.step(max_norm=bad)
    opt.step(max_norm=None)
    assert int(opt.state[other]["step"]) == 1


def test_hooks_profiler_and_subclasses(dev):
    """Step hooks of the optimizer and of all optimizers run once a step, with the step's arguments, also where a subclass
    overrides step(); the profiler sees the step."""
    from geomae_amd.optim import MultiTensorAdamW
    from torch.optim.optimizer import register_optimizer_step_post_hook, register_optimizer_step_pre_hook

    class Counting(MultiTensorAdamW):
        def step(self, *args, **kw):
            self.count = getattr(self, "count", 0) + 1
            return super().step(*args, **kw)
    for cls in (MultiTensorAdamW, Counting):
        p = torch.nn.Parameter(torch.ones(40, device=dev))
        p.grad = torch.full_like(p, 2.0)
        opt, seen = cls([p], lr=LR), []
        handles = [register_optimizer_step_pre_hook(lambda o, a, k: seen.append("all before")),
                   register_optimizer_step_post_hook(lambda o, a, k: seen.append("all after"))]
        opt.step()
        assert seen == ["all before", "all after"]
        for h in handles:
            h.remove()
        opt.step()
        assert len(seen) == 2 and int(opt.state[p]["step"]) == 2
        seen.clear()
        handle = opt.register_step_pre_hook(lambda o, a, k: seen.append(p.grad.mul_(0.5)))
        opt.step(max_norm=float("inf"))
        assert len(seen) == 1 and abs(float(opt.grad_norm) - 40 ** 0.5) < 1e-5
        handle.remove()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
            opt.step()
        assert sum(f"Optimizer.step#{cls.__name__}.step" in e.name for e in prof.events()) == 1
        assert int(opt.state[p]["step"]) == 4 and getattr(opt, "count", 4) == 4


def test_codes_stay_with_their_exponents_in_another_memory_order(dev):
    """An 8-bit state is refused by a parameter of the same shape in another memory order (32 elements that share an exponent are
    others there) and leaves the optimizer as it was; in its own order it is the same whatever the saved tensors' strides are;
    32 bits go across."""
    gen = torch.Generator().manual_seed(1)
    base = torch.randn(64, 16, 3, 3, generator=gen) * torch.exp(2 * torch.randn(64, 16, 3, 3, generator=gen))
    lin = torch.randn(24, 40, generator=gen)
    kinds = {"rows": (base, lin), "columns": (base.to(memory_format=torch.channels_last), lin.t().contiguous().t())}

    def stepped(kind, bits):
        params = [torch.nn.Parameter(t.to(dev, copy=True)) for t in kinds[kind]]
        for p in params:
            p.grad = torch.sin(1e3 * p.detach()) * p.detach().abs()
        opt = new(params, state_bits=bits, seed=4)
        opt.step()
        return opt, params
    for src, dst in (("rows", "columns"), ("columns", "rows"), ("rows", "rows"), ("columns", "columns")):
        for bits in (8, 32):
            a, ps = stepped(src, bits)
            sd = a.state_dict()
            flat = {**sd, "state": {i: {k: v.contiguous() for k, v in st.items()} for i, st in sd["state"].items()}}
            old = {k: v for k, v in sd.items() if k != "memory_orders"}                    # (as it was written before)
            for state in (sd, flat, old):
                b, qs = stepped(dst, bits)
                held = [t.clone() for t in b._arena.values()]
                if bits == 8 and src != dst:
                    with pytest.raises(ValueError, match="memory order"):
                        b.load_state_dict(state)
                    assert all(torch.equal(x, y) for x, y in zip(held, b._arena.values()))
                    continue
                b.load_state_dict(state)
                for p, q in zip(ps, qs):
                    assert all(torch.equal(a.state[p][k], b.state[q][k]) for k in a.state[p])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_group_is_refused_beside_a_changed_parameter(dev, bits):
    """A parameter that was cut, cast or re-ordered in the meantime: the new group is refused, and with the parameter as it was the
    optimizer goes on as if nothing had been asked of it."""
    changes = (lambda t: t[:3], lambda t: t.half(), lambda t: t.contiguous(memory_format=torch.channels_last), lambda t: t.transpose(0, 1))
    for change in changes:
        params = [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(7)).bfloat16().to(dev)) for s in ((8, 6, 5, 3), (70,))]
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for p, q in zip(params, twins):
            p.grad = torch.randn_like(p)
            q.grad = p.grad
        a, b = (new(s, state_bits=bits, master_weights=True) for s in (params, twins))
        a.step()
        b.step()
        grad, kept = params[0].grad, params[0].data
        params[0].grad, params[0].data = None, change(kept)
        with pytest.raises(RuntimeError, match="shape, layout"):
            a.add_param_group({"params": [torch.nn.Parameter(torch.zeros(9, device=dev))]})
        assert len(a.param_groups) == 1 and len(a.state) == 2
        params[0].data, params[0].grad = kept, grad
        a.step(max_norm=1.0)
        b.step(max_norm=1.0)
        assert all(torch.equal(p, q) for p, q in zip(params, twins))
        assert all(torch.equal(a.state[p][k], v) for p, q in zip(params, twins) for k, v in b.state[q].items())


@pytest.mark.parametrize("eps", [1e-8, 0.0, 1e-39])
def test_the_first_step_is_the_same_in_8_bits(dev, eps):
    """From zero moments nothing has been rounded to codes yet: the same parameters as with 32-bit moments, operation by operation, also
    where squares underflow or overflow and eps is below fp32's normal numbers.  (In 8 bits the root and the quotients are within 0.5000003
    units of the last place: one element in 10^5 may differ by its last bit.)"""
    gen = torch.Generator(device=dev).manual_seed(0)
    n = 1 << 20
    grad = torch.randn(n, generator=gen, device=dev)
    grad[n // 2:] *= torch.exp(torch.empty(n - n // 2, device=dev).uniform_(-88.0, 48.0, generator=gen))
    grad[::5] = 0.0
    for base in (torch.zeros(n, device=dev), torch.randn(n, generator=gen, device=dev)):
        out = []
        for bits in (32, 8):
            p = torch.nn.Parameter(base.clone())
            p.grad = grad
            new([p], state_bits=bits, eps=eps).step()
            out.append(p.detach())
        a, b = out
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        differ = (a != b) & ~a.isnan()
        assert int(differ.sum()) <= 1e-5 * n
        assert not differ.any() or float(((a - b).abs() / a.abs())[differ].max()) <= 4 * H


def test_every_nan_is_held_as_one(dev):
    """A NaN of any sign and payload in a gradient makes both moments NaN, whatever the draw, and nothing else of its block."""
    for dtype, nans in ((torch.bfloat16, (0xffff, 0x7fff, 0xff81, 0x7f81)), (torch.float16, (0xffff, 0x7fff, 0xfc01, 0x7c01)),
                        (torch.float32, (0xffffffff, 0x7fffffff, 0xff800001, 0x7f800001))):
        n = 32 * 64 * len(nans)
        p = torch.nn.Parameter(torch.zeros(n, device=dev, dtype=dtype))
        grad = torch.ones(n, dtype=dtype)
        raw = grad.numpy().view("uint16" if grad.element_size() == 2 else "uint32") if dtype != torch.bfloat16 else grad.view(torch.int16).numpy().view("uint16")
        for k, bits in enumerate(nans):
            raw[32 * k::32 * len(nans)] = bits
        p.grad = grad.to(dev)
        assert int(p.grad.isnan().sum()) == n // 32
        opt = new([p], state_bits=8)
        for _ in range(3):
            opt.step()
            m, r = opt.moments()
            hit = p.grad.isnan()
            assert m[hit].isnan().all() and r[hit].isnan().all() and m[~hit].isfinite().all() and r[~hit].isfinite().all()


@pytest.mark.parametrize("max_norm", [1e-30, 1e-44, 1e-50])
def test_the_smallest_norms_clip(dev, max_norm):
    p = torch.nn.Parameter(torch.zeros(64, device=dev))
    p.grad = torch.ones(64, device=dev)
    opt = new([p])
    opt.step(max_norm=max_norm)
    assert float(opt.grad_norm) == 8.0 and float(opt.moments()[0].abs().max()) <= max_norm / 8 * 0.1 * 1.01 + 2.0 ** -149


def test_load_hooks_run(dev):
    """As torch's optimizers: pre-hooks get a shallow copy and may change or replace it, post-hooks come after the load."""
    params, _ = make(dev, torch.float32, [40])
    opt = new(params)
    opt.step()
    sd, seen = opt.state_dict(), []

    def replace(o, state):
        seen.append(("pre", int(opt.state[params[0]]["step"])))
        return {**state, "state": {0: {**state["state"][0], "step": torch.tensor(7)}}}
    handles = [opt.register_load_state_dict_pre_hook(lambda o, state: state.__setitem__("seed", 5)), opt.register_load_state_dict_pre_hook(replace),
               opt.register_load_state_dict_post_hook(lambda o: seen.append(("post", int(o.state[params[0]]["step"]))))]
    opt.load_state_dict(sd)
    assert seen == [("pre", 1), ("post", 7)] and opt.seed == 5 and sd["seed"] == 0
    for h in handles:
        h.remove()
    opt.load_state_dict(sd)
    assert len(seen) == 2 and int(opt.state[params[0]]["step"]) == 7 and opt.seed == 0


def test_buffers_outlive_steps_on_other_streams(dev):
    """The moments, the table and the workspace are the optimizer's own: made on one stream, stepped on a second at once, and dropped while
    that step is still to run, they are neither read before they are there nor given to somebody else."""
    side = torch.cuda.Stream()
    for drop in ("optimizer", "table", "group"):
        params, _ = make(dev, torch.float32, [40_000, 77])
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for p, q in zip(params, twins):
            q.grad = p.grad
        want = new(twins)
        want.step()
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)
        opt = new(params)
        sizes = [t.numel() for t in opt._arena.values()] + [opt._table.numel() // 4, opt._chunks.numel(), opt._workspace.numel() // 4]
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            opt.step()
        if drop == "optimizer":
            del opt
            gc.collect()
        elif drop == "table":
            kept = params[1].data                                          # (the parameter's memory is the caller's)
            params[1].data = kept.clone()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                opt.step()
            want.step()
        else:
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(9, device=dev))]})
            with torch.cuda.stream(side):
                opt.step()
            want.step()
        other = [torch.full((n,), float("nan"), device=dev) for n in sizes for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(params[0], twins[0]) and (drop == "table" or torch.equal(params[1], twins[1]))
        assert all(t.isnan().all() for t in other)


def test_groups_without_parameters(dev):
    """A group may be empty, the first one too, as with torch's optimizers (a model without biases, everything frozen in one of them)."""
    params, _ = make(dev, torch.float32, [40, 33])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, twins):
        q.grad = p.grad
    a = new([{"params": [], "weight_decay": 0.0}, {"params": params[:1]}, {"params": []}, {"params": params[1:], "lr": 1e-2}])
    b = new([{"params": twins[:1]}, {"params": twins[1:], "lr": 1e-2}])
    for o in (a, b):
        o.step(max_norm=0.1)
    a.add_param_group({"params": []})
    a.load_state_dict(a.state_dict())
    for o in (a, b):
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins)) and len(a.param_groups) == 5


def test_parameters_and_state_replaced_behind_the_optimizer(dev):
    """A parameter object replaced by another of its shape, two swapped, one removed, the state cleared: a step would use another's moments, or
    ones that the caller thinks are gone.  Each is refused and changes nothing; a state_dict with an empty state does begin anew."""
    import collections
    params = [torch.nn.Parameter(torch.randn(64, device=dev)) for _ in range(3)]
    for p in params:
        p.grad = torch.randn_like(p)
    opt = new(params)
    opt.step()
    held, before = list(params), [p.detach().clone() for p in params]
    other = torch.nn.Parameter(params[1].detach().clone())
    other.grad = params[1].grad
    group = opt.param_groups[0]
    for wrong in ([held[0], other, held[2]], [held[1], held[0], held[2]], held[:2], held + [other]):
        group["params"] = wrong
        with pytest.raises(RuntimeError, match="make a new optimizer"):
            opt.step()
        with pytest.raises(RuntimeError, match="make a new optimizer"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, device=dev))]})
    group["params"] = held
    state = opt.state
    opt.state = collections.defaultdict(dict)
    with pytest.raises(RuntimeError, match="state was cleared"):
        opt.step()
    opt.state = state
    assert all(torch.equal(p, q) for p, q in zip(held, before)) and (opt._arena["step"] == 1).all()
    opt.load_state_dict({**opt.state_dict(), "state": {}})
    assert not opt.moments()[0].any() and not opt._arena["step"].any()
    opt.step()
    assert (opt._arena["step"] == 1).all()


def test_state_may_hold_other_entries(dev):
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    p.grad = torch.ones(8, device=dev)
    opt = new([p])
    opt.state["count"] = 3                                                 # (torch's optimizers take it too)
    opt.step()
    assert int(opt.state[p]["step"]) == 1
