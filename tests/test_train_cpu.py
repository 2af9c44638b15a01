"""Host logic of the training step on CPU: flat buffers, AdamW vs torch.optim.AdamW, clip, and the
world_size-2 gradient exchange / naiveSyncBN1d over gloo."""
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch import nn

from geomae_amd.norm import NaiveSyncBatchNorm1d
from geomae_amd.train import FlatAdamW, FlatParams, allreduce_gradients, clip_grad_norm


class Toy(nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = nn.Linear(6, 5)
        self.norm = nn.LayerNorm(5)
        self.out = nn.Linear(5, 3)

    def forward(self, x):
        return self.out(self.norm(torch.relu(self.lin(x))))


@pytest.mark.parametrize("late", [(), ("norm.", "out."), (("norm.",), ("out.",))])
def test_flat_adamw_matches_torch_adamw(late):
    torch.manual_seed(0)
    a, b = Toy(), Toy()
    b.load_state_dict(a.state_dict())
    flat = FlatParams(a, no_decay_keys=("norm",), late_keys=late)
    opt = FlatAdamW(flat, lr=1e-2, weight_decay=0.05)
    nd = [p for n, p in b.named_parameters() if "norm" in n]
    dc = [p for n, p in b.named_parameters() if "norm" not in n]
    ref = torch.optim.AdamW([dict(params=nd, weight_decay=0.0), dict(params=dc, weight_decay=0.05)], lr=1e-2)
    assert late or flat.n_no_decay == sum(p.numel() for p in nd)
    covered = sum(e - s for s, e in flat.decay_ranges()) + sum(e - s for s, e in flat.nd_ranges)
    assert covered == flat.total and len(flat.nd_ranges) <= 2
    for it in range(5):
        x = torch.randn(16, 6)
        flat.zero_grad()
        a(x).pow(2).sum().backward()
        flat.check_views()
        gn = clip_grad_norm(flat, 10.0)
        opt.step()
        ref.zero_grad()
        b(x).pow(2).sum().backward()
        gn_ref = torch.nn.utils.clip_grad_norm_(b.parameters(), 10.0)
        ref.step()
        assert torch.allclose(gn, gn_ref, rtol=1e-5)
        for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
            assert torch.allclose(p, q, rtol=1e-5, atol=1e-6), (it, n)
    # parameters still alias the flat buffer
    assert all(p.data_ptr() >= flat.flat.data_ptr() for p in a.parameters())


def _worker(rank, world, port, tmp):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ.setdefault("GLOO_SOCKET_IFNAME", "lo")          # the container's hostname may not resolve
    os.environ["MASTER_PORT"] = str(port)
    import faulthandler
    faulthandler.dump_traceback_later(240, exit=True)          # a stuck rank reports where and leaves
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.manual_seed(0)
        m = Toy()
        flat = FlatParams(m)
        x = torch.randn(8, 6, generator=torch.Generator().manual_seed(100 + rank))
        flat.zero_grad()
        m(x).pow(2).sum().backward()
        flat.check_views()
        local = flat.grad.clone()
        allreduce_gradients(flat)
        gathered = [torch.zeros_like(local) for _ in range(world)]
        dist.all_gather(gathered, local)
        assert torch.allclose(flat.grad, sum(gathered) / world, atol=1e-6)
        # naiveSyncBN1d: equal weight per rank, different point counts per rank
        bn = NaiveSyncBatchNorm1d(4, eps=1e-3, momentum=0.01).train()
        xs = [torch.randn(10 + 7 * r, 4, generator=torch.Generator().manual_seed(r)) for r in range(world)]
        xin = xs[rank].clone().requires_grad_(True)
        y = bn(xin)
        mean = sum(t.mean(0) for t in xs) / world
        msq = sum((t * t).mean(0) for t in xs) / world
        var = msq - mean * mean
        want = (xs[rank] - mean) * torch.rsqrt(var + 1e-3)
        assert torch.allclose(y, want, atol=1e-5)
        assert torch.allclose(bn.running_var, 1 + 0.01 * (var - 1), atol=1e-6)
        y.sum().backward()
        assert torch.isfinite(xin.grad).all()
        # ---- the module against what the REFERENCE's NaiveSyncBatchNorm1d produced at world size 2
        # (tests/golden/g_syncbn_w2.npz part 1, oracle/make_golden_syncbn.py: N_0 = 37, N_1 = 53 rows, C = 8)
        import numpy as np
        from geomae_amd.norm import NaiveSyncBatchNorm2d
        gold = np.load(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "g_syncbn_w2.npz"))
        G = lambda k: torch.as_tensor(gold[f"r{rank}.{k}"])
        g = torch.Generator().manual_seed(40 + rank)
        n = (37, 53)[rank]
        x, w = torch.randn(n, 8, generator=g) * 2.0 + 0.5, torch.randn(n, 8, generator=g)
        for variant in ("1d", "2d"):
            mod = (NaiveSyncBatchNorm1d if variant == "1d" else NaiveSyncBatchNorm2d)(8, eps=1e-3, momentum=0.01).train()
            with torch.no_grad():
                mod.weight.copy_(torch.linspace(0.5, 1.5, 8))
                mod.bias.copy_(torch.linspace(-0.2, 0.3, 8))
            xin = x.clone().requires_grad_(True)
            shaped = xin if variant == "1d" else xin.t().reshape(1, 8, n, 1)         # same statistics as [n, 8]
            y = mod(shaped)
            y2 = y if variant == "1d" else y.reshape(8, n).t()
            (y2 * w).sum().backward()
            assert torch.allclose(y2, G("m_y"), rtol=1e-5, atol=1e-5), (variant, float((y2 - G("m_y")).abs().max()))
            assert torch.allclose(xin.grad, G("m_dx"), rtol=1e-4, atol=1e-5), (variant, float((xin.grad - G("m_dx")).abs().max()))
            assert torch.allclose(mod.weight.grad, G("m_dgamma"), rtol=1e-4, atol=1e-5), variant
            assert torch.allclose(mod.bias.grad, G("m_dbeta"), rtol=1e-4, atol=1e-5), variant
            assert torch.allclose(mod.running_mean, G("m_running_mean"), rtol=1e-5, atol=1e-6), variant
            assert torch.allclose(mod.running_var, G("m_running_var"), rtol=1e-5, atol=1e-6), variant
            assert int(mod.num_batches_tracked) == int(gold[f"r{rank}.m_num_batches_tracked"]) == 0
        # ---- Trainer construction makes the replicas identical (what MMDistributedDataParallel's constructor does):
        # parameters AND buffers come from rank 0 whatever each rank seeded
        from geomae_amd.train import Trainer

        class WithBuffer(nn.Module):
            def __init__(self):
                super().__init__()
                self.lin = nn.Linear(6, 5)
                self.bn = nn.BatchNorm1d(5)

            def forward_train(self, x, metas, **kw):
                return dict(loss=self.bn(self.lin(x)).pow(2).mean())

        torch.manual_seed(1000 + rank)                       # DIFFERENT initial weights per rank
        mb = WithBuffer()
        with torch.no_grad():
            mb.bn.running_mean.fill_(float(rank + 1))
            mb.bn.num_batches_tracked.fill_(7 * (rank + 1))
        tr = Trainer(mb)
        mine = torch.cat([tr.flat.flat, mb.bn.running_mean, mb.bn.num_batches_tracked.float().reshape(1)])
        both = [torch.zeros_like(mine) for _ in range(world)]
        dist.all_gather(both, mine)
        assert torch.equal(both[0], both[1]) and float(mb.bn.running_mean[0]) == 1.0 and int(mb.bn.num_batches_tracked) == 7
        # ... and stay identical through training steps on different data (gradients averaged, same update)
        for it in range(3):
            xs_ = torch.randn(12, 6, generator=torch.Generator().manual_seed(10 * it + rank))
            tr.train_step(xs_)
        mine = tr.flat.flat.clone()
        gathered = [torch.zeros_like(mine) for _ in range(world)]
        dist.all_gather(gathered, mine)
        assert torch.allclose(gathered[0], gathered[1], rtol=0, atol=0)
        torch.save(dict(ok=True), os.path.join(tmp, f"ok{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_world_size_2_gloo(tmp_path):
    import socket
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    assert all(os.path.exists(tmp_path / f"ok{r}.pt") for r in range(2))


def test_syncbn_single_process_is_plain_bn():
    bn = NaiveSyncBatchNorm1d(4, eps=1e-3, momentum=0.01).train()
    ref = nn.BatchNorm1d(4, eps=1e-3, momentum=0.01).train()
    x = torch.randn(32, 4)
    assert torch.allclose(bn(x), ref(x))
    assert torch.allclose(bn.running_var, ref.running_var)


def test_cyclic_lr_matches_mmcv_formula():
    """CyclicLrUpdaterHook restated (cosine_2x.py:10-15): target_ratio (100, 1e-3), cyclic_times 1, step_ratio_up 0.1."""
    import math
    from geomae_amd.train import CyclicLr
    base, T = 1e-5, 1000
    sch = CyclicLr(base, T)
    up = int(0.1 * T)
    assert sch.lr_at(0) == pytest.approx(base)
    assert sch.lr_at(up) == pytest.approx(base * 100)                       # top of the cycle
    assert sch.lr_at(up // 2) == pytest.approx(base * (100 + 0.5 * (1 - 100) * (math.cos(math.pi * 0.5) + 1)))
    assert base * 1e-3 <= sch.lr_at(T - 1) <= base * 2e-3                    # last iteration, one step before the bottom
    lrs = [sch.lr_at(i) for i in range(T)]
    assert all(a <= b for a, b in zip(lrs[:up], lrs[1:up + 1])) and all(a >= b for a, b in zip(lrs[up:-1], lrs[up + 1:]))


def test_checkpoint_roundtrip_mmcv_layout(tmp_path):
    """{'meta','state_dict','optimizer'} with torch.optim.AdamW-shaped optimizer state (one group per parameter)."""
    import torch.nn as nn
    from geomae_amd.train import FlatAdamW, FlatParams, Trainer

    class Tiny(nn.Module):
        def __init__(self):
            super().__init__()
            self.lin = nn.Linear(4, 3)
            self.norm = nn.LayerNorm(3)

        def forward_train(self, points, metas, **kw):
            return dict(loss=self.norm(self.lin(points)).pow(2).mean())

    torch.manual_seed(0)
    tr = Trainer(Tiny())
    x = torch.randn(5, 4)
    for _ in range(3):
        tr.train_step(x)
    path = str(tmp_path / "epoch_1.pth")
    tr.save_checkpoint(path, meta=dict(epoch=1))
    ck = torch.load(path, weights_only=False)
    assert set(ck) == {"meta", "state_dict", "optimizer"} and ck["meta"]["epoch"] == 1 and ck["meta"]["iter"] == 3
    groups = ck["optimizer"]["param_groups"]
    assert len(groups) == 4
    # ... in model.named_parameters() order (what mmcv / torch.optim index by), NOT the flat buffer's segment order
    model_params = [p for _, p in tr.model.named_parameters()]
    assert [tuple(ck["optimizer"]["state"][i]["exp_avg"].shape) for i in range(4)] == [tuple(p.shape) for p in model_params]
    assert [g["weight_decay"] for g in groups] == [0.05, 0.05, 0.0, 0.0]           # lin.weight, lin.bias, norm.weight, norm.bias
    ref = torch.optim.AdamW([dict(params=[nn.Parameter(torch.zeros_like(p))]) for p in model_params])   # loads into torch's own
    ref.load_state_dict(dict(state=ck["optimizer"]["state"],
                             param_groups=[dict(g, maximize=False, foreach=None, capturable=False, differentiable=False,
                                                fused=None, decoupled_weight_decay=True) for g in groups]))
    torch.manual_seed(1)
    tr2 = Trainer(Tiny())
    tr2.load_checkpoint(path)
    assert tr2.iter == 3 and tr2.opt.step_count == 3
    for a, b in zip(tr.flat.params, tr2.flat.params):
        assert torch.equal(a, b)
    l1, _ = tr.train_step(x)
    l2, _ = tr2.train_step(x)
    assert torch.equal(l1["loss"], l2["loss"])
    for a, b in zip(tr.flat.params, tr2.flat.params):
        assert torch.equal(a, b)
    # torch.optim.AdamW built on the MODEL's parameter list continues identically from the same checkpoint
    torch.manual_seed(2)
    m3 = Tiny()
    m3.load_state_dict(ck["state_dict"])
    ps = list(m3.parameters())
    o3 = torch.optim.AdamW([dict(params=[p], weight_decay=g["weight_decay"]) for p, g in zip(ps, groups)], lr=groups[0]["lr"])
    sd3 = o3.state_dict()
    sd3["state"] = {i: {k: (v.clone() if torch.is_tensor(v) else v) for k, v in st.items()} for i, st in ck["optimizer"]["state"].items()}
    o3.load_state_dict(sd3)
    torch.manual_seed(1)
    tr4 = Trainer(Tiny())
    tr4.load_checkpoint(path)
    out = m3.forward_train(x, None)["loss"]
    out.backward()
    torch.nn.utils.clip_grad_norm_(ps, tr4.grad_clip["max_norm"])
    o3.step()
    tr4.train_step(x)
    for (n, a), b in zip(tr4.model.named_parameters(), ps):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-7), n
    # a checkpoint of another parameter order / model is refused, not silently mis-assigned
    bad = dict(ck["optimizer"])
    bad["state"] = {0: ck["optimizer"]["state"][2], 1: ck["optimizer"]["state"][1], 2: ck["optimizer"]["state"][0],
                    3: ck["optimizer"]["state"][3]}
    with pytest.raises(ValueError, match="shape"):
        tr4.opt.load_state_dict(bad)


def test_zero_arena_carves_aligned_zero_views():
    """ops.ZeroArena: one zero-filled buffer handed out as typed, 256-byte aligned views (the accumulator buffers of a
    training step); carving past the sized total is an error, not a silent overlap."""
    from geomae_amd.ops import ZeroArena
    specs = [((5, 3), torch.float32), ((7,), torch.float64), ((2, 128), torch.float32), ((6,), torch.int64)]
    total = ZeroArena.nbytes(*specs)
    assert total % 256 == 0 and total >= sum(torch.empty(s, dtype=d).numel() * torch.empty((), dtype=d).element_size() for s, d in specs)
    arena = ZeroArena(total, "cpu")
    views = [arena.take(s, d) for s, d in specs]
    for v, (s, d) in zip(views, specs):
        assert v.shape == torch.Size(s) and v.dtype == d and not v.any() and v.data_ptr() % 256 == arena.buf.data_ptr() % 256
    views[0].fill_(1.0)                                   # views do not overlap
    assert not views[1].any() and not views[2].any() and not views[3].any()
    with pytest.raises(RuntimeError):
        arena.take((1024,), torch.float32)


def test_checkpoint_indices_count_frozen_parameters(tmp_path):
    """A frozen parameter (the fine-tune configs freeze parts of the model) keeps its slot in the optimizer
    checkpoint's index space -- mmcv's DefaultOptimizerConstructor / torch.optim list every parameter of the model, so
    skipping the frozen ones would shift every later index."""
    import torch.nn as nn
    from geomae_amd.train import Trainer

    class Tiny(nn.Module):
        def __init__(self):
            super().__init__()
            self.a = nn.Linear(4, 3)
            self.frozen = nn.Linear(3, 3)
            self.b = nn.Linear(3, 2)
            for p in self.frozen.parameters():
                p.requires_grad_(False)

        def forward_train(self, points, metas, **kw):
            return dict(loss=self.b(self.frozen(self.a(points))).pow(2).mean())

    torch.manual_seed(0)
    tr = Trainer(Tiny())
    x = torch.randn(5, 4)
    for _ in range(2):
        tr.train_step(x)
    sd = tr.opt.state_dict()
    names = [n for n, _ in tr.model.named_parameters()]
    assert names == ["a.weight", "a.bias", "frozen.weight", "frozen.bias", "b.weight", "b.bias"]
    assert len(sd["param_groups"]) == 6 and sorted(sd["state"]) == [0, 1, 4, 5]
    assert tuple(sd["state"][4]["exp_avg"].shape) == (2, 3) and tuple(sd["state"][5]["exp_avg"].shape) == (2,)
    path = str(tmp_path / "ck.pth")
    tr.save_checkpoint(path)
    torch.manual_seed(1)
    tr2 = Trainer(Tiny())
    tr2.load_checkpoint(path)
    assert torch.equal(tr2.opt.exp_avg, tr.opt.exp_avg) and torch.equal(tr2.opt.exp_avg_sq, tr.opt.exp_avg_sq)
    l1, _ = tr.train_step(x)
    l2, _ = tr2.train_step(x)
    assert torch.equal(l1["loss"], l2["loss"])


def test_flat_adamw_refuses_codes_and_a_refused_state_changes_nothing():
    """8-bit codes (optim.MultiTensorAdamW) of the parameters' shapes are not moments; a state whose last entry does not fit leaves the
    first ones alone."""
    torch.manual_seed(0)
    flat = FlatParams(Toy(), no_decay_keys=("norm",))
    opt = FlatAdamW(flat)
    opt.exp_avg.normal_()
    opt.exp_avg_sq.uniform_()
    good = opt.state_dict()
    kept = opt.exp_avg.clone(), opt.exp_avg_sq.clone()
    codes = {i: dict(step=torch.tensor(3), exp_avg=torch.full_like(st["exp_avg"], 56, dtype=torch.uint8),
                     exp_avg_sq=torch.full_like(st["exp_avg_sq"], 99, dtype=torch.uint8)) for i, st in good["state"].items()}
    other = {i: dict(step=torch.tensor(3.0), exp_avg=torch.ones_like(st["exp_avg"]), exp_avg_sq=torch.ones_like(st["exp_avg_sq"]))
             for i, st in good["state"].items()}
    last = max(other)
    short = {**other, last: {**other[last], "exp_avg_sq": torch.ones(1)}}
    for sd, match in ((dict(good, state=codes), "uint8"), (dict(good, state=other, state_bits=8), "8 bits"), (dict(good, state=short), "shape"),
                      (dict(good, state={**other, 99: other[0]}), "does not have")):
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(sd)
        assert torch.equal(opt.exp_avg, kept[0]) and torch.equal(opt.exp_avg_sq, kept[1]) and opt.step_count == 0
    opt.load_state_dict(dict(good, state=other))
    assert opt.step_count == 3 and all((opt.exp_avg[o:o + p.numel()] == 1).all() for p, o in zip(flat.params, flat.offsets))


def test_flat_adamw_refuses_a_state_in_the_order_of_groups():
    """Same shapes at other places: a state in the order [decayed | undecayed] would go to other parameters without an error."""
    class Square(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.a = nn.Parameter(torch.ones(4)), nn.Parameter(torch.ones(4))
    opt = FlatAdamW(FlatParams(Square(), no_decay_keys=("norm",)))
    entry = lambda v: dict(step=torch.tensor(1), exp_avg=torch.full((4,), v), exp_avg_sq=torch.full((4,), v))
    groups = [dict(params=[0], lr=1e-3), dict(params=[1], lr=1e-3)]
    state = dict(state={0: entry(1.0), 1: entry(2.0)}, param_groups=groups, state_bits=32, master_weights=False, seed=0)
    with pytest.raises(ValueError, match="order of its groups"):
        opt.load_state_dict(state)
    assert not opt.exp_avg.any() and opt.step_count == 0
    opt.load_state_dict(dict(state, parameter_order="model"))
    assert (opt.exp_avg[opt.flat.offsets[opt.flat.names.index("a")]:][:4] == 2.0).all()
    opt.load_state_dict(dict(state, param_groups=[dict(params=[0, 1], lr=1e-3)]))
