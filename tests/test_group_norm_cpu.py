"""Group norm with an activation: its place in the registry and the fine-tune model, and what it refuses (no GPU)."""
import pytest
import torch
from torch import nn


def test_gn_resolves_and_has_group_norms_parameters():
    from geomae_amd.norm import GroupNormAct, build_norm_relu
    from geomae_amd.registry import build_norm_layer
    name, m = build_norm_layer(dict(type="GN", num_groups=8, eps=1e-3, requires_grad=True), 64)
    assert name == "GN" and isinstance(m, GroupNormAct) and m.eps == 1e-3 and m.activation is None
    assert m.state_dict().keys() == nn.GroupNorm(8, 64).state_dict().keys()
    m.load_state_dict(nn.GroupNorm(8, 64).state_dict())
    assert not list(GroupNormAct(64, 8, affine=False).parameters())
    norm, act = build_norm_relu(dict(type="GN", num_groups=8), 64)
    assert norm.activation == "relu" and isinstance(act, nn.Identity)
    norm, act = build_norm_relu(dict(type="GN", num_groups=8, activation="silu"), 64)
    assert norm.activation == "silu"
    norm, act = build_norm_relu(dict(type="BN"), 64)
    assert isinstance(norm, nn.BatchNorm2d) and isinstance(act, nn.ReLU)
    with pytest.raises(ValueError, match="divide"):
        GroupNormAct(64, 7)


def test_finetune_model_keeps_its_parameter_names():
    import geomae_amd
    from geomae_amd.configs import pre_sst_model
    cfg = pre_sst_model(num_blocks=1, conv_out_channels=(32, 32, 64), layer_nums=(1, 1, 1))
    cfg.pop("bbox_head")
    names = set(geomae_amd.build_model(cfg).state_dict())
    gn = dict(type="GN", num_groups=8)
    cfg["backbone"]["norm_cfg"], cfg["neck"]["norm_cfg"] = gn, gn
    model = geomae_amd.build_model(cfg)
    running = ("running_mean", "running_var", "num_batches_tracked")
    conv = lambda n: n.startswith(("backbone.conv_blocks.", "neck."))
    assert set(model.state_dict()) == {n for n in names if not (conv(n) and n.endswith(running))}
    assert all(m.activation == "relu" for n, m in model.named_modules() if type(m).__name__ == "GroupNormAct")


def test_layouts_are_recognised():
    from geomae_amd import ops
    x = torch.randn(2, 6, 3, 4)
    assert not ops._channels_last(x) and ops._channels_last(x.to(memory_format=torch.channels_last))
    assert ops._channels_last(torch.randn(5, 6)) and not ops._channels_last(torch.randn(6, 5).t())
    assert ops._channels_last(torch.randn(2, 4, 6).transpose(1, 2)) and not ops._channels_last(torch.randn(2, 6, 4))
    assert ops._channels_last(ops._to_channels_last(x)) and torch.equal(ops._to_channels_last(x), x)
    assert not ops._channels_last(torch.randn(2, 4, 5, 8).movedim(-1, 1)[:, :6])


def test_refusals_need_no_gpu():
    from geomae_amd import ops
    from geomae_amd.norm import GroupNormAct
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.group_norm_act(torch.zeros(2, 4), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        GroupNormAct(4, 2)(torch.zeros(2, 4, 3, 3))


def test_entry_points_check_their_arguments():
    from geomae_amd import _lib
    lib = _lib.load()
    wsb, rows = lib.geomae_group_norm_workspace_bytes, 100_000            # rows of a group that no workgroup holds
    assert wsb(0, rows, 8, 2, 0, 0) == 0 and wsb(2, 0, 8, 2, 0, 1) == 0
    assert 0 < wsb(2, rows, 8, 2, 0, 0) and 0 < wsb(2, rows, 8, 2, 0, 1) < wsb(200, rows, 8, 2, 0, 1)
    assert wsb(2, 10, 8, 2, 0, 0) >= 0 and wsb(2, 10, 8, 2, 0, 1) > 0
    for bad in ((2, rows, 8, 3, 0, 0), (-1, rows, 8, 2, 0, 0), (2, rows, 0, 1, 0, 0), (2, rows, 8, 2, 3, 0), (2, rows, 4096, 2048, 0, 0)):
        assert wsb(*bad) == -1, bad

    def forward(x=64, dtype=0, n=2, rows=rows, c=8, groups=2, eps=1e-5, act=0, ws=64, bytes_=1 << 20):
        return lib.geomae_group_norm_forward(x, dtype, n, rows, c, groups, None, None, 0, eps, act, 64, 64, ws, bytes_, None)
    assert forward(n=0) == 0 and forward(rows=0) == 0
    assert forward(x=None) < 0 and b"null" in lib.geomae_last_error()
    assert forward(groups=3) < 0 and b"divide" in lib.geomae_last_error()
    assert forward(act=4) < 0 and forward(eps=-1.0) < 0 and forward(dtype=7) < 0
    assert forward(bytes_=8) == -3 and forward(ws=None) == -3

    def backward(dy=64, n=2, bytes_=1 << 20):
        return lib.geomae_group_norm_backward(64, dy, 0, n, rows, 8, 2, None, None, 0, 0, 64, 64, None, None, 64, bytes_, None)
    assert backward(n=0) == 0 and backward(dy=None) < 0 and backward(bytes_=8) == -3


def test_more_threads_than_a_launch_counts_are_refused():
    """Rows [N, C] as samples of one row each: one workgroup of 64 threads for up to 128 bytes of a row."""
    from geomae_amd import _lib
    lib = _lib.load()
    ok = lib.geomae_group_norm_workspace_bytes((1 << 26) - 1, 1, 64, 8, 1, 0)
    assert ok == 0
    assert lib.geomae_group_norm_workspace_bytes(1 << 26, 1, 64, 8, 1, 0) == -1 and b"too many" in lib.geomae_last_error()
    assert lib.geomae_group_norm_forward(64, 1, 1 << 26, 1, 64, 8, None, None, 0, 1e-5, 0, 64, 64, None, 0, None) < 0
    assert lib.geomae_group_norm_backward(64, 64, 1, 1 << 26, 1, 64, 8, None, None, 0, 0, 64, 64, None, None, None, 0, None) < 0


def test_channels_that_32_bit_offsets_do_not_reach_are_refused():
    from geomae_amd import _lib
    lib = _lib.load()
    assert lib.geomae_group_norm_workspace_bytes(1, 5, 1 << 22, 1024, 0, 0) >= 0
    assert lib.geomae_group_norm_workspace_bytes(1, 5, (1 << 22) + 1024, 1024, 0, 0) == -1 and b"channels" in lib.geomae_last_error()


def test_forward_mode_and_traces_are_refused():
    """A dual tensor does not require a gradient, and a trace records no kernel: both would come back without an error as a zero
    derivative and as memory that nothing wrote."""
    import torch.autograd.forward_ad as fwAD
    from geomae_amd import ops
    x, w, b = torch.randn(2, 4), torch.ones(4), torch.zeros(4)
    for grad in (torch.enable_grad, torch.no_grad):
        with grad(), fwAD.dual_level():
            for k in range(3):
                args = [fwAD.make_dual(t, torch.ones_like(t)) if i == k else t for i, t in enumerate((x, w, b))]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    ops.group_norm_act(args[0], 2, args[1], args[2])
        with grad(), pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(lambda t: ops.group_norm_act(t, 2), (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="CUDA"):                       # (outside of both it is the device that is refused)
        ops.group_norm_act(x, 2, w, b)
