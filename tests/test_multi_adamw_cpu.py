"""The 8-bit moments' format and rounding, by their definition (no GPU), and what MultiTensorAdamW refuses."""
import adamw_definition as D
import numpy as np
import pytest
import torch


def test_codes_are_increasing_and_exact_in_bfloat16():
    for table, top in ((D.SIGNED[:127], 448.0), (D.ROOT[:255], 480.0)):
        assert (np.diff(table) > 0).all() and table[0] == 0 and table[-1] == top
        as_bf16 = torch.tensor(table, dtype=torch.float64).to(torch.bfloat16).double().numpy()
        assert np.array_equal(as_bf16, table)


@pytest.mark.parametrize("table", [D.SIGNED, D.ROOT], ids=["first", "second"])
def test_a_value_that_a_code_stands_for_is_kept(table):
    """Re-encoding a decoded block changes nothing, whatever the draw: no drift where the moments stand still."""
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 127 if table is D.SIGNED else 255, 32 * 40)
    x = D.decode(codes, rng.integers(40, 200, 40), table)
    for u in (0, 1, 40000, 65535):
        back, _, _ = D.encode(x, np.full(x.size, u), table)
        assert np.array_equal(back, x)


@pytest.mark.parametrize("table", [D.SIGNED, D.ROOT], ids=["first", "second"])
def test_rounding_is_unbiased(table):
    """Over many draws the mean of a rounded value is the value: within 5 standard errors, the error of one draw being at most
    a step, 2^-3 resp. 2^-4 of the value."""
    n, x0 = 20000, 0.6180339
    u = D.draws(7, 3, 11, n)[0 if table is D.SIGNED else 1]
    x = np.full(n, x0)
    val, _, _ = D.encode(x, u, table)
    step = 2.0 ** -(4 if table is D.SIGNED else 5)                        # of a value in [0.5, 1)
    assert set(np.round((val - val.min()) / step).astype(int)) == {0, 1}
    assert abs(val.mean() - x0) < 5 * (step / 2) / np.sqrt(n)


def test_draws_are_even_and_unrelated():
    """Each 16-bit half is even over its range and unrelated to the other half, the next element, the next step and the next
    tensor: correlations and 64-bin counts within 5 standard errors."""
    n = 1 << 16
    a, b = (h.astype(np.float64) for h in D.draws(0, 0, 1, n))
    others = [a[1:], D.draws(0, 0, 2, n)[0], D.draws(0, 1, 1, n)[0], D.draws(1, 0, 1, n)[0], b]
    for x in (a, b):
        counts = np.bincount((x // 1024).astype(int), minlength=64)
        assert np.abs(counts - n / 64).max() < 5 * np.sqrt(n / 64)
        assert abs(x.mean() - 32767.5) < 5 * 18918 / np.sqrt(n)
    for x in others:
        r = np.corrcoef(a[:x.size], x.astype(np.float64))[0, 1]
        assert abs(r) < 5 / np.sqrt(n)


def test_the_second_moment_follows_its_gradients():
    """What the stochastic rounding is for: with beta2 = 0.999 the held root decays when the gradients vanish (to the nearest
    it would stay where it is for ever).  After 2000 steps without a gradient: exp(-1) of the start, within 20 %."""
    r = np.full(32 * 8, 1.0)
    for s in range(1, 2001):
        r, _, _ = D.encode(np.sqrt(r * r * 0.999), D.draws(0, 0, s, r.size)[1], D.ROOT)
    assert abs(r.mean() / np.exp(-1.0) - 1) < 0.2


def test_refusals_need_no_gpu():
    from geomae_amd.optim import MultiTensorAdamW, _dense
    p = torch.nn.Parameter(torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        MultiTensorAdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        MultiTensorAdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="betas"):
        MultiTensorAdamW([p], betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="negative"):
        MultiTensorAdamW([p], eps=-1.0)
    with pytest.raises(ValueError, match="seed"):
        MultiTensorAdamW([p], seed=-1)
    assert _dense(torch.empty(2, 3, 4, 5).to(memory_format=torch.channels_last)) and _dense(torch.empty(3, 4).t())
    assert not _dense(torch.empty(4, 6)[:, :3]) and not _dense(torch.empty(1, 5).expand(3, 5))
    assert _dense(torch.empty(())) and _dense(torch.empty(0, 5))


def test_entry_points_check_their_arguments():
    import ctypes
    from geomae_amd import _lib
    lib = _lib.load()
    chunk = lib.geomae_multi_adamw_chunk()
    assert chunk > 0 and chunk % 32 == 0
    assert lib.geomae_multi_adamw_workspace_bytes(-1) == -1
    small, large = lib.geomae_multi_adamw_workspace_bytes(1), lib.geomae_multi_adamw_workspace_bytes(1000)
    assert 0 < small < large

    def call(n, bits=32, ws=None, wsb=0, hyper=0):
        one = (ctypes.c_int64 * 2)(0, 1)
        grads, which = (ctypes.c_void_p * 1)(64), (ctypes.c_int32 * 1)(hyper)
        hypers = (_lib.GeomaeAdamwHyper * 1)()
        return lib.geomae_multi_adamw_step(64, 64, one, n, grads, which, ctypes.addressof(hypers), 1, bits, 0.0, 1.0, None, 0, 0,
                                           None, ws, wsb, None)
    assert call(0) == 0                                                # nothing to do
    assert call(-1) < 0 and call(1, bits=16) < 0 and b"state_bits" in lib.geomae_last_error()
    assert call(1) == -3 and b"workspace" in lib.geomae_last_error()
    assert call(1, ws=256, wsb=1 << 20, hyper=1) < 0 and b"out of range" in lib.geomae_last_error()
    assert lib.geomae_multi_adamw_step(None, None, None, 1, None, None, None, 0, 32, 0.0, 1.0, None, 0, 0, None, None, 0, None) < 0
    assert lib.geomae_adamw_moments8(None, None, None, None, 33, None, None, None) < 0
    assert lib.geomae_adamw_moments8(None, None, None, None, 32, None, None, None) < 0
    assert lib.geomae_adamw_moments8(None, None, None, None, 0, None, None, None) == 0


def test_a_plan_notices_a_parameter_cut_or_cast_where_it_lies():
    """The device table holds lengths: a parameter at the same address but of another size, order or type is not stepped."""
    from geomae_amd import _lib
    for change in (lambda t: t[:3], lambda t: t.t(), lambda t: t.view(torch.int32), lambda t: t.reshape(-1), lambda t: t[:1].expand(4, 5)):
        p = torch.nn.Parameter(torch.zeros(4, 5), requires_grad=False)
        plan = _lib.host().AdamwPlan([p], [0, 1], 0, 0, 0, 0, 0, 32)
        where = p.data_ptr()
        p.data = change(p.data)
        assert p.data_ptr() == where
        group = dict(params=[p], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
        assert plan.step([group], 0.0, 1.0, None, False) is False
        assert plan.step([dict(group, params=[])], 0.0, 1.0, None, False) is False


def test_a_clipping_norm_is_not_negative():
    import ctypes
    from geomae_amd import _lib
    lib = _lib.load()
    one, grads, which = (ctypes.c_int64 * 2)(0, 1), (ctypes.c_void_p * 1)(64), (ctypes.c_int32 * 1)(0)
    hypers = (_lib.GeomaeAdamwHyper * 1)()
    for bad in (-1.0, float("nan")):
        assert lib.geomae_multi_adamw_step(64, 64, one, 1, grads, which, ctypes.addressof(hypers), 1, 32, bad, 1.0, None, 0, 0, None, None,
                                           0, None) < 0 and b"max_norm" in lib.geomae_last_error()


def test_memory_orders():
    from geomae_amd.optim import _memory_order
    x = torch.empty(2, 3, 4, 5)
    assert _memory_order(x) == [0, 1, 2, 3] and _memory_order(x.to(memory_format=torch.channels_last)) == [0, 2, 3, 1]
    assert _memory_order(torch.empty(3, 4).t()) == [1, 0] and _memory_order(torch.empty(())) == [] == _memory_order(torch.empty(0, 4))
    one = torch.empty(6, 1, 5, 1)                                         # dimensions of one element do not count
    assert _memory_order(one) == [0, 2] == _memory_order(one.to(memory_format=torch.channels_last))


def test_no_parameter_at_all_is_refused():
    from geomae_amd.optim import MultiTensorAdamW
    for none in ([{"params": []}], [{"params": []}, {"params": []}], []):
        with pytest.raises(ValueError, match="no parameter|empty parameter list"):
            MultiTensorAdamW(none)
