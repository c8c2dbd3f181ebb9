"""lpgnn.optim on the CPU: refusals, the rounding's hash and format (no kernels run)."""
import pytest
import torch

import adamw_ref as R


def test_refuses_host_tensors_and_bad_settings():
    from lpgnn import optim

    t = [torch.ones(3)]
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.adamw_step(t, t, t, t, step=1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        optim.clip_scale(t, 1.0)
    with pytest.raises(RuntimeError, match="no gradients"):
        optim.clip_scale([], 1.0)
    with pytest.raises(RuntimeError, match="max_norm"):
        optim.clip_scale(t, -1.0)
    optim.adamw_step([], [], [], [], step=1)  # nothing to do
    p = [torch.nn.Parameter(torch.ones(3))]
    for kw in (dict(state_bits=16), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **kw)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0)):
        with pytest.raises(RuntimeError, match="need lr"):
            optim.AdamW(p, **kw)
    o = optim.AdamW(p)
    p[0].grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        o.step()


def test_c_entry_refusals():
    import ctypes

    from lpgnn import _lib

    L = _lib.lib()
    ok = (0.9, 0.1, 0.999, 0.001, 1.0, 1e-8, 1.0, 1e-3)
    h = _lib.LpgAdamwHyper(*ok)
    p = 1 << 20  # never dereferenced
    i64 = lambda *a: (ctypes.c_int64 * len(a))(*a)
    good, good8 = i64(p, p, p, p, 4), i64(p, p, p, p, p, p, 4, 0)
    for call, row, name in ((L.lpg_adamw, good, b"lpg_adamw"), (L.lpg_adamw8, good8, b"lpg_adamw8")):
        assert call(1, 1, row, h, None, None) == 1 and name in L.lpg_last_error()
        assert call(2, -1, row, h, None, None) == 1
        assert call(2, 1, None, h, None, None) == 1
        assert call(2, 1, row, None, None, None) == 1
        bad = row[:]
        bad[-1 if call is L.lpg_adamw else -2] = -1
        assert call(2, 1, i64(*bad), h, None, None) == 1
        for k in range(4 if call is L.lpg_adamw else 6):
            bad = row[:]
            bad[k] = 0
            assert call(2, 1, i64(*bad), h, None, None) == 1, k
        for k, v in ((0, 1.0), (0, -0.1), (2, 1.0), (5, -1.0), (5, float("nan"))):
            hh = list(ok)
            hh[k] = v
            assert call(2, 1, row, _lib.LpgAdamwHyper(*hh), None, None) == 1
        assert call(2, 0, None, h, None, None) == 0
    assert L.lpg_grad_norm_workspace_bytes(-1, None) == -1
    assert L.lpg_grad_norm_workspace_bytes(1, i64(p, -1)) == -1
    # one fp64 sum a chunk of 4096 numbers, of 16384 above 2^24 in all
    assert L.lpg_grad_norm_workspace_bytes(2, i64(p, 16384, p, 16385)) == 8 * (4 + 5)
    assert L.lpg_grad_norm_workspace_bytes(2, i64(p, 2 ** 24, p, 1)) == 8 * (1024 + 1)
    assert L.lpg_grad_norm(2, 1, i64(p, 4), -1.0, p, p, p, None) == 1
    assert L.lpg_grad_norm(0, 1, i64(0, 4), 1.0, p, p, p, None) == 1
    assert L.lpg_grad_norm(2, 1, i64(p, 4), 1.0, None, p, p, None) == 1
    big = i64(p, p, p, p, (1 << 31) * 4096)
    assert L.lpg_adamw(2, 1, big, h, None, None) == 3 and b"too large" in L.lpg_last_error()


def test_keys_are_the_reference_hash():
    from lpgnn import optim

    for seed in (0, 5, (7 << 32) | 9):
        assert optim.rounding_keys(range(3), 11, seed) == [R.key(t, 11, seed) for t in range(3)]
    assert len({k for s in range(50) for k in optim.rounding_keys(range(50), s, 1)}) > 2495


def test_reference_rounding_is_right_on_average():
    """The mean over all 65536 random values of a number's rounding is the number, to 2^-17 of a step."""
    u = torch.arange(65536)
    for t in (0.3, 5.7e-3, 440.0, 0.015624):
        x = torch.zeros(65536, R.BLOCK)
        x[:, 0], x[:, 1] = 448.0, t
        v, s = R.encode32(x, u[:, None].expand(-1, R.BLOCK))
        assert (s == 1).all() and (v[:, 0] == 448).all()
        step = 2.0 ** (max(torch.frexp(torch.tensor(t)).exponent.item() - 1, -6) - 3)
        assert set(v[:, 1].tolist()) <= {int(t / step) * step, (int(t / step) + 1) * step}
        assert abs(v[:, 1].double().mean().item() - torch.tensor(t).item()) <= step * 2.0 ** -16


def test_state_dict_round_trip_keeps_types():
    from lpgnn import optim

    p = torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16))
    o = optim.AdamW([p], state_bits=8)
    o.state[p].update(o._init(p))
    o.state[p]["m_scale"][1] = 1 / 3
    o.state[p]["step"] = 7
    q = optim.AdamW([torch.nn.Parameter(p.detach().clone())], state_bits=8)
    q.load_state_dict(o.state_dict())
    st = q.state[q.param_groups[0]["params"][0]]
    assert st["step"] == 7 and st["m8"].dtype == torch.float8_e4m3fn and st["r_scale"].dtype == torch.float32
    assert torch.equal(st["m_scale"], o.state[p]["m_scale"]) and st["m_scale"].data_ptr() != o.state[p]["m_scale"].data_ptr()


def test_refuses_forward_mode_tangents():
    """The updates drop a tangent, as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    from lpgnn import optim

    t = lambda: torch.ones(3)
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(t(), t())
        for k in range(4):
            ts = [[t()] for _ in range(4)]
            ts[k] = [dual]
            with pytest.raises(RuntimeError, match="forward-mode"):
                optim.adamw_step(*ts, step=1)
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim.adamw_step([t()], [t()], [t()], [t()], step=1, grad_scale=dual)
        for k in (0, 1, 3, 5):
            ts = [[t()] for _ in range(6)]
            ts[k] = [dual]
            with pytest.raises(RuntimeError, match="forward-mode"):
                optim.adamw_step_8bit(*ts, step=1)
        with pytest.raises(RuntimeError, match="forward-mode"):
            optim.clip_scale([dual], 1.0)


@pytest.mark.parametrize("flag", ["maximize", "amsgrad"])
def test_refuses_other_updates_of_a_loaded_state(flag):
    """torch's options that change the update: from a state dict, from a group, and set later."""
    from lpgnn import optim

    p = torch.nn.Parameter(torch.ones(3))
    t = torch.optim.AdamW([p], **{flag: True})
    p.grad = torch.ones(3)
    t.step()
    o = optim.AdamW([p])
    with pytest.raises(RuntimeError, match=flag):
        o.load_state_dict(t.state_dict())
    assert not o.state and flag not in o.param_groups[0]  # nothing of it was taken
    with pytest.raises(RuntimeError, match=flag):
        optim.AdamW([{"params": [p], flag: True}])
    with pytest.raises(RuntimeError, match=flag):
        optim.AdamW([p]).add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], flag: True})
    o.param_groups[0][flag] = True
    with pytest.raises(RuntimeError, match=flag):
        o.step()
    plain = torch.optim.AdamW([p], **{flag: False})
    plain.step()
    optim.AdamW([p]).load_state_dict(plain.state_dict())


def test_loads_moments_of_other_types():
    """torch keeps the moments of bf16 parameters in bf16 (of fp64 ones in fp64): they become the fp32 the step takes."""
    from lpgnn import optim

    for dtype in (torch.bfloat16, torch.float64):
        p = torch.nn.Parameter(torch.ones(5, dtype=dtype))
        p.grad = torch.linspace(-1, 1, 5).to(dtype)
        t = torch.optim.AdamW([p])
        t.step()
        q = torch.nn.Parameter(torch.ones(5, dtype=torch.bfloat16))
        o = optim.AdamW([q])
        o.load_state_dict(t.state_dict())
        assert o.state[q]["step"] == 1
        for k in ("exp_avg", "exp_avg_sq"):
            assert t.state[p][k].dtype == dtype and o.state[q][k].dtype == torch.float32
            assert torch.equal(o.state[q][k], t.state[p][k].float())


def test_copies_and_pickles_keep_the_settings():
    """torch's Optimizer pickles and deep-copies its groups and state only."""
    import copy
    import io

    from lpgnn import optim

    p = torch.nn.Parameter(torch.ones(300))
    o = optim.AdamW([p], state_bits=8, max_grad_norm=0.5, seed=7)
    o.state[p].update(o._init(p))
    o.last_norm = torch.tensor(3.0)
    buf = io.BytesIO()
    torch.save(o, buf)
    buf.seek(0)
    for c in (copy.deepcopy(o), torch.load(buf, weights_only=False)):
        assert (c.state_bits, c.max_grad_norm, c.seed, c.last_norm) == (8, 0.5, 7, 3.0)
        assert c.param_groups[0]["params"][0] is not p and len(c.state) == 1
        assert c.state_dict().keys() == o.state_dict().keys()


def test_seed_is_checked_where_it_is_given():
    """The 8-bit rounding's seed is 64 bits: refused where it is given, not in the first step."""
    from lpgnn import optim

    p = torch.nn.Parameter(torch.ones(3))
    for seed in (-1, 1 << 64):
        with pytest.raises(ValueError, match="seed"):
            optim.AdamW([p], state_bits=8, seed=seed)
    assert optim.AdamW([p], state_bits=8, seed=(1 << 64) - 1).seed == (1 << 64) - 1


def test_c_entries_refuse_more_blocks_than_a_launch_holds():
    """Fewer than 2^32 threads a launch: 2^24 blocks of 256 are too many (numbers a block: 4096, 1024, 16384)."""
    import ctypes

    from lpgnn import _lib

    L = _lib.lib()
    h = _lib.LpgAdamwHyper(0.9, 0.1, 0.999, 0.001, 1.0, 1e-8, 1.0, 1e-3)
    p = 1 << 20  # never dereferenced
    i64 = lambda *a: (ctypes.c_int64 * len(a))(*a)
    assert L.lpg_adamw(2, 1, i64(p, p, p, p, 1 << 36), h, None, None) == 3 and b"too large" in L.lpg_last_error()
    assert L.lpg_adamw8(2, 1, i64(p, p, p, p, p, p, 1 << 34, 0), h, None, None) == 3
    assert b"too large" in L.lpg_last_error()
    assert L.lpg_grad_norm(2, 1, i64(p, 1 << 38), 1.0, p, p, p, None) == 3 and b"too large" in L.lpg_last_error()


def test_c_entries_refuse_before_the_first_launch():
    """A tensor too large behind others that are not: nothing of the call may run (here a launch would be error 2)."""
    import ctypes

    from lpgnn import _lib

    L = _lib.lib()
    h = _lib.LpgAdamwHyper(0.9, 0.1, 0.999, 0.001, 1.0, 1e-8, 1.0, 1e-3)
    p = 1 << 20  # never dereferenced
    i64 = lambda *a: (ctypes.c_int64 * len(a))(*a)
    assert L.lpg_adamw(2, 2, i64(p, p, p, p, 4, p, p, p, p, 1 << 36), h, None, None) == 3
    assert L.lpg_adamw8(2, 2, i64(p, p, p, p, p, p, 4, 0, p, p, p, p, p, p, 1 << 34, 0), h, None, None) == 3
    assert L.lpg_grad_norm(2, 2, i64(p, 4, p, 1 << 38), 1.0, p, p, p, None) == 3
