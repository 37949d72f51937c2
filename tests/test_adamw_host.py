"""AdamW and gradient norm: refusals, the 8-bit codec and host-side checks; no GPU needed."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as O
from src.gcn.hip import fused_adamw as A
from src.gcn.hip import lib as L


def _args(n=5, dtype=torch.float32, **k):
    p = torch.ones(n, dtype=dtype)
    return [[p], [p.clone()], [torch.zeros(n)], [torch.zeros(n)]], dict(step=1, lr=1e-3, **k)


def test_cpu_tensors_are_refused():
    lists, k = _args()
    with pytest.raises(L.GcnHipError, match="no CPU fallback"):
        A.adamw_step_(*lists, **k)
    with pytest.raises(L.GcnHipError, match="no CPU fallback"):
        A.grad_norm(lists[1])
    with pytest.raises(L.GcnHipError):
        A.adamw_advance_(torch.zeros((), dtype=torch.int64), torch.zeros(64, dtype=torch.uint8), lr=1e-3)


@pytest.mark.parametrize("change, error", [
    (lambda a, k: k.update(step=0), ValueError),
    (lambda a, k: k.update(step=1.5), ValueError),
    (lambda a, k: a[1].append(torch.ones(5)), ValueError),
    (lambda a, k: a.__setitem__(1, [torch.ones(4)]), ValueError),
    (lambda a, k: a.__setitem__(1, [torch.ones(5, dtype=torch.bfloat16)]), TypeError),
    (lambda a, k: a.__setitem__(2, [torch.zeros(5, dtype=torch.float64)]), TypeError),
    (lambda a, k: a.__setitem__(2, [torch.zeros(10)[::2]]), ValueError),
    (lambda a, k: a.__setitem__(0, [torch.ones(5, dtype=torch.float64)]), TypeError),
    (lambda a, k: k.update(masters=[torch.ones(5)]), ValueError),
    (lambda a, k: k.update(exp_avg_exps=[torch.zeros(1, dtype=torch.uint8)]), ValueError),
    (lambda a, k: k.update(exp_avg_exps=[torch.zeros(1, dtype=torch.uint8)], exp_avg_sq_exps=[torch.zeros(1, dtype=torch.uint8)]), TypeError),
])
def test_bad_arguments_are_refused(change, error):
    lists, k = _args()
    change(lists, k)
    with pytest.raises(error):
        A.adamw_step_(*lists, **k)


def test_16_bit_parameters_need_masters():
    p = [torch.ones(5, dtype=torch.bfloat16)]
    with pytest.raises(ValueError, match="master"):
        A.adamw_step_(p, p, [torch.zeros(5)], [torch.zeros(5)], step=1, lr=1e-3)


def test_8_bit_states_need_as_many_exponents_as_blocks():
    p = [torch.ones(129)]
    code = lambda: [torch.zeros(129, dtype=torch.uint8)]
    with pytest.raises(ValueError, match="sizes"):
        A.adamw_step_(p, p, code(), code(), step=1, lr=1e-3, exp_avg_exps=[torch.zeros(1, dtype=torch.uint8)],
                      exp_avg_sq_exps=[torch.zeros(2, dtype=torch.uint8)])


def test_norm_refusals():
    with pytest.raises(TypeError):
        A.grad_norm([])
    with pytest.raises(TypeError):
        A.grad_norm([torch.ones(2), torch.ones(2, dtype=torch.bfloat16)])
    with pytest.raises(ValueError):
        A.grad_norm([torch.ones(2)], max_norm=-1.0)
    with pytest.raises(ValueError):
        A.grad_norm([torch.ones(4)[::2]])


def test_optimizer_argument_checks():
    p = [torch.nn.Parameter(torch.ones(3))]
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(weight_decay=-1.0),
                dict(state_bits=16), dict(max_grad_norm=-1.0), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            A.FusedAdamW(p, **bad)
    p[0].grad = torch.ones(3)
    with pytest.raises(L.GcnHipError):
        A.FusedAdamW(p).step()


def test_c_entry_points_refuse_without_touching_memory():
    lib = L.load()
    d = L.AdamWDesc(n=1, param_type=0, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
    one = (ctypes.c_void_p * 1)(16)
    null = (ctypes.c_void_p * 1)(None)
    odd = (ctypes.c_void_p * 1)(18)
    size = (ctypes.c_longlong * 1)(4)

    def call(desc=d, p=one, g=one, mast=None, m=one, v=one, em=None, ev=None, n=size):
        return lib.gcn_adamw_step(None if desc is None else ctypes.byref(desc), p, g, mast, m, v, em, ev, n, None, None, None, None)

    assert call(desc=None) < 0 and call(p=None) < 0 and call(p=null) < 0 and call(g=odd) < 0 and call(n=(ctypes.c_longlong * 1)(-1)) < 0
    assert call(mast=one) < 0 and b"master" in lib.gcn_last_error()
    assert call(em=one, ev=one) < 0 and b"8-bit" in lib.gcn_last_error()
    for field, bad in (("step", 0), ("n", -1), ("param_type", 3), ("state_bits", 16), ("lr", -1.0), ("beta1", 1.0), ("beta2", float("nan"))):
        keep = getattr(d, field)
        setattr(d, field, bad)
        assert call() < 0, field
        setattr(d, field, keep)
    d.n = 0
    assert call(p=None, g=None, m=None, v=None, n=None) == 0           # nothing to do
    assert lib.gcn_adamw_advance(ctypes.byref(d), None, None, None, None) < 0
    assert lib.gcn_grad_norm_ws_bytes(1, size) == 8 and lib.gcn_grad_norm_ws_bytes(-1, size) == 0
    assert lib.gcn_grad_norm(1, 0, one, size, None, 1.0, None, one, 8, None) < 0
    assert lib.gcn_grad_norm(1, 5, one, size, None, 1.0, one, one, 8, None) < 0
    assert lib.gcn_grad_norm(1, 0, null, size, None, 1.0, one, one, 8, None) < 0
    assert lib.gcn_grad_norm(1, 0, one, size, None, 1.0, one, one, 4, None) < 0 and b"workspace" in lib.gcn_last_error()
    assert lib.gcn_grad_norm(1, 0, one, size, None, float("nan"), one, one, 8, None) < 0


def test_state8_codec_against_the_definition():
    rng = np.random.default_rng(3)
    for n in (1, 127, 128, 129, 1000):
        x = (rng.standard_normal(n) * np.exp2(rng.uniform(-12, 2, n))).astype(np.float32)
        x[rng.random(n) < 0.1] = 0
        codes, exps = A.state8_encode(torch.from_numpy(x))
        assert codes.dtype == exps.dtype == torch.uint8 and exps.numel() == -(-n // 128)
        back = A.state8_decode(codes, exps).numpy()
        np.testing.assert_array_equal(back, O.decode(codes.numpy(), exps.numpy()).astype(np.float32))
        # nearest: off by half a step, 2^-4 of the value, or half of 2^-9 of the block's scale
        scale = np.repeat(np.exp2(exps.numpy().astype(np.float64) - 127), 128)[:n]
        assert (np.abs(back - x) <= np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** -10 * scale)).all()
    tiny = torch.tensor([1.0, 1e-12, 0.0])
    codes, exps = A.state8_encode(tiny, never_zero=True)
    assert codes.tolist()[1:] == [1, 0]
    codes, exps = A.state8_encode(torch.zeros(5))
    assert not codes.any() and A.state8_decode(codes, exps).eq(0).all()


def test_oracle_hash_and_rounding_are_unbiased():
    n = 1 << 16
    r = O.random32(n, 7, 3, 2)
    assert abs((r & 0xFFFF).mean() / 65536 - 0.5) < 5 * 0.29 / 256 and abs((r >> 16).mean() / 65536 - 0.5) < 5 * 0.29 / 256
    x = np.full(n, 1.03)
    value, exps, _, step = O.encode(x, (r & 0xFFFF).astype(np.int64), False)
    assert set(np.unique(value)) == {1.0, 1.125} and (exps == 120).all()
    assert abs(value.mean() - 1.03) < 5 * step[0] * 0.5 / 256


@pytest.mark.parametrize("seed", [-1, 1 << 64])
def test_seeds_have_64_bits(seed):
    with pytest.raises(ValueError, match="seed"):
        A.FusedAdamW([torch.nn.Parameter(torch.ones(3))], seed=seed)


@pytest.mark.parametrize("source, change", [
    (torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.AdamW, dict(maximize=True)), (torch.optim.AdamW, dict(differentiable=True)),
    (torch.optim.Adam, dict(weight_decay=0.1)), (torch.optim.AdamW, "max_exp_avg_sq"), (torch.optim.AdamW, "step"), (torch.optim.AdamW, "size"),
    (torch.optim.AdamW, "groups")])
def test_checkpoints_of_another_update_are_refused(source, change):
    """Each of them changes what a step does; nothing of a refused checkpoint is loaded."""
    theirs = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(4))]
    opt = source(theirs, lr=0.5, foreach=False, **(change if isinstance(change, dict) else {}))
    for p in theirs:
        p.grad = torch.ones_like(p)
    if change != dict(differentiable=True):
        opt.step()
    saved = opt.state_dict()
    if change == "max_exp_avg_sq":
        saved["state"][1]["max_exp_avg_sq"] = torch.ones(4)
    elif change == "step":
        del saved["state"][1]["step"]
    elif change == "size":
        saved["state"][1]["exp_avg"] = torch.ones(5)
    elif change == "groups":
        saved["param_groups"][0]["params"] = [0]
    ours = A.FusedAdamW([torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(4))], lr=1e-3)
    with pytest.raises(ValueError):
        ours.load_state_dict(saved)
    assert not ours.state and ours.param_groups[0]["lr"] == 1e-3 and "maximize" not in ours.param_groups[0]


def test_groups_with_options_of_another_update_are_refused():
    p = lambda: torch.nn.Parameter(torch.ones(3))
    for name in ("amsgrad", "maximize", "differentiable"):
        with pytest.raises(ValueError, match=name):
            A.FusedAdamW([{"params": [p()], name: True}])
        opt = A.FusedAdamW([{"params": [p()], name: False}])
        with pytest.raises(ValueError, match=name):
            opt.add_param_group({"params": [p()], name: True})
        assert len(opt.param_groups) == 1


@pytest.mark.parametrize("source", [torch.optim.AdamW, torch.optim.Adam])
def test_checkpoints_of_the_same_update_are_taken(source):
    theirs = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(4))]
    opt = source(theirs, lr=0.5, foreach=False)
    for p in theirs:
        p.grad = torch.full_like(p, 2.0)
    opt.step()
    mine = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(4))]
    ours = A.FusedAdamW(mine)
    ours.load_state_dict(opt.state_dict())
    assert ours.param_groups[0]["lr"] == 0.5 and ours.param_groups[0]["decoupled_weight_decay"] is True
    for p, q in zip(mine, theirs):
        assert torch.equal(ours.state[p]["exp_avg"], opt.state[q]["exp_avg"]) and float(ours.state[p]["step"]) == 1
    assert ours.state[mine[0]]["step"] is ours.state[mine[1]]["step"]


def test_fused_adam_refuses_8_bit_moments():
    """Their codes are not moments; by way of a 32-bit FusedAdamW they are taken."""
    from src.gcn.hip.fused_adam import FusedAdam
    mine = [torch.nn.Parameter(torch.ones(300))]
    narrow = A.FusedAdamW(mine, state_bits=8, min_8bit_numel=1, weight_decay=0.0)
    moments = torch.linspace(-1, 1, 300)
    st = {"step": torch.tensor(1.0)}
    for key, x in (("exp_avg", moments), ("exp_avg_sq", moments.abs())):
        st[key], st[key + "_exp"] = A.state8_encode(x, never_zero=key == "exp_avg_sq")
    narrow.state[mine[0]] = st
    other = [torch.nn.Parameter(torch.ones(300))]
    adam = FusedAdam(other)
    with pytest.raises(ValueError, match="8 bits"):
        adam.load_state_dict(narrow.state_dict())
    assert not adam.state
    wide = A.FusedAdamW([torch.nn.Parameter(torch.ones(300))], weight_decay=0.0)
    wide.load_state_dict(narrow.state_dict())
    adam.load_state_dict(wide.state_dict())
    # nearest code: off by half a step, 2^-4 of the value, or half of 2^-9 of the block's scale (the largest value is 1: 2^-7)
    assert bool(((adam.state[other[0]]["exp_avg"] - moments).abs() <= (moments.abs() * 2.0 ** -4).clamp(min=2.0 ** -17)).all())
