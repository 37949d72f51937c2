"""Rules on logits: refusals and host-side checks; no GPU needed."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import logits_oracle as O
from src.gcn.hip import lib as L
from src.gcn.hip.logits import pack_mask, process_logits

X = torch.zeros(2, 3, 10)


def test_cpu_tensors_are_refused():
    with pytest.raises(L.GcnHipError, match="no CPU fallback"):
        process_logits(X)


@pytest.mark.parametrize("kind, error", [
    (dict(dim=3), ValueError),
    (dict(history=torch.zeros(2, 3, 4)), TypeError),
    (dict(history=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(history=torch.zeros(3, 2, 4, dtype=torch.int64)), ValueError),
    (dict(history=torch.zeros(2, 2, 3, 4, dtype=torch.int64)), ValueError),
    (dict(history_lens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(history=torch.zeros(3, 4, dtype=torch.int64), history_lens=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(history=torch.zeros(3, 4, dtype=torch.int64), history_lens=torch.zeros(3)), TypeError),
    (dict(history=torch.zeros(3, 4, dtype=torch.int64), history_lens=torch.zeros(3, dtype=torch.int64),
          prompt_lens=torch.zeros(3, dtype=torch.int32)), TypeError),
    (dict(repetition_penalty=0.0), ValueError), (dict(repetition_penalty=float("nan")), ValueError), (dict(temperature=0.0), ValueError),
    (dict(temperature=-1.0), ValueError), (dict(presence_penalty=float("inf")), ValueError),
    (dict(temperature=torch.ones(3, dtype=torch.float64)), TypeError), (dict(temperature=torch.ones(2)), ValueError),
    (dict(mask=torch.ones(3, 10)), TypeError), (dict(mask=torch.ones(3, 9, dtype=torch.bool)), ValueError),
    (dict(mask=torch.ones(3, 2, dtype=torch.int32)), ValueError), (dict(mask=torch.ones(2, 10, dtype=torch.bool)), ValueError),
    (dict(bias=torch.ones(10, dtype=torch.bfloat16)), TypeError), (dict(bias=torch.ones(11)), ValueError),
    (dict(bias=torch.ones(2, 10)), ValueError), (dict(out=torch.zeros(2, 3, 9)), ValueError),
    (dict(out=torch.zeros(2, 3, 20)[:, :, ::2]), ValueError), (dict(out=torch.zeros(10).expand(2, 3, 10)), ValueError),
    (dict(out=torch.zeros(2, 3, 10, dtype=torch.float16)), ValueError),
])
def test_bad_arguments_are_refused(kind, error):
    with pytest.raises(error):
        process_logits(X, **kind)


def test_other_refusals():
    with pytest.raises(TypeError):
        process_logits(X.double())
    with pytest.raises(ValueError):
        process_logits(torch.zeros(()))
    with pytest.raises(ValueError, match="gradients"):
        process_logits(X.clone().requires_grad_(), out=torch.zeros(2, 3, 10))


def test_pack_mask():
    gen = torch.Generator().manual_seed(0)
    for v in (1, 31, 32, 33, 100):
        m = torch.rand(3, v, generator=gen) < 0.5
        w = pack_mask(m)
        assert w.shape == (3, -(-v // 32)) and w.dtype == torch.int32
        bits = np.unpackbits(w.numpy().view(np.uint8), axis=1, bitorder="little")[:, :v]
        assert np.array_equal(bits.astype(bool), m.numpy())
    with pytest.raises(TypeError):
        pack_mask(torch.ones(3))


def test_row_stride():
    stride = L.binding().row_stride
    x = torch.zeros(4, 6, 10)
    assert stride(x, 2) == 10 and stride(x, 1) == 60 and stride(x, 0) == 240
    assert stride(x[:, :, :7], 2) == 10 and stride(x[:, :, ::2], 2) == -1
    assert stride(x[:, :3], 2) == -1                              # rows not evenly spaced
    assert stride(x[:1, :3], 2) == 10 and stride(x[:, :1], 2) == 60
    assert stride(torch.zeros(10).expand(4, 10), 1) == 0
    assert stride(x.transpose(0, 1), 2) == -1


def test_c_entry_points_refuse_without_touching_memory():
    lib = L.load()
    ok = dict(rows=4, vocab=8, inner=1, in_stride=8, out_stride=8, history_rows=1, bias_rows=1, mask_rows=1, repetition_rows=1, presence_rows=1,
              frequency_rows=1, temperature_rows=1, type=0, repetition=1.0, temperature=1.0)

    def call(**k):
        d = L.LogitsDesc(**{**ok, **k})
        return lib.gcn_logits_process(ctypes.byref(d), None, None, None)

    assert call() == -1 and b"null pointer" in lib.gcn_last_error()
    assert lib.gcn_logits_process(None, None, None, None) == -1
    assert call(rows=0) == 0
    for bad in (dict(type=3), dict(vocab=0), dict(inner=0), dict(rows=-1), dict(out_stride=7), dict(in_stride=-1), dict(mask_type=1),
                dict(mask_type=3, mask=16), dict(mask=16), dict(repetition=0.0), dict(temperature=float("nan")), dict(history_lens=16),
                dict(history=16, history_len=-1), dict(history=16, history_len=5, history_rows=3), dict(bias=16, bias_rows=3),
                dict(mask=16, mask_type=2, mask_rows=5), dict(temperature_t=16, temperature_rows=0)):
        assert call(**bad) == -1, bad
        assert b"null pointer" not in lib.gcn_last_error(), bad
    for big in (dict(vocab=1 << 31, out_stride=1 << 31), dict(vocab=1 << 20, inner=1 << 11, out_stride=1 << 31), dict(rows=1 << 31)):
        assert call(**big) == -2, big
    d = L.LogitsDesc(**ok)
    assert lib.gcn_logits_process_bwd(ctypes.byref(d), None, None, None, 16, None, 0, None) == -1 and b"bias" in lib.gcn_last_error()
    assert lib.gcn_logits_process_bwd(ctypes.byref(d), 16, 16, None, None, None, 0, None) == -1


def test_oracle_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, b = rng.standard_normal((4, 6, 3)), rng.standard_normal((2, 6))
    hist = rng.integers(-1, 7, (2, 5))
    mask = rng.random((4, 6)) < 0.7
    kind = dict(history=hist, prompts=[1, 0], rho=1.3, alpha_p=0.2, alpha_f=0.1, mask=mask, tau=np.array([0.5, 2.0]), masked=-3.0)
    dy = rng.standard_normal(x.shape)
    _, slope, slope_b, _ = O.process(x, bias=b, **kind)
    dx, db, _ = O.gradient(dy, slope, slope_b, 2)
    f = lambda x, b: float((O.process(x, bias=b, **kind)[0] * dy).sum())
    for grad, arr, at in ((dx, x, 0), (db, b, 1)):
        for k in np.ndindex(arr.shape):
            step = np.zeros_like(arr)
            step[k] = 1e-6
            args = [(x + step, b), (x - step, b)] if at == 0 else [(x, b + step), (x, b - step)]
            assert abs((f(*args[0]) - f(*args[1])) / 2e-6 - grad[k]) < 1e-6


def test_workspace_of_the_bias_gradient():
    lib = L.load()
    ok = dict(vocab=1000, inner=1, in_stride=1000, out_stride=1000, history_rows=1, mask_rows=1, repetition_rows=1, presence_rows=1,
              frequency_rows=1, temperature_rows=1, type=0, repetition=1.0, temperature=1.0)
    ws = lambda **k: lib.gcn_logits_bwd_ws_bytes(ctypes.byref(L.LogitsDesc(**{**ok, **k})))
    assert ws(rows=8) == 0                                         # no bias
    assert ws(rows=8, bias=16, bias_rows=8) == 0                   # a row of its own for each: nothing to add
    shared = ws(rows=2000, bias=16, bias_rows=1)
    assert shared > 0 and shared % 4000 == 0                       # whole rows of sums
    assert ws(rows=2, vocab=4, inner=100000, out_stride=400000, bias=16, bias_rows=1) == 0
    d = L.LogitsDesc(**{**ok, "rows": 2000, "bias": 16, "bias_rows": 1})
    assert lib.gcn_logits_process_bwd(ctypes.byref(d), 16, 16, 16, 16, None, 0, None) == -2 and b"workspace" in lib.gcn_last_error()


def test_rows_near_the_end_of_32_bits_are_refused():
    """The backward kernels count rows in turns of 32: a count that starts below 2^31 must not pass it."""
    lib = L.load()
    one = dict(vocab=1, inner=1, in_stride=1, out_stride=1, type=2, repetition=1.0, temperature=1.0)
    for rows, rc in (((1 << 31) - 1, -2), ((1 << 31) - 32, -2), ((1 << 31) - 4096, -2), ((1 << 31) - 4097, -1)):     # -1: the null pointers
        d = L.LogitsDesc(rows=rows, **one)
        assert lib.gcn_logits_process(ctypes.byref(d), None, None, None) == rc, rows
        assert lib.gcn_logits_process_bwd(ctypes.byref(d), None, None, None, None, None, 0, None) == rc, rows


@pytest.mark.parametrize("name", ["repetition_penalty", "presence_penalty", "frequency_penalty", "temperature"])
def test_numbers_that_are_not_finite_in_float32_are_refused(name):
    """1e39 is a finite double and an infinite float; the reciprocal of 1e-39 is infinite, and makes NaN of a logit of 0."""
    for value in (1e39, -1e39) + ((1e-39,) if name in ("repetition_penalty", "temperature") else ()):
        with pytest.raises(ValueError):
            process_logits(X, **{name: value})
    with pytest.raises(L.GcnHipError, match="no CPU fallback"):              # allowed
        process_logits(X, **{name: 1e-37})


def test_c_entry_points_refuse_numbers_that_are_not_finite():
    lib = L.load()
    ok = dict(rows=4, vocab=8, inner=1, in_stride=8, out_stride=8, repetition=1.0, temperature=1.0)
    for bad in (dict(repetition=math.inf), dict(repetition=1e-39), dict(temperature=math.inf), dict(temperature=1e-39), dict(presence=math.nan),
                dict(presence=math.inf), dict(frequency=-math.inf)):
        d = L.LogitsDesc(**{**ok, **bad})
        assert lib.gcn_logits_process(ctypes.byref(d), None, None, None) == -1 and b"null pointer" not in lib.gcn_last_error(), bad


@pytest.mark.parametrize("lead, rows, fits", [
    ((6,), (6,), True), ((6,), (3,), True), ((6,), (2,), True), ((6,), (1,), True), ((6,), (4,), False), ((6,), (12,), False), ((6,), (0,), False),
    ((4, 3), (4, 3), True), ((4, 3), (3,), True), ((4, 3), (2, 3), True), ((4, 3), (1, 3), True), ((4, 3), (4, 1), False), ((4, 3), (3, 3), False),
    ((4, 6), (3,), True), ((4, 6), (2, 3), False), ((4, 6), (4,), False), ((6,), (1, 3), True), ((), (2,), False), ((), (1,), True)])
def test_rows_of_an_argument(lead, rows, fits):
    """All leading dimensions, the last few, one row, or a divisor at the outermost; what fits is refused for being on the CPU."""
    x = torch.zeros(*lead, 10)
    for kind in (dict(bias=torch.zeros(*rows, 10)), dict(mask=torch.ones(*rows, 10, dtype=torch.bool)), dict(temperature=torch.ones(*rows)),
                 dict(history=torch.zeros(*rows, 4, dtype=torch.int64))):
        with pytest.raises(L.GcnHipError if fits else ValueError, match="no CPU fallback" if fits else "leading dimensions"):
            process_logits(x, **kind)


def test_a_saved_tensor_comes_back_as_what_it_was():
    """Hooks on saved tensors may change strides and addresses, and nothing else."""
    same = L.binding().check_saved
    x = torch.zeros(3, 10, dtype=torch.bfloat16)
    for now in (x, x.clone(), torch.zeros(10, 3, dtype=torch.bfloat16).t(), torch.zeros(3, 16, dtype=torch.bfloat16)[:, :10]):
        same(x, now)
    for now in (x.float(), x.half(), x[:2], x[:, :9], x.view(30), x.view(1, 3, 10), x.to("meta"), x.to_sparse()):
        with pytest.raises(RuntimeError, match="was saved as"):
            same(x, now)


@pytest.mark.parametrize("name", ["logits", "bias", "out"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    """No forward-mode derivative: with a tangent the result would be a constant without a word."""
    import torch.autograd.forward_ad as fwAD
    given = dict(logits=torch.zeros(3, 10), bias=torch.zeros(10), out=torch.zeros(3, 10))
    if name != "out":
        del given["out"]
    with fwAD.dual_level():
        given[name] = fwAD.make_dual(given[name].requires_grad_(grad and name != "out"), torch.ones_like(given[name]))
        with pytest.raises(L.GcnHipError, match=f"{name} carries a tangent"):
            process_logits(given.pop("logits"), **given)


def test_rows_that_meet_against_the_elements_they_hold():
    """Views [rows, n] of one buffer, their rows dense: they meet if they share an element."""
    meet = L.binding().rows_meet
    base = torch.zeros(60)
    views = [base.as_strided((rows, n), (step, 1), at) for rows in (1, 2, 4) for n in (1, 3, 7) for step in (n, n + 1, 9, 12) if step >= n
             for at in (0, 1, 5, 8, 13) if at + (rows - 1) * step + n <= 60]
    shared = [base.as_strided((3, 4), (0, 1), at) for at in (0, 6, 30)]           # expanded: read, never written
    cells = lambda v: {v.storage_offset() + i * v.stride(0) + j for i in range(v.shape[0]) for j in range(v.shape[1])}
    met = 0
    for a in views:
        for b in views + shared:
            want = bool(cells(a) & cells(b))
            assert meet(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
            met += want
    assert 0 < met < len(views) * len(views)
