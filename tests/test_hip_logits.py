"""Rules on logits and their gradient on the GPU against the formulas in double precision.

Tolerances count roundings, u = 2^-24 each, and half a step (finfo.eps / 2) of the logits' type for the result:
  y: |err| <= 8 u (|x1| + n |alpha_f| + |alpha_p| + |bias|) / tau + eps / 2 |y|       1/rho, product, penalty (2), sums (2), 1/tau, product
  dx: |err| <= 4 u |dx| + eps / 2 |dx|
  dbias: sums of N terms of 2 roundings each, in any order: |err| <= (N + 2) u sum |terms|
fp16 adds its smallest subnormal step's half, 2^-25."""
import math

import numpy as np
import pytest
import torch

from oracle import logits_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


def case(dev, rows, vocab, inner=1, length=20, dtype=torch.float32, seed=0, mask="bits", bias_rows=1, per_row=True, wide=True, hist_rows=None):
    """Arguments of process_logits for logits [rows, vocab(, inner)], and those of the oracle."""
    from src.gcn.hip.logits import pack_mask
    rng = np.random.default_rng(seed)
    hist_rows = rows if hist_rows is None else hist_rows
    x = torch.from_numpy(3 * rng.standard_normal((rows, vocab, inner)).astype(np.float32)).to(dtype)
    ints = torch.int64 if wide else torch.int32
    few = rng.integers(-2, vocab + 2, max(1, length // 3) + 1)                   # entries that occur often, some of them invalid
    hist = torch.from_numpy(np.where(rng.random((hist_rows, length)) < 0.5, rng.choice(few, (hist_rows, length)),
                                     rng.integers(0, vocab, (hist_rows, length)))).to(ints)
    lens = torch.from_numpy(rng.integers(-1, length + 2, hist_rows)).to(ints)
    prompts = torch.from_numpy(rng.integers(0, length // 2 + 1, hist_rows)).to(ints)
    number = lambda lo, hi: torch.from_numpy(rng.uniform(lo, hi, rows).astype(np.float32)) if per_row else round(float(rng.uniform(lo, hi)), 3)
    rho, ap, af, tau = number(0.7, 1.6), number(-0.5, 1.0), number(-0.2, 0.5), number(0.4, 2.0)
    bias = torch.from_numpy(rng.standard_normal((bias_rows, vocab)).astype(np.float32)) if bias_rows else None
    allowed = None
    if mask:
        allowed = rng.random((rows, vocab)) < rng.random((rows, 1))
        allowed[rows // 2] = False                                               # a row with nothing left
        allowed = torch.from_numpy(allowed)
    # rows shared by several leading positions: those of the last leading dimension
    period = next((n for n in (bias_rows, hist_rows) if n not in (0, 1, rows)), None)
    lead = (rows,) if period is None else (rows // period, period)
    rows_of = lambda t: t.view(*(lead if t.shape[0] == rows and rows > 1 else t.shape[:1]), *t.shape[1:])
    put = lambda t: rows_of(t).to(dev) if isinstance(t, torch.Tensor) else t
    kind = dict(dim=len(lead), history=put(hist), history_lens=put(lens), prompt_lens=put(prompts), repetition_penalty=put(rho), presence_penalty=put(ap),
                frequency_penalty=put(af), temperature=put(tau), bias=put(bias),
                mask=None if allowed is None else put(pack_mask(allowed) if mask == "bits" else allowed))
    np64 = lambda t: t.double().numpy() if isinstance(t, torch.Tensor) else t
    want = dict(history=hist.numpy(), lens=lens.numpy(), prompts=prompts.numpy(), rho=np64(rho), alpha_p=np64(ap), alpha_f=np64(af), tau=np64(tau),
                bias=None if bias is None else bias.numpy(), mask=None if allowed is None else allowed.numpy())
    return x.to(dev).view((*lead, vocab) if inner == 1 else (*lead, vocab, inner)), kind, want


def host(t, shape=None):
    a = t.detach().double().cpu().numpy()
    return a if shape is None else a.reshape(shape)


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def near(got, want, tol, masked=None):
    finite = np.isfinite(want)
    assert np.array_equal(finite, np.isfinite(got)) and np.array_equal(got[~finite], want[~finite], equal_nan=True)
    off = np.abs(got[finite] - want[finite]) - tol[finite]
    assert (off <= 0).all(), float(off.max())


def check(x, kind, want, masked=-math.inf, out=None, got=None):
    from src.gcn.hip.logits import process_logits
    y = process_logits(x, masked_value=masked, out=out, **kind) if got is None else got
    assert y.shape == x.shape and y.dtype == x.dtype
    rows, vocab = math.prod(x.shape[:kind["dim"]]), x.shape[kind["dim"]]
    ref, _, _, bound = O.process(host(x, (rows, vocab, -1)), masked=float(torch.tensor(masked, dtype=torch.float32).to(x.dtype)), **want)
    near(host(y, ref.shape), ref, 8 * U * bound + half_step(x.dtype) * np.abs(np.nan_to_num(ref, neginf=0.0)) + 2.0 ** -25 * (x.dtype == torch.float16))
    return y


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [1, 7, 8, 31, 33, 2047, 2048, 2049, 5000])
def test_rows_match_the_formula(dev, dtype, vocab):
    for rows, length, mask, bias_rows, per_row, wide in ((1, 1, "bits", 1, True, True), (6, 40, "bits", 6, True, False), (6, 300, "bool", 3, False, True),
                                                         (4, 17, None, 0, True, True)):
        check(*case(dev, rows, vocab, length=length, dtype=dtype, seed=vocab, mask=mask, bias_rows=bias_rows, per_row=per_row, wide=wide))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab, inner", [(1, 1), (1, 5), (14, 10), (33, 3), (200, 7), (9, 513), (2500, 2)])
def test_inner_dimensions(dev, dtype, vocab, inner):
    for mask, bias_rows, hist_rows in (("bool", 3, 3), ("bits", 6, 6), (None, 1, 1)):
        check(*case(dev, 6, vocab, inner, length=25, dtype=dtype, seed=inner, mask=mask, bias_rows=bias_rows, per_row=False, hist_rows=hist_rows),
              masked=-1e4)


@pytest.mark.parametrize("rows, vocab, length", [(1, 100000, 3000), (3, 50021, 40000), (700, 3000, 64), (2, 131072, 1)])
def test_long_rows_and_long_histories(dev, rows, vocab, length):
    x, kind, want = case(dev, rows, vocab, length=length, dtype=torch.bfloat16, seed=3, mask="bits")
    check(x, kind, want)


def test_lengths_of_zero(dev):
    from src.gcn.hip.logits import process_logits
    x, kind, want = case(dev, 4, 100, length=9, seed=2)
    empty = {**kind, "history": kind["history"][:, :0], "history_lens": None, "prompt_lens": None}
    check(x, empty, {**want, "history": None})
    none = {**kind, "history_lens": torch.zeros_like(kind["history_lens"])}
    check(x, none, {**want, "lens": np.zeros(4)})
    long_prompt = {**kind, "prompt_lens": torch.full_like(kind["prompt_lens"], 100)}
    check(x, long_prompt, {**want, "prompts": np.full(4, 100)})
    assert process_logits(x[:0], dim=1).shape == (0, 100)
    assert torch.equal(process_logits(x), x)
    with pytest.raises(ValueError, match="is on cpu"):
        process_logits(x, history=kind["history"].cpu())


def test_strided_rows_views_and_in_place(dev):
    from src.gcn.hip.logits import process_logits
    for dtype in TYPES:
        x, kind, want = case(dev, 5, 1001, length=30, dtype=dtype, seed=5)
        big = torch.full((5, 1100), 9.0, dtype=dtype, device=dev)
        big[:, 3:1004] = x
        view = big[:, 3:1004]
        ref = check(view, kind, want)
        assert torch.equal(ref, check(x, kind, want))
        out = torch.full((5, 1003), 5.0, dtype=dtype, device=dev)
        check(view, kind, want, out=out[:, 1:1002])
        assert torch.equal(out[:, 1:1002], ref) and bool((out[:, 0] == 5).all()) and bool((out[:, 1002] == 5).all())
        got = process_logits(view, out=view, masked_value=-math.inf, **kind)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, ref)
        assert bool((big[:, :3] == 9).all()) and bool((big[:, 1004:] == 9).all())
        steps = x.repeat_interleave(2, 1)[:, ::2]                     # every second element
        assert torch.equal(process_logits(steps, **kind), ref)
        cols = x.t().contiguous().t()
        assert torch.equal(process_logits(cols, **kind), ref)
        same = x[:1].expand(5, -1)
        check(same, kind, want)
        three = torch.stack([x, x]).transpose(0, 1)                   # [5, 2, V], the rows not evenly spaced
        lead = {**{k: v for k, v in kind.items() if k in ("temperature", "bias")}, "dim": 2}
        lead["temperature"] = kind["temperature"].view(5, 1).expand(5, 2)
        assert torch.equal(process_logits(three, **lead)[:, 0], process_logits(x, dim=1, temperature=kind["temperature"], bias=kind["bias"]))


def test_leading_dimensions_and_shared_rows(dev):
    """[B, V, V, C] scores: history, bias and mask of all graphs, of every graph, of one node; all equal their expanded forms."""
    from src.gcn.hip.logits import process_logits
    gen = torch.Generator(dev).manual_seed(0)
    y = torch.randn(3, 5, 7, 2, device=dev, generator=gen)
    hist = torch.randint(-1, 7, (5, 4), device=dev, generator=gen)
    bias, mask = torch.randn(5, 7, device=dev, generator=gen), torch.rand(5, 7, device=dev, generator=gen) < 0.6
    got = process_logits(y, dim=2, history=hist, bias=bias, mask=mask, repetition_penalty=1.5, frequency_penalty=0.3, masked_value=-1e9)
    want = process_logits(y.reshape(15, 7, 2), dim=1, history=hist.repeat(3, 1), bias=bias.repeat(3, 1), mask=mask.repeat(3, 1), repetition_penalty=1.5,
                          frequency_penalty=0.3, masked_value=-1e9).view(y.shape)
    assert torch.equal(got, want)
    one = process_logits(y, dim=-2, history=hist[:1], bias=bias[0], mask=mask[:1], masked_value=-1e9)
    two = process_logits(y, dim=2, history=hist[:1].expand(3, 5, 4), bias=bias[0].expand(3, 5, 7), mask=mask[0].expand(3, 5, 7), masked_value=-1e9)
    assert torch.equal(one, two)


def test_bad_values_in_masked_places_and_outside(dev):
    from src.gcn.hip.logits import process_logits
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 1.0, -2.0, float("nan"), -float("inf"), 3.0]], device=dev)
    on = torch.tensor([[0, 0, 0, 1, 1, 1, 1, 1]], device=dev, dtype=torch.bool)
    hist = torch.tensor([[0, 3, 4, 4, 6]], device=dev)
    for dtype in TYPES:
        for masked in (-math.inf, float(torch.finfo(dtype).min), 0.0):
            y = process_logits(x.to(dtype), history=hist, repetition_penalty=2.0, frequency_penalty=0.5, mask=on, masked_value=masked)
            want = [masked] * 3 + [0.0, -5.0, float("nan"), -math.inf, 3.0]
            assert np.array_equal(host(y)[0], np.array(want), equal_nan=True)
    z = x.clone().requires_grad_()
    bias = torch.zeros(8, device=dev, requires_grad=True)
    y = process_logits(z, history=hist, repetition_penalty=2.0, bias=bias, mask=on)
    dy = torch.tensor([[float("nan"), float("inf"), 1.0, 1.0, 1.0, 1.0, 1.0, 1.0]], device=dev)
    dx, db = torch.autograd.grad(y, [z, bias], dy)
    assert host(dx)[0].tolist() == [0, 0, 0, 0.5, 2, 1, 2, 1] and host(db).tolist() == [0, 0, 0, 1, 1, 1, 1, 1]


def grads(x, kind, want, bias_rows, dy, masked=-1e4):
    from src.gcn.hip.logits import process_logits
    z, b = x.detach().requires_grad_(), None if kind["bias"] is None else kind["bias"].clone().requires_grad_()
    y = process_logits(z, masked_value=masked, **{**kind, "bias": b})
    check(x, kind, want, masked=masked, got=y)
    got = torch.autograd.grad(y, [z] if b is None else [z, b], dy)
    rows, vocab = math.prod(x.shape[:kind["dim"]]), x.shape[kind["dim"]]
    shape = (rows, vocab, x.numel() // (rows * vocab))
    _, slope, slope_b, _ = O.process(host(x, shape), masked=masked, **want)
    dx, db, size = O.gradient(host(dy, shape), slope, slope_b, max(bias_rows, 1))
    eps = half_step(x.dtype)
    assert got[0].dtype == x.dtype and got[0].shape == x.shape
    assert (np.abs(host(got[0], shape) - dx) <= (4 * U + eps) * np.abs(dx) + 2.0 ** -25 * (x.dtype == torch.float16)).all()
    if b is not None:
        terms = shape[2] * rows // bias_rows
        assert got[1].dtype == torch.float32 and got[1].shape == kind["bias"].shape
        assert (np.abs(host(got[1]) - db) <= (terms + 2) * U * size + 1e-44).all()
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows, vocab, inner, bias_rows", [
    (1, 1, 1, 1), (6, 2049, 1, 1), (6, 33, 1, 3), (6, 100, 1, 6), (6, 100, 1, 0), (12, 14, 10, 4), (12, 14, 10, 12), (12, 14, 10, 1), (8, 200, 100, 4),
    (3, 5, 700, 3), (2, 9, 4097, 1), (300, 50, 1, 1), (513, 2500, 1, 1), (64, 17, 3, 2)])
def test_gradient_matches_the_formula(dev, dtype, rows, vocab, inner, bias_rows):
    for mask, per_row in (("bits", True), ("bool", False), (None, False)):
        x, kind, want = case(dev, rows, vocab, inner, length=20, dtype=dtype, seed=rows, mask=mask, bias_rows=bias_rows, per_row=per_row)
        dy = torch.randn(x.shape, device=dev, generator=torch.Generator(dev).manual_seed(1)).to(dtype)
        first = grads(x, kind, want, bias_rows, dy)
        again = grads(x, kind, want, bias_rows, dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))                  # the same bits every time


def test_gradient_with_strides_and_broadcasts(dev):
    from src.gcn.hip.logits import process_logits
    x, kind, want = case(dev, 6, 40, 3, seed=4, bias_rows=2, per_row=False)          # logits [3, 2, 40, 3]
    dy = torch.randn(3, 2, 40, 3, device=dev)
    base = grads(x, kind, want, 2, dy)
    part = torch.zeros(3, 2, 50, 3, device=dev)
    part[:, :, 2:42] = x
    assert all(torch.equal(a, b) for a, b in zip(base, grads(part[:, :, 2:42], kind, want, 2, dy)))
    assert all(torch.equal(a, b) for a, b in zip(base, grads(x, kind, want, 2, dy.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0))))
    one = torch.ones((), device=dev).expand(3, 2, 40, 3)                             # what sum().backward() passes
    grads(x, kind, want, 2, one)
    # an expanded bias and expanded logits: autograd adds over the expansion
    b = torch.randn(40, device=dev, requires_grad=True)
    z = x[:1, :1].clone().requires_grad_()
    y = process_logits(z.expand(3, 2, 40, 3), **{**kind, "bias": b.expand(2, 40)}, masked_value=0.0)
    dz, db = torch.autograd.grad(y, [z, b], dy)
    z2, b2 = x[:1, :1].repeat(3, 2, 1, 1).requires_grad_(), b.detach().requires_grad_()
    y2 = process_logits(z2, **{**kind, "bias": b2}, masked_value=0.0)
    dz2, db2 = torch.autograd.grad(y2, [z2, b2], dy)
    # sums of at most 18 terms, in two orders
    assert float((dz - dz2.sum((0, 1), keepdim=True)).abs().max()) <= 2 * 18 * U * float(dz2.abs().sum((0, 1)).max())
    assert float((db - db2).abs().max()) <= 2 * 18 * U * 18 * float(dz2.abs().max() + dy.abs().max())
    # only one of the two
    y = process_logits(x, **{**kind, "bias": b2}, masked_value=0.0)
    (only,) = torch.autograd.grad(y, [b2], dy)
    z = x.detach().requires_grad_()
    _, both = torch.autograd.grad(process_logits(z, **{**kind, "bias": b2}, masked_value=0.0), [z, b2], dy)
    assert torch.equal(only, both)
    (only,) = torch.autograd.grad(process_logits(z, **kind, masked_value=0.0), [z], dy)
    assert torch.equal(only, torch.autograd.grad(process_logits(z, **{**kind, "bias": None}, masked_value=0.0), [z], dy)[0])


def test_changed_inputs_are_noticed_by_backward(dev):
    from src.gcn.hip.logits import process_logits
    x, kind, _ = case(dev, 3, 20, seed=1)
    z = x.detach().requires_grad_()
    y = process_logits(z, **kind)
    kind["history"].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = process_logits(z, **kind)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        (g,) = torch.autograd.grad(y.masked_fill(y.isinf(), 0).square().sum(), [z], create_graph=True)
        g.sum().backward()


def test_capture_forward_and_backward(dev):
    """Replays on new inputs, with eager work between them, against eager calls."""
    from src.gcn.hip.logits import process_logits
    x, kind, _ = case(dev, 16, 3000, length=50, dtype=torch.bfloat16, seed=6)
    dy = torch.randn(x.shape, device=dev).to(x.dtype)
    bias = kind.pop("bias")

    def both():
        z, b = x.detach().requires_grad_(), bias.detach().requires_grad_()
        y = process_logits(z, bias=b, masked_value=-1e4, **kind)
        return [y.detach(), *torch.autograd.grad(y, [z, b], dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = both()
    with torch.cuda.graph(second):
        other = both()
    for k in range(4):
        x.copy_(torch.randn(x.shape, device=dev))
        kind["history"].copy_(torch.randint(0, 3000, kind["history"].shape, device=dev))
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        want = both()
        for a, b, c in zip(static, want, other):
            assert torch.equal(a, b) and torch.equal(a, c), k


def test_two_streams(dev):
    from src.gcn.hip.logits import process_logits
    jobs = [case(dev, 40, 20000, length=200, seed=s, bias_rows=1) for s in (1, 2)]
    want = [process_logits(x, **kind) for x, kind, _ in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for st, (x, kind, _) in zip(streams, jobs):
        with torch.cuda.stream(st):
            got.append(process_logits(x, **kind))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_offsets_beyond_32_bits(dev):
    """More than 2^31 elements: the last rows against the same rows alone."""
    from src.gcn.hip.logits import process_logits
    rows, vocab = 17000, 131072
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(0))
    hist = torch.randint(0, vocab, (rows, 8), device=dev)
    bias = torch.randn(vocab, device=dev)
    kind = dict(repetition_penalty=1.3, frequency_penalty=0.5, bias=bias)
    y = process_logits(x, history=hist, **kind)
    for part in (slice(0, 3), slice(16380, 16390), slice(rows - 3, rows)):
        assert torch.equal(y[part], process_logits(x[part], history=hist[part], **kind))
    z = x.requires_grad_()
    y = process_logits(z, history=hist, **kind)
    (dx,) = torch.autograd.grad(y, [z], y.detach())
    last = x[-3:].detach().requires_grad_()
    (ref,) = torch.autograd.grad(process_logits(last, history=hist[-3:], **kind), [last], y[-3:].detach())
    assert torch.equal(dx[-3:], ref)


def test_empty_logits_and_their_gradients(dev):
    from src.gcn.hip.logits import process_logits
    for shape in ((0, 8), (3, 0, 8), (4, 8, 0)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        b = torch.zeros(8, device=dev, requires_grad=True)
        y = process_logits(x, dim=len(shape) - (2 if shape[-1] == 0 else 1), bias=b)
        assert y.shape == x.shape
        dx, db = torch.autograd.grad(y.sum(), [x, b])
        assert dx.shape == x.shape and not bool(db.any())


def test_in_place_without_gradients_on_a_tensor_that_needs_them(dev):
    from src.gcn.hip.logits import process_logits
    x = torch.randn(3, 8, device=dev, requires_grad=True)
    y = x * 2
    z = (y * y).sum()
    with torch.no_grad():
        want = process_logits(y, temperature=2.0)
        assert process_logits(y, temperature=2.0, out=y) is y and torch.equal(y, want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        w = torch.randn(3, 8, device=dev)
        ref = process_logits(w, temperature=2.0)
        assert torch.equal(process_logits(w, temperature=2.0, out=w), ref)


def test_more_workgroups_than_one_grid_dimension(dev):
    """2^23 rows of a few entries: more than 2^32 threads of 512 in one dimension."""
    from src.gcn.hip.logits import process_logits
    rows, vocab = (1 << 23) + 5, 3
    x = torch.randn(rows, vocab, device=dev, generator=torch.Generator(dev).manual_seed(0))
    bias = torch.randn(rows, vocab, device=dev)
    z, b = x.requires_grad_(), bias.requires_grad_()
    y = process_logits(z, bias=b, temperature=0.5)
    assert torch.equal(y, (x + bias) * 2)
    dx, db = torch.autograd.grad(y, [z, b], torch.ones_like(y))
    assert bool((dx == 2).all()) and bool((db == 2).all())


def test_capture_over_a_leaf_of_a_living_graph_is_refused(dev):
    """The refusal comes before anything is recorded; once the eager graph is gone, the capture works."""
    from src.gcn.hip.logits import process_logits
    x = torch.randn(4, 100, device=dev).requires_grad_()
    bias = torch.randn(100, device=dev).requires_grad_()
    for kept in (lambda: process_logits(x, temperature=2.0), lambda: bias * 2):
        alive = kept()
        with pytest.raises(RuntimeError, match="leaf of a graph that lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                process_logits(x, bias=bias)
        with torch.no_grad():                                # no gradient, no refusal
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                process_logits(x, bias=bias)
        del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(process_logits(x, bias=bias, temperature=2.0), [x], torch.ones(4, 100, device=dev))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert bool((dx == 0.5).all())
        dx.zero_()


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("inner", [1, 3])
def test_entries_that_equal_a_place_modulo_2_to_the_32_are_skipped(dev, wide, inner):
    """Padding of any kind, in forward and backward: negative entries, the type's ends, and in 64 bits those that differ from a place
    by a multiple of 2^32 or 2^31.  Histories shorter and longer than a turn of the walk, with prompts of every kind."""
    from src.gcn.hip.logits import process_logits
    vocab = 9000
    pads = [-1, -vocab, vocab, 2 ** 31 - 1, -2 ** 31, vocab + 4096]
    if wide == torch.int64:
        pads += [2 ** 32 + 5, 2 ** 31 + 5, -2 ** 32 + 5, 2 ** 40 + 5, 2 ** 63 - 1, -2 ** 63, 2 ** 32 + 5000, -2 ** 32 + 8999]
    gen = torch.Generator().manual_seed(4)
    for length in (40, 2500, 9000):
        real = torch.randint(0, vocab, (2, length), generator=gen)
        keep = torch.rand(2, length, generator=gen) < 0.5
        padded = torch.where(keep, real, torch.tensor(pads)[torch.randint(0, len(pads), (2, length), generator=gen)]).to(wide)
        # the same entries without padding: those that count, in place; the rest become one entry outside
        plain = torch.where(keep, real, -1).to(wide)
        prompt = torch.tensor([length // 3, -5], dtype=wide, device=dev)
        shape = (2, vocab) if inner == 1 else (2, vocab, inner)
        x = torch.randn(shape, generator=gen).to(dev).requires_grad_()
        kind = dict(dim=1, repetition_penalty=1.5, presence_penalty=0.5, frequency_penalty=0.25, prompt_lens=prompt)
        got, want = (process_logits(x, history=h.to(dev), **kind) for h in (padded, plain))
        assert torch.equal(got, want)
        counts = torch.zeros(2, vocab, dtype=torch.float64)
        seen = torch.zeros(2, vocab, dtype=torch.bool)
        for r in range(2):
            first = max(0, int(prompt[r]))
            counts[r] = torch.bincount(real[r, first:][keep[r, first:]], minlength=vocab).double()
            seen[r] = torch.bincount(real[r][keep[r]], minlength=vocab) > 0
        z = x.detach().cpu().double().view(2, vocab, inner)
        slope = torch.where(seen.unsqueeze(-1), torch.where(z > 0, 1 / 1.5, 1.5), 1.0)
        y = z * slope - (counts * 0.25 + (counts > 0) * 0.5).unsqueeze(-1)
        # 1 / 1.5 and the product, the two terms' sum and the difference: four roundings of at most 2^-24 of what they round
        bound = 4 * 2.0 ** -24 * ((z * slope).abs() + (counts * 0.25 + 0.5).unsqueeze(-1)) + 1e-37
        assert bool(((got.detach().cpu().double().view(2, vocab, inner) - y).abs() <= bound).all())
        dx, = torch.autograd.grad(got, [x], torch.ones_like(got))
        assert bool(((dx.cpu().double().view(2, vocab, inner) - slope).abs() <= 2.0 ** -23 * slope).all())


@pytest.mark.parametrize("rows, vocab, inner, period", [(12, 6, 10, 6), (28, 14, 5, 14), (30, 100, 1, 5), (6, 2049, 1, 2), (7, 9, 3, 1), (8, 8, 4, 8)])
def test_flat_rows_take_the_rows_of_an_argument_in_turn(dev, rows, vocab, inner, period):
    """Logits with one leading dimension and arguments with a divisor of it: row o uses row o mod R, with its gradient."""
    x, kind, want = case(dev, rows, vocab, inner, seed=period, bias_rows=period, hist_rows=period)
    lead = x.dim() - (1 if inner == 1 else 2)
    flat = {k: v.flatten(0, lead - 1) if isinstance(v, torch.Tensor) and v.dim() > 1 and v.shape[:lead] == x.shape[:lead] else v for k, v in kind.items()}
    flat = {**flat, "dim": 1, **{k: flat[k].reshape(rows) for k in ("repetition_penalty", "presence_penalty", "frequency_penalty", "temperature")}}
    assert flat["bias"].shape == (period, vocab) and flat["history"].shape[0] == period and flat["mask"].shape[0] == rows
    z = x.reshape(rows, vocab) if inner == 1 else x.reshape(rows, vocab, inner)
    check(z, flat, want)
    dy = torch.randn(z.shape, device=dev, generator=torch.Generator(dev).manual_seed(2))
    got = grads(z, flat, want, period, dy)
    base = grads(x, kind, want, period, dy.view(x.shape))
    assert torch.equal(got[0].view(x.shape), base[0]) and torch.equal(got[1], base[1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("inner", [1, 3])
def test_saved_tensors_may_come_back_elsewhere(dev, dtype, inner):
    """Hooks on saved tensors return copies: dense where the logits had padded, expanded or shifted rows, or with other strides."""
    from src.gcn.hip.logits import process_logits
    rows, vocab = 7, 37
    x, kind, _ = case(dev, rows, vocab, inner, length=30, dtype=dtype, seed=5, bias_rows=rows)
    lead = x.shape[1:]
    padded = torch.full((rows, vocab + 8, *lead[1:]), 1e3, device=dev, dtype=dtype)
    padded[:, 3:3 + vocab] = x
    layouts = {"dense": x, "padded": padded[:, 3:3 + vocab], "expanded": x[:1].expand(rows, *lead),
               "every other row": torch.stack([x, -x], 1).flatten(0, 1)[::2], "transposed": x.transpose(0, 1).contiguous().transpose(0, 1)}

    def apart(t):                                  # dense rows further apart
        if t.dim() == 0 or not t.numel():
            return t.clone()
        wide = torch.zeros(*t.shape[:1], 2, *t.shape[1:], device=t.device, dtype=t.dtype)
        wide[:, 1] = t
        return wide[:, 1]

    turned = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.clone()
    same = lambda t: t
    for name, z in layouts.items():
        z, b = z.detach().requires_grad_(), kind["bias"].detach().requires_grad_()
        dy = torch.randn(z.shape, device=dev, generator=torch.Generator(dev).manual_seed(3)).to(dtype)
        step = lambda: torch.autograd.grad(process_logits(z, **{**kind, "bias": b}, masked_value=-1e4), [z, b], dy)
        base = step()
        assert float(base[0].abs().sum()) > 0
        for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                      torch.autograd.graph.saved_tensors_hooks(apart, same), torch.autograd.graph.saved_tensors_hooks(same, turned)):
            with hooks:
                got = step()
            assert all(torch.equal(g, w) for g, w in zip(got, base)), (name, hooks)
        for bad in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:1], lambda t: t.unsqueeze(0)):
            with torch.autograd.graph.saved_tensors_hooks(same, bad):
                y = process_logits(z, **{**kind, "bias": b}, masked_value=-1e4)
                with pytest.raises(RuntimeError, match="was saved as"):
                    torch.autograd.grad(y, [z, b], dy)


def test_saved_arguments_are_held_by_autograd_alone(dev):
    """What a hook moves to the host leaves the GPU: the call keeps no second reference to history and mask."""
    from src.gcn.hip.logits import process_logits
    z = torch.randn(4, 1000, device=dev, requires_grad=True)
    torch.cuda.synchronize()
    with torch.autograd.graph.save_on_cpu():
        before = torch.cuda.memory_allocated()
        y = process_logits(z, history=torch.zeros(4, 1 << 20, dtype=torch.int64, device=dev), repetition_penalty=1.5,
                           mask=torch.ones(4, 1000, dtype=torch.bool, device=dev))
        assert torch.cuda.memory_allocated() - before < 1 << 20
    y.sum().backward()
    want = torch.ones(4, 1000, device=dev)
    want[:, 0] = torch.where(z[:, 0] > 0, 1 / torch.tensor(1.5, device=dev), torch.tensor(1.5, device=dev)).detach()
    assert torch.equal(z.grad, want)


def test_lengths_of_an_empty_history_with_gradient(dev):
    from src.gcn.hip.logits import process_logits
    z = torch.randn(3, 9, device=dev, requires_grad=True)
    n = torch.zeros(3, dtype=torch.int64, device=dev)
    y = process_logits(z, history=torch.zeros(3, 0, dtype=torch.int64, device=dev), history_lens=n, prompt_lens=n, repetition_penalty=2.0)
    assert torch.equal(torch.autograd.grad(y.sum(), [z])[0], torch.ones_like(z))


def test_out_that_overlaps_is_refused(dev):
    from src.gcn.hip.logits import process_logits
    buffer = torch.randn(6, 40, device=dev)
    left, right = buffer[:, :16], buffer[:, 16:32]
    want = process_logits(left.clone(), temperature=2.0)
    assert torch.equal(process_logits(left, temperature=2.0, out=right), want)       # rows in turn, apart
    assert torch.equal(process_logits(left, temperature=2.0, out=left), want)        # in place
    keep = buffer.clone()
    flat = buffer.view(-1)
    for x, out in ((buffer[:, :16], buffer[:, 15:31]), (buffer[:5, :16], buffer[1:, :16]), (flat[:160].view(10, 16), flat[1:161].view(10, 16)),
                   (flat[:16].expand(10, 16), flat[:160].view(10, 16))):
        with pytest.raises(ValueError, match="overlaps the logits"):
            process_logits(x, out=out)
    x = torch.randn(6, 16, device=dev)
    for name, kind in (("bias", dict(bias=left[0])), ("bias", dict(bias=flat[3:19])), ("temperature", dict(temperature=left[2, 3:4])),
                       ("mask", dict(mask=left[1, :1].view(torch.int32))), ("history", dict(history=right[2, :4].view(torch.int32)))):
        out = right if name == "history" else left
        with pytest.raises(ValueError, match=f"out overlaps {name}"):
            process_logits(x, out=out, **kind)
    assert torch.equal(process_logits(x, bias=buffer[2, 24:40], out=left), process_logits(x, bias=keep[2, 24:40].clone()))   # between out's rows
    assert torch.equal(buffer[:, 32:], keep[:, 32:])


def vectorised(x, hist, lens, rho, tau, allowed, dy, bias_rows):
    """dx, dbias and the magnitude of dbias' terms in double precision for logits [rows, vocab, inner], all rows at once."""
    rows, vocab, _ = x.shape
    seen = np.zeros((rows, vocab + 1), dtype=bool)
    used = (np.arange(hist.shape[1]) < lens[:, None]) & (hist >= 0) & (hist < vocab)
    seen[np.arange(rows)[:, None], np.where(used, hist, vocab)] = True
    seen = seen[:, :vocab, None]
    g = np.where(allowed[:, :, None], dy / tau[:, None, None], 0.0)
    dx = g * np.where(seen, np.where(x > 0, 1 / rho[:, None, None], rho[:, None, None]), 1.0)
    per = g.reshape(rows // bias_rows, bias_rows, vocab, -1)
    return dx, per.sum((0, 3)), np.abs(per).sum((0, 3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bias_rows, times, vocab, inner, mask", [
    (1024, 9, 14, 10, "bits"), (1024, 17, 6, 7, "bool"), (512, 20, 50, 100, "bits"), (1030, 8, 5, 3, None), (1024, 16, 3, 2, "bits"),
    (1024, 33, 21, 1, "bits"), (1024, 70, 9, 1, "bool"), (512, 64, 4100, 1, None), (1025, 32, 8, 1, "bits"), (1024, 31, 40, 1, "bits"),
    (1, 50000, 3, 1, "bits"), (4, 9000, 14, 10, "bits"), (3, 12000, 33, 1, None)])
def test_gradient_over_many_rows_of_a_workgroup(dev, dtype, bias_rows, times, vocab, inner, mask):
    """More than 1024 (bias row, range) pairs, so that a workgroup takes all `times` rows of a bias row, or so many rows that each of up to
    1024 parts has dozens: several turns of 8 (scores) or 32 rows (tokens), the last one cut off, with histories that differ from row
    to row; every row of dx, and dbias."""
    from src.gcn.hip.logits import pack_mask, process_logits
    rng, rows = np.random.default_rng(times), bias_rows * times
    if rows * vocab * inner > 1 << 25 and dtype == torch.float32:
        dtype = torch.float16                                                    # half the memory on the host, and the third type
    x = torch.from_numpy(rng.standard_normal((rows, vocab, inner), dtype=np.float32)).to(dtype)
    dy = torch.from_numpy(rng.standard_normal((rows, vocab, inner), dtype=np.float32)).to(dtype)
    length = 12
    hist, lens = rng.integers(-1, vocab + 1, (rows, length)), rng.integers(0, length + 1, rows)
    rho, tau = rng.uniform(0.6, 1.7, rows).astype(np.float32), rng.uniform(0.5, 2.0, rows).astype(np.float32)
    allowed = rng.random((rows, vocab)) < 0.8 if mask else np.ones((rows, vocab), dtype=bool)
    put = lambda a: torch.from_numpy(a).to(dev)
    shape = (rows, vocab) if inner == 1 else (rows, vocab, inner)
    z = x.to(dev).view(shape).requires_grad_()
    b = torch.zeros(bias_rows, vocab, device=dev, requires_grad=True)
    kind = dict(dim=1, history=put(hist), history_lens=put(lens), repetition_penalty=put(rho), temperature=put(tau), masked_value=-1e4,
                mask=None if mask is None else pack_mask(put(allowed)) if mask == "bits" else put(allowed))
    got = torch.autograd.grad(process_logits(z, bias=b, **kind), [z, b], dy.to(dev).view(shape))
    dx, db, size = vectorised(host(x), hist, lens, rho.astype(np.float64), tau.astype(np.float64), allowed, host(dy), bias_rows)
    assert (np.abs(host(got[0], dx.shape) - dx) <= (4 * U + half_step(dtype)) * np.abs(dx) + 2.0 ** -25 * (dtype == torch.float16)).all()
    assert (np.abs(host(got[1]) - db) <= (times * inner + 2) * U * size + 1e-44).all()
    # without a bias: the rows are dealt to at most 1024 parts
    (only,) = torch.autograd.grad(process_logits(z, **kind), [z], dy.to(dev).view(shape))
    assert torch.equal(only, got[0])
