"""AdamW step (fp32 and 8-bit states) and gradient norm on the GPU against the formulas in double precision.

Tolerances count roundings, u = 2^-24 each (inputs are taken exactly):
  m: |err| <= 6 u (|b1 m| + |(1-b1) g'|)       constants, scale, two products, one sum
  v: |err| <= 8 u v                            g' enters squared
  p: |err| <= 4 u |p| + 20 u lr / (1-b1^t) (|b1 m| + |(1-b1) g'|) / (sqrt(v) / sqrt(1-b2^t) + eps)
16-bit parameters: half a step of the type more (2^-9 of the value in bf16's 8 bits, 2^-12 in fp16's 11: torch.finfo.eps / 2).
8-bit codes have to be those of the definition but where the error of the value, as above, can turn the decision."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
SIZES = [1, 2, 7, 0, 127, 128, 129, 2047, 2048, 2049, 4096, 4097, 12345]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a ROCm GPU")
    return torch.device("cuda:0")


@pytest.fixture
def A():
    from src.gcn.hip import fused_adamw
    return fused_adamw


def make(A, dev, sizes, dtype, bits, seed=0, offset=0):
    """Parameters, gradients and states on the device, each inside a larger buffer of its own (offset elements in, with sentinels
    around), and the sentinels' check."""
    rng = np.random.default_rng(seed)
    buffers = []

    def place(x, dtype, off):
        x = torch.from_numpy(np.ascontiguousarray(x)).to(dtype)
        buf = torch.full((x.numel() + 64 + off,), 77, dtype=dtype, device=dev)
        view = buf[32 + off:32 + off + x.numel()]
        view.copy_(x.to(dev))
        buffers.append((buf, off, x.numel()))
        return view

    s = {k: [] for k in ("p", "g", "m", "v", "master", "em", "ev")}
    for n in sizes:
        size = np.exp2(rng.uniform(-10, 1, n))
        w, g = 0.1 * rng.standard_normal(n), size * rng.standard_normal(n) * (rng.random(n) > 0.05)
        m, v = 0.5 * size * rng.standard_normal(n), size ** 2 * np.exp2(rng.uniform(-1, 1, n))
        s["p"].append(place(w.astype(np.float32), dtype, offset))
        s["g"].append(place(g.astype(np.float32), dtype, offset))
        if dtype != torch.float32:
            s["master"].append(place(w.astype(np.float32), torch.float32, offset))
        if bits == 32:
            s["m"].append(place(m.astype(np.float32), torch.float32, offset))
            s["v"].append(place(v.astype(np.float32), torch.float32, offset))
        else:
            for key, x, nz in (("m", m, False), ("v", np.sqrt(v), True)):
                codes, exps = A.state8_encode(torch.from_numpy(x.astype(np.float32)), never_zero=nz)
                s[key].append(place(codes.numpy(), torch.uint8, offset))
                s["e" + key].append(place(exps.numpy(), torch.uint8, offset))

    def intact():
        for buf, off, n in buffers:
            keep = torch.cat([buf[:32 + off], buf[32 + off + n:]])
            assert bool((keep == 77).all()), "an element beside a tensor was written"
    return s, intact


def call(A, s, step=5, **k):
    eight, half = bool(s["em"]), bool(s["master"])
    A.adamw_step_(s["p"], s["g"], s["m"], s["v"], step=step, masters=s["master"] if half else None,
                  exp_avg_exps=s["em"] if eight else None, exp_avg_sq_exps=s["ev"] if eight else None, **{**HYPER, **k})


def host(s):
    return {k: [t.detach().float().cpu().numpy().astype(np.float64) if t.dtype != torch.uint8 else t.cpu().numpy() for t in ts] for k, ts in s.items()}


def check(before, after, dtype, step, scale=1.0, seed=0, hyper=HYPER, first=0):
    b1, b2 = hyper["betas"]
    eight = bool(before["em"])
    for k in range(len(before["p"])):
        p0 = before["master"][k] if before["master"] else before["p"][k]
        g = before["g"][k]
        m0 = O.decode(before["m"][k], before["em"][k]) if eight else before["m"][k]
        v0 = O.decode(before["v"][k], before["ev"][k]) ** 2 if eight else before["v"][k]
        p, m, v = O.step(p0, g, m0, v0, t=step, lr=hyper["lr"], b1=b1, b2=b2, eps=hyper["eps"], wd=hyper["weight_decay"], scale=scale)
        spread = np.abs(b1 * m0) + np.abs((1 - b1) * g * scale)
        tol_p = 4 * U * np.abs(p) + 20 * U * hyper["lr"] / (1 - b1 ** step) * spread / (np.sqrt(v / (1 - b2 ** step)) + hyper["eps"])
        got = after["master"][k] if after["master"] else after["p"][k]
        assert (np.abs(got - p) <= tol_p).all()
        if after["master"]:
            half = torch.finfo(dtype).eps / 2
            assert (np.abs(after["p"][k] - after["master"][k]) <= half * np.abs(p) + 2.0 ** -25).all()
        if not eight:
            assert (np.abs(after["m"][k] - m) <= 6 * U * spread + 1e-44).all()
            assert (np.abs(after["v"][k] - v) <= 8 * U * v + 1e-44).all()
            continue
        r = O.random32(p.size, seed, step, first + k).astype(np.int64)
        for key, x, err, bits, nz in (("m", m, 6 * U * spread, r & 0xFFFF, False), ("v", np.sqrt(v), 5 * U * np.sqrt(v), r >> 16, True)):
            want, exps, margin, unit = O.encode(x, bits, nz)
            got_e = after["e" + key][k].astype(np.int64)
            same = np.repeat(got_e == exps, O.BLOCK)[:p.size]
            if not same.all():                       # the block's largest value is a power of two but for its error
                near = np.abs(np.abs(x) / np.exp2(np.round(np.log2(np.maximum(np.abs(x), 1e-300)))) - 1) <= 8 * U
                for blk in np.flatnonzero(got_e != exps):
                    assert near[blk * O.BLOCK:(blk + 1) * O.BLOCK].any()
            got = O.decode(after[key][k], after["e" + key][k])
            off = np.abs(got - want)
            assert (off <= unit * (1 + 1e-9))[same].all()
            assert ((off == 0) | (margin * unit <= err + 1e-12 * unit))[same].all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("offset", [0, 1])
def test_step_matches_the_formula(dev, A, dtype, bits, offset):
    s, intact = make(A, dev, SIZES, dtype, bits, seed=1, offset=offset)
    before = host(s)
    call(A, s, seed=99, first_tensor=4)
    check(before, host(s), dtype, 5, seed=99, first=4)
    intact()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scale_and_clip_coefficient(dev, A, dtype, bits):
    s, _ = make(A, dev, [5, 3000, 128], dtype, bits, seed=2)
    before = host(s)
    scale, clip = torch.tensor(0.37, device=dev), torch.tensor([0.011], device=dev)
    call(A, s, step=1, grad_scale=scale, clip_coef=clip)
    check(before, host(s), dtype, 1, scale=float(scale) * float(clip))
    assert all(np.array_equal(a, b) for a, b in zip(before["g"], host(s)["g"]))


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_from_zero_states_and_late_steps(dev, A, bits):
    for step in (1, 2, 1000000):
        s, _ = make(A, dev, [1000], torch.float32, bits, seed=3)
        for key in ("m", "v", "em", "ev"):
            for t in s[key]:
                t.zero_()
        before = host(s)
        call(A, s, step=step)
        check(before, host(s), torch.float32, step)


@pytest.mark.parametrize("hyper", [dict(lr=0.0), dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(eps=1e-3, betas=(0.5, 0.9))])
@pytest.mark.parametrize("bits", [32, 8])
def test_other_hyperparameters(dev, A, bits, hyper):
    s, _ = make(A, dev, [777], torch.float32, bits, seed=4)
    before = host(s)
    call(A, s, **hyper)
    check(before, host(s), torch.float32, 5, hyper={**HYPER, **hyper})


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_equal_one_at_a_time(dev, A, bits):
    sizes = [(37 * k * k) % 3001 if k % 9 else 0 for k in range(150)]
    s, intact = make(A, dev, sizes, torch.bfloat16, bits, seed=5)
    one = {k: [t.clone() for t in ts] for k, ts in s.items()}
    call(A, s, seed=3)
    for k in range(len(sizes)):
        call(A, {key: ts[k:k + 1] for key, ts in one.items()}, seed=3, first_tensor=k)
    for key in s:
        assert all(torch.equal(a, b) for a, b in zip(s[key], one[key])), key
    intact()


@pytest.mark.parametrize("bits", [32, 8])
def test_equal_calls_give_equal_bits(dev, A, bits):
    runs = []
    for seed in (7, 7, 8):
        s, _ = make(A, dev, [100001, 50], torch.float32, bits, seed=6)
        call(A, s, seed=seed)
        runs.append(s)
    for key in ("p", "m", "v", "em", "ev"):
        assert all(torch.equal(a, b) for a, b in zip(runs[0][key], runs[1][key])), key
    assert torch.equal(runs[0]["m"][0], runs[2]["m"][0]) == (bits == 32)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_bad_gradient_stays_with_its_element(dev, A, bits, bad):
    s, _ = make(A, dev, [500], torch.float32, bits, seed=7)
    good = {k: [t.clone() for t in ts] for k, ts in s.items()}
    # a small element of its block, so that the block's scale does not hang on it
    at = int(torch.where((good["g"][0].abs() < good["g"][0].abs().max() / 4), 1, 0)[:128].nonzero()[5])
    for t in (good["g"][0],):
        t[at] = 0
    if bits == 8:
        good["m"][0][at] = 0
    else:
        good["m"][0][at] = 0.0
    s = {k: [t.clone() for t in ts] for k, ts in good.items()}
    s["g"][0][at] = bad
    call(A, good)
    call(A, s)
    assert bool(s["p"][0][at].isnan())
    keep = torch.arange(500, device=dev) != at
    assert torch.equal(s["p"][0][keep], good["p"][0][keep])
    if bits == 32:
        for key in ("m", "v"):
            assert torch.equal(s[key][0][keep], good[key][0][keep])
            assert not bool(s[key][0][at].isfinite())
    else:
        assert torch.equal(s["m"][0][keep], good["m"][0][keep])
        # the largest code in the place of what is not finite; neighbours as far as the element was not the block's largest
        assert int(s["m"][0][at]) & 127 == 126 and int(s["v"][0][at]) == 126


def test_8_bit_rounding_keeps_the_mean_and_the_moments_move(dev, A):
    """With constant second moments of gradients, v stays near them: its SR noise raises E[r^2] by Var(r): one step changes
    sqrt(v) by |d| <= 0.5e-3 |g^2/v - 1| relative, rounding in steps of at most 1/8 adds at most d / 8 of variance per step, and
    the memory of 500 steps of relative size 1e-3 each in r^2 leaves at most 0.97 * 0.5e-3 / 8 / 1e-3 < 0.07 of r^2.
    Rounding to the nearest would stop at about 30 steps' worth: 0.03."""
    n, steps = 1 << 16, 3000
    gen = torch.Generator(dev).manual_seed(1)
    p, m, v = torch.zeros(n, device=dev), torch.zeros(n, dtype=torch.uint8, device=dev), torch.zeros(n, dtype=torch.uint8, device=dev)
    em, ev = (torch.zeros(n // 128, dtype=torch.uint8, device=dev) for _ in range(2))
    exact_v = exact_m = 0.0
    for t in range(1, steps + 1):
        g = torch.randn(n, device=dev, generator=gen)
        A.adamw_step_([p], [g], [m], [v], step=t, lr=1e-3, exp_avg_exps=[em], exp_avg_sq_exps=[ev])
        exact_v = 0.999 * exact_v + 0.001 * g.double() ** 2
        exact_m = 0.9 * exact_m + 0.1 * g.double()
    got = A.state8_decode(v, ev).double() ** 2
    ratio = float(got.mean() / exact_v.mean())
    assert 0.99 < ratio < 1.07, ratio
    # the first moment follows element by element: errors of at most 1/8 per step that fade by 0.9 each: std < 0.125 / sqrt(1 - 0.81)
    diff = (A.state8_decode(m, em).double() - exact_m)
    assert abs(float(diff.mean())) < 5 * float(diff.std()) / n ** 0.5 + 1e-9
    assert float(diff.std() / exact_m.std()) < 0.125 / (1 - 0.81) ** 0.5


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_captured_steps_count_on(dev, A, bits, dtype):
    """Graph replays, with eager work between them, against eager steps: equal bits."""
    def fresh():
        s, _ = make(A, dev, [3000, 17, 128 * 20], dtype, bits, seed=8)
        return s
    grads = [torch.randn(sum([3000, 17, 128 * 20]), device=dev, generator=torch.Generator(dev).manual_seed(k)).to(dtype) for k in range(5)]

    def feed(s, k):
        for t, x in zip(s["g"], grads[k].split([3000, 17, 128 * 20])):
            t.copy_(x)

    def both(s, **k):
        _, coef = A.grad_norm(s["g"], max_norm=1.0)
        call(A, s, clip_coef=coef, **k)
    want = fresh()
    for k in range(5):
        feed(want, k)
        both(want, step=11 + k, seed=5)
    s = fresh()
    count, hyper = torch.tensor(10, device=dev), A.adamw_hyper(dev)
    options = {**HYPER, "seed": 5}
    warm = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(warm, step=1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.adamw_advance_(count, hyper, **options)
        both(s, step=0, hyper=hyper, seed=5)
    assert int(count) == 10
    for k in range(5):
        feed(s, k)
        graph.replay()
        torch.cuda.synchronize()
        _ = torch.randn(1000, device=dev).sum().item()       # eager work and a synchronisation between the replays
    assert int(count) == 15
    for key in s:
        assert all(torch.equal(a, b) for a, b in zip(s[key], want[key])), key
    with pytest.raises(RuntimeError, match="step count"):
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2):
            both(s, step=3)


def test_steps_on_two_streams(dev, A):
    want, _ = make(A, dev, [200000], torch.float32, 8, seed=9)
    other, _ = make(A, dev, [200000], torch.float32, 8, seed=10)
    ref = [{k: [t.clone() for t in ts] for k, ts in x.items()} for x in (want, other)]
    norms = []
    for x in ref:
        n, coef = A.grad_norm(x["g"], max_norm=1.0)
        norms.append(float(n))
        call(A, x, clip_coef=coef)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for st, x in zip(streams, (want, other)):
        with torch.cuda.stream(st):
            n, coef = A.grad_norm(x["g"], max_norm=1.0)
            call(A, x, clip_coef=coef)
            got.append(n)
    torch.cuda.synchronize()
    assert [float(n) for n in got] == norms
    for x, y in zip((want, other), ref):
        for key in x:
            assert all(torch.equal(a, b) for a, b in zip(x[key], y[key])), key


# ---------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [[1], [0], SIZES, [3_000_001], [5] * 200], ids=str)
def test_norm(dev, A, dtype, sizes):
    gen = torch.Generator(dev).manual_seed(2)
    grads = [torch.randn(n + 1, device=dev, generator=gen).to(dtype)[k % 2:][:n] for k, n in enumerate(sizes)]
    want = float(np.sqrt(sum(float((g.double() ** 2).sum()) for g in grads)))
    norm, none = A.grad_norm(grads)
    assert none is None and norm.dtype == torch.float32
    # one rounding to fp32 (double sums in another order: 1e-13)
    assert abs(float(norm) - want) <= (U + 1e-12) * want
    for scale in (None, torch.tensor(-0.5, device=dev)):
        norm, coef = A.grad_norm(grads, max_norm=0.3, grad_scale=scale)
        w = want * (1.0 if scale is None else 0.5)
        assert abs(float(norm) - w) <= (U + 1e-12) * w
        c = min(1.0, 0.3 / (w + 1e-6))
        assert abs(float(coef) - c) <= (U + 1e-12) * c


def test_norm_of_extreme_and_bad_gradients(dev, A):
    for value in (1e30, 1e-30, 3e38):
        g = [torch.full((1000,), value, device=dev)]
        want = float(g[0][0].double()) * 1000 ** 0.5
        norm, coef = A.grad_norm(g, max_norm=1.0)
        if want < 3.4e38:
            assert abs(float(norm) - want) <= (U + 1e-12) * want
        else:
            assert np.isinf(float(norm))
        assert abs(float(coef) - min(1.0, 1 / (want + 1e-6))) <= 2 * U * float(coef) + 1e-45
    bad = torch.ones(10, device=dev)
    bad[3] = float("inf")
    norm, coef = A.grad_norm([bad], max_norm=1.0)
    assert np.isinf(float(norm)) and float(coef) == 0
    bad[4] = float("nan")
    norm, coef = A.grad_norm([bad], max_norm=1.0)
    assert np.isnan(float(norm)) and np.isnan(float(coef))
    norm, coef = A.grad_norm([torch.zeros(7, device=dev)], max_norm=0.0)
    assert float(norm) == 0 and float(coef) == 0


# ---------------------------------------------------------------------------------------------------- optimizer
def model(dev, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s).to(dev, dtype)) for s in ((70, 90), (90,), (33,), (5000,))]


def feed_grads(params, k, skip=()):
    gen = torch.Generator(params[0].device).manual_seed(1000 + k)
    for i, p in enumerate(params):
        g = torch.randn(p.shape, device=p.device, generator=gen)
        p.grad = None if i in skip else g.to(p.dtype)


def test_optimizer_follows_torch_adamw_and_exchanges_checkpoints(dev, A):
    """Five steps beside torch.optim.AdamW; both are within 24 u |p|-scale of the formula per step, so 10 steps' worth apart."""
    a, b = model(dev), model(dev)
    ours = A.FusedAdamW(a, lr=1e-2, weight_decay=0.1)
    theirs = torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1, foreach=False)
    for k in range(5):
        for ps in (a, b):
            feed_grads(ps, k, skip=(2,) if k == 2 else ())
        ours.step()
        theirs.step()
    assert [float(ours.state[p]["step"]) for p in a] == [5, 5, 4, 5]
    for x, y in zip(a, b):
        # an update is at most about lr per element; 24 roundings of parameter and update per step and side
        assert float((x - y).detach().abs().max()) <= 10 * 24 * U * (float(y.detach().abs().max()) + 1e-2)
    c = model(dev)
    with torch.no_grad():
        for x, y in zip(c, b):
            x.copy_(y)
    moved = A.FusedAdamW(c, lr=1e-2, weight_decay=0.1)
    moved.load_state_dict(theirs.state_dict())
    back = torch.optim.AdamW(a, lr=1e-2, weight_decay=0.1, foreach=False)
    back.load_state_dict(ours.state_dict())
    for ps in (a, b, c):
        feed_grads(ps, 9)
    for opt in (moved, back, theirs):
        opt.step()
    assert [float(moved.state[p]["step"]) for p in c] == [6, 6, 5, 6]
    for x, y, z in zip(a, b, c):
        assert float((x - y).detach().abs().max()) <= 12 * 24 * U * (float(y.detach().abs().max()) + 1e-2)
        assert float((z - y).detach().abs().max()) <= 2 * 24 * U * (float(y.detach().abs().max()) + 1e-2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_checkpoint_continues_bit_for_bit(dev, A, tmp_path, dtype, bits, capturable):
    kind = dict(lr=1e-2, state_bits=bits, min_8bit_numel=1000, max_grad_norm=1.0, capturable=capturable, seed=4)
    a = model(dev, dtype)
    one = A.FusedAdamW(a, **kind)
    for k in range(3):
        feed_grads(a, k)
        one.step()
    st = one.state[a[0]]
    assert ("exp_avg_exp" in st) == (bits == 8) and "exp_avg_exp" not in one.state[a[1]]
    assert ("master" in st) == (dtype != torch.float32)
    assert len({id(one.state[p]["step"]) for p in a}) == 1
    torch.save(one.state_dict(), tmp_path / "opt.pt")
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    two = A.FusedAdamW(b, **kind)
    two.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    for k in range(3, 5):
        for ps, opt in ((a, one), (b, two)):
            feed_grads(ps, k)
            opt.step()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
        for key in one.state[x]:
            if key != "step":
                assert torch.equal(one.state[x][key], two.state[y][key]), key
    assert float(one.grad_norm) == float(two.grad_norm) > 0


def test_checkpoints_change_width(dev, A):
    a = model(dev)
    wide = A.FusedAdamW(a, lr=1e-2)
    feed_grads(a, 0)
    wide.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    narrow = A.FusedAdamW(b, lr=1e-2, state_bits=8, min_8bit_numel=1000)
    narrow.load_state_dict(wide.state_dict())
    st, ref = narrow.state[b[0]], wide.state[a[0]]
    m = A.state8_decode(st["exp_avg"], st["exp_avg_exp"])
    scale = float(ref["exp_avg"].abs().max())
    assert bool(((m - ref["exp_avg"]).abs() <= 2.0 ** -4 * ref["exp_avg"].abs() + 2.0 ** -17 * scale).all())
    feed_grads(b, 1)
    narrow.step()
    c = [torch.nn.Parameter(p.detach().clone()) for p in b]
    again = A.FusedAdamW(c, lr=1e-2)
    again.load_state_dict(narrow.state_dict())
    assert torch.equal(again.state[c[0]]["exp_avg"], A.state8_decode(narrow.state[b[0]]["exp_avg"], narrow.state[b[0]]["exp_avg_exp"]))
    assert float(again.state[c[0]]["step"]) == 2
    feed_grads(c, 2)
    again.step()
    broken = narrow.state_dict()
    broken["state"][0] = {**broken["state"][0], "exp_avg": torch.zeros(3, dtype=torch.uint8)}
    with pytest.raises(ValueError):
        again.load_state_dict(broken)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_captured_with_clipping(dev, A, bits):
    """The whole step, clipping included, replayed from a graph, against the same steps made eagerly."""
    kind = dict(lr=1e-2, state_bits=bits, min_8bit_numel=1000, max_grad_norm=0.5, capturable=True)
    a, b = model(dev, torch.bfloat16), model(dev, torch.bfloat16)
    oa, ob = A.FusedAdamW(a, **kind), A.FusedAdamW(b, **kind)
    fixed = [torch.zeros_like(p) for p in b]
    for k in range(5):
        feed_grads(a, k)
        oa.step()
        if k == 0:
            feed_grads(b, 0)
            ob.step()
            graph = torch.cuda.CUDAGraph()
            for p, g in zip(b, fixed):
                p.grad = g
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                ob.step()
        else:
            for p, q in zip(a, fixed):
                q.copy_(p.grad)
            graph.replay()
            torch.cuda.synchronize()
            assert float(ob.grad_norm) == float(oa.grad_norm)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert [int(ob.state[p]["step"]) for p in b] == [5] * 4


def test_optimizer_mixed_types_and_groups(dev, A):
    wide, half = model(dev)[:2], model(dev, torch.bfloat16, seed=3)[:2]
    opt = A.FusedAdamW([{"params": wide}, {"params": half, "lr": 1e-3, "weight_decay": 0.0}], lr=1e-2, max_grad_norm=1.0)
    feed_grads(wide, 0)
    feed_grads(half, 1)
    before = [p.detach().clone() for p in wide + half]
    opt.step()
    want = np.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in wide + half))
    assert abs(float(opt.grad_norm) - want) <= 4 * U * want
    for p, b in zip(wide + half, before):
        lr, wd = (1e-2, 1e-2) if p.dtype == torch.float32 else (1e-3, 0.0)
        coef = min(1.0, 1.0 / (want + 1e-6))
        master = b.double().cpu().numpy()
        g = p.grad.double().cpu().numpy()
        q, _, _ = O.step(master, g, 0 * g, 0 * g, t=1, lr=lr, b1=0.9, b2=0.999, eps=1e-8, wd=wd, scale=coef)
        got = opt.state[p]["master"] if "master" in opt.state[p] else p.detach()
        assert np.abs(got.double().cpu().numpy() - q).max() <= 30 * U * (np.abs(q).max() + lr)
    with torch.no_grad():
        half[0].fill_(1.0)
    opt.sync_masters()
    assert bool((opt.state[half[0]]["master"] == 1).all())


def test_optimizer_without_gradients_and_refusals(dev, A):
    p = torch.nn.Parameter(torch.ones(4, device=dev))
    opt = A.FusedAdamW([p], max_grad_norm=1.0)
    opt.step()
    assert not opt.state[p]
    q = torch.nn.Parameter(torch.ones(8, 4, device=dev).t())
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="contiguous"):
        A.FusedAdamW([q]).step()
    r = torch.nn.Parameter(torch.ones(4, dtype=torch.float64, device=dev))
    r.grad = torch.ones_like(r)
    with pytest.raises(TypeError):
        A.FusedAdamW([r]).step()
    p.grad = torch.ones(8, device=dev)[::2]                  # a gradient with strides
    opt.step()
    assert float(opt.state[p]["step"]) == 1
    cap = A.FusedAdamW([torch.nn.Parameter(torch.ones(4, device=dev))], capturable=True)
    cap.param_groups[0]["params"][0].grad = torch.ones(4, device=dev)
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cap.step()


def test_device_learning_rate(dev, A):
    lr = torch.tensor(1e-2, device=dev)
    a, b = model(dev), model(dev)
    oa, ob = A.FusedAdamW(a, lr=lr, capturable=True), A.FusedAdamW(b, lr=float(lr))
    for k in range(2):
        for ps, opt in ((a, oa), (b, ob)):
            feed_grads(ps, k)
            opt.step()
        lr.mul_(0.5)
        ob.param_groups[0]["lr"] = float(lr)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_copied_and_pickled_optimizers_keep_their_options(dev, A):
    import copy
    a = model(dev)
    opt = A.FusedAdamW(a, lr=1e-2, state_bits=8, min_8bit_numel=1000, max_grad_norm=0.5, seed=9)
    feed_grads(a, 0)
    opt.step()
    twin = copy.deepcopy(opt)
    assert (twin.state_bits, twin.min_8bit_numel, twin.max_grad_norm, twin.seed) == (8, 1000, 0.5, 9)
    b = twin.param_groups[0]["params"]
    for ps, o in ((a, opt), (b, twin)):
        feed_grads(ps, 1)
        o.step()
    for x, y in zip(a, b):
        assert x is not y and torch.equal(x, y)
    assert len({id(st["step"]) for st in opt.state_dict()["state"].values()}) == 4


def test_a_parameter_twice_is_refused(dev, A):
    s, _ = make(A, dev, [100, 50], torch.float32, 32)
    twice = {k: [ts[0], ts[0]] if ts else [] for k, ts in s.items()}
    before = s["p"][0].clone()
    with pytest.raises(ValueError, match="twice"):
        call(A, twice)
    assert torch.equal(s["p"][0], before)
    empty, _ = make(A, dev, [0, 0], torch.float32, 32)
    call(A, {k: [ts[0], ts[0]] if ts else [] for k, ts in empty.items()})


def test_autograd_hears_of_the_update(dev, A):
    p = torch.nn.Parameter(torch.ones(10, device=dev))
    y = (p * p).sum()
    opt = A.FusedAdamW([p])
    p.grad = torch.ones(10, device=dev)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_parameters_that_overlap_are_refused(dev, A):
    """One that starts inside another; neighbours in one buffer are allowed."""
    buffer = torch.ones(40, device=dev)

    def step(a, b):
        state = [[torch.zeros_like(x) for x in (a, b)] for _ in range(2)]
        A.adamw_step_([a, b], [torch.ones_like(a), torch.ones_like(b)], *state, step=1, lr=1e-2)
    with pytest.raises(ValueError, match="overlap"):
        step(buffer[:20], buffer[19:])
    with pytest.raises(ValueError, match="twice"):
        step(buffer[:20], buffer[:30])
    assert torch.equal(buffer, torch.ones_like(buffer))
    step(buffer[20:], buffer[:20])
    assert bool((buffer < 1).all())


def test_a_refused_capture_counts_no_step(dev, A):
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    p.grad = torch.ones_like(p)
    opt = A.FusedAdamW([p])
    opt.step()
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert float(opt.state[p]["step"]) == 1 and torch.equal(p.detach(), before)
    opt.step()
    assert float(opt.state[p]["step"]) == 2


def _turn(p):
    p.data = torch.ones(p.shape[::-1], device=p.device).t()


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("name", ["layout", "learning rate", "beta", "weight decay", "gradient scale", "norm", "new parameter"])
def test_a_refused_step_counts_nothing_and_updates_nothing(dev, A, name, capturable):
    """Two groups, the second of which is refused; afterwards the optimizer goes on as one that was never refused."""
    def build():
        a, b = model(dev)[:2], model(dev, torch.bfloat16, seed=3)[:2]
        opt = A.FusedAdamW([{"params": a}, {"params": b}], lr=1e-2, capturable=capturable, max_grad_norm=1.0)
        feed_grads(a + b, 0)
        opt.step()
        return a, b, opt

    a, b, opt = build()
    before = [[x.clone() for x in (p.detach(), *(v for k, v in sorted(opt.state[p].items())))] for p in a + b]
    group, kind, new = opt.param_groups[1], {}, []
    if name == "layout":
        keep = b[0].data
        _turn(b[0])
    elif name == "learning rate":
        group["lr"] = torch.tensor(1e-2, dtype=torch.float64, device=dev) if capturable else -1.0
    elif name == "beta":
        group["betas"] = (0.9, 1.0)
    elif name == "weight decay":
        group["weight_decay"] = -0.5
    elif name == "gradient scale":
        kind["grad_scale"] = torch.ones((), dtype=torch.float64, device=dev)
    elif name == "norm":
        kind["max_grad_norm"] = -1.0
    else:
        new = [torch.nn.Parameter(torch.ones(5, device=dev)), torch.nn.Parameter(torch.ones(8, 4, device=dev).t())]
        opt.add_param_group({"params": new})
        for q in new:
            q.grad = torch.ones_like(q)
    feed_grads(a + b, 1)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        opt.step(**kind)
    if name == "layout":
        b[0].data = keep
    for p, want in zip(a + b, before):
        now = [p.detach(), *(v for k, v in sorted(opt.state[p].items()))]
        assert len(now) == len(want) and all(torch.equal(x, y) for x, y in zip(now, want))
    assert not any(opt.state.get(q) for q in new)
    # mended, it goes on
    group.update(lr=1e-2, betas=(0.9, 0.999), weight_decay=1e-2)
    for q in new:
        q.grad = None
    other_a, other_b, other = build()
    for ps, o in ((a + b, opt), (other_a + other_b, other)):
        feed_grads(ps, 1)
        o.step()
    assert all(torch.equal(x, y) for x, y in zip(a + b, other_a + other_b))
    assert {int(opt.state[p]["step"]) for p in a + b} == {2}


def test_a_call_keeps_its_tensors(dev, A):
    """What the optimizer prepares outlives the lists that it was made from."""
    from src.gcn.hip import lib as L
    p, g = [torch.ones(1000, device=dev)], [torch.ones(1000, device=dev)]
    m, v = [torch.zeros(1000, device=dev)], [torch.zeros(1000, device=dev)]
    keep = p[0]
    call_ = L.binding().AdamwCall(p, g, m, v, None, None, None)
    for ts in (p, g, m, v):
        ts.clear()
    junk = [torch.full((1000,), 7.0, device=dev) for _ in range(4)]
    call_.run(1, 0.5, 0.9, 0.999, 1e-8, 0.0, 0, 0, None, None, None)
    assert float((keep - 0.5).abs().max()) <= 1e-6 and all(bool((j == 7).all()) for j in junk)


@pytest.mark.parametrize("why", ["types", "step counts"])
def test_lists_of_one_group_round_with_bits_of_their_own(dev, A, why):
    """A group that falls into several 8-bit lists: equal values and gradients in each, and the oracle's bits for the tensors numbered one
    after the other.  Equal bits would give equal codes; of 4096 elements rounded at random about half or more differ."""
    n = 4096
    grads = [torch.from_numpy(np.random.default_rng(7).standard_normal(n).astype(np.float32)).to(torch.bfloat16).float().to(dev) for _ in range(4)]
    types = [torch.float32, torch.bfloat16, torch.float32, torch.bfloat16] if why == "types" else [torch.float32] * 4
    small = torch.nn.Parameter(torch.ones(8, device=dev))                    # fp32 moments: takes no number
    params = [torch.nn.Parameter(torch.ones(n, device=dev, dtype=t)) for t in types]
    opt = A.FusedAdamW([small, *params], lr=1e-2, state_bits=8, seed=5)
    small.grad = torch.ones_like(small)
    if why == "step counts":                                                  # two of them miss a step; then all states are made equal
        for p in params[:2]:
            p.grad = torch.ones_like(p)
        opt.step()
        for p in params[2:]:
            p.grad = torch.ones_like(p)
        opt.step()
        for p in params:
            for key in ("exp_avg", "exp_avg_sq", "exp_avg_exp", "exp_avg_sq_exp"):
                opt.state[p][key].zero_()
        with torch.no_grad():
            for p in params[2:]:
                opt.state[p]["step"].fill_(2.0)                               # a count of their own, of the same value
    for p, g in zip(params, grads):
        p.grad = g.to(p.dtype)
    opt.step()
    codes = [opt.state[p]["exp_avg"].cpu().numpy() for p in params]
    for i in range(4):
        for j in range(i):
            assert (codes[i] != codes[j]).mean() > 0.25, (i, j)
    step = 1 if why == "types" else 3
    order = [0, 2, 1, 3] if why == "types" else [0, 1, 2, 3]
    m = (np.float32(1 - 0.9) * grads[0].cpu().numpy()).astype(np.float64)
    for number, k in enumerate(order):
        want, exps, margin, unit = O.encode(m, (O.random32(n, 5, step, number) & 0xFFFF).astype(np.int64), False)
        off = np.abs(O.decode(codes[k], opt.state[params[k]]["exp_avg_exp"].cpu().numpy()) - want)
        assert ((off == 0) | (margin * unit <= 4 * U * np.abs(m))).all()


@pytest.mark.parametrize("capturable", [False, True])
def test_parameters_that_skip_a_step_together_stay_one_list(dev, A, capturable):
    """Ten parameters without a gradient for a step, three of them for another: lists afterwards, and counts."""
    params = [torch.nn.Parameter(torch.ones(20 + k, device=dev)) for k in range(16)]
    opt = A.FusedAdamW(params, lr=1e-2, capturable=capturable)
    lists = []
    for skipped in ((), range(6, 16), (), range(13, 16), ()):
        for k, p in enumerate(params):
            p.grad = None if k in skipped else torch.ones_like(p)
        lists.append(len(opt._collect()[0]))
        opt.step()
    assert lists == [1, 1, 2, 2, 3]
    assert [int(opt.state[p]["step"]) for p in params] == [5] * 6 + [4] * 7 + [3] * 3
    assert len({id(opt.state[p]["step"]) for p in params}) == 3


def test_8_bit_states_with_two_strides_a_workgroup(dev, A):
    """Lists of more than 2^25 elements give a workgroup two strides: equal bits to the same tensors in calls of their own, which give one."""
    sizes, gen = [12_000_001, 11_999_999, 10_002_177], torch.Generator(dev).manual_seed(12)
    assert sum(sizes) > 1 << 25 and max(sizes) < 1 << 25
    sets = []
    for n in sizes:
        p = torch.randn(n, device=dev, generator=gen)
        m, v = 1e-2 * torch.randn(n, device=dev, generator=gen), 1e-2 * torch.rand(n, device=dev, generator=gen)
        sets.append([p, torch.randn(n, device=dev, generator=gen) * 1e-2, *A.state8_encode(m), *A.state8_encode(v, never_zero=True)])
    alone = [[t.clone() for t in s] for s in sets]
    kind = dict(step=3, lr=1e-3, seed=77)

    def step(group, first):
        p, g, m, em, v, ev = (list(ts) for ts in zip(*group))
        A.adamw_step_(p, g, m, v, exp_avg_exps=em, exp_avg_sq_exps=ev, first_tensor=first, **kind)
    step(sets, 4)
    for k, s in enumerate(alone):
        before = s[0].clone()
        step([s], 4 + k)
        assert not torch.equal(before, s[0])
    for a, b in zip(sets, alone):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
