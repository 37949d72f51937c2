"""Workloads of the optimizer and logits operators: the multi-tensor AdamW step (states in 32 or in 8 bits, with an
optional clip to a global gradient norm) and the rules on logits (penalties for repeated tokens, bias, masks) with their
gradient.  ``run`` computes a workload in elementary torch operations, or, with ``own`` set, through the package's entry
points; ``exact`` computes it in 64 bits."""
import itertools
import math
import os
import random
import sys

import torch

own = False

BLOCK = 128            # elements that share a scale in an 8-bit state
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM, SEED = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 1.0, 20240229
FIRST_STEP = 100       # the inputs are those of a run that is under way
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _package():
    root = os.path.join(os.getcwd(), "graph-convnet-uelb_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from src.gcn.hip import fused_adamw, logits
    return fused_adamw, logits


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the trainer's step on the default configuration (64 channels, 10 layers): many small tensors, latency counts
        {"name": "adamw_gcn_h64", "op": "adamw", "bits": 32, "kind": "gcn", "width": 64, "layers": 10, "many": 10, "type": "fp32", "clip": False},
        # a stack of wide blocks with a large embedding, trained in bf16 with an fp32 master copy
        {"name": "adamw_blocks_bf16", "op": "adamw", "bits": 32, "kind": "blocks", "width": 1280, "layers": 4, "many": 32000, "type": "bf16", "clip": False},
        # hundreds of tensors from one element to millions, odd sizes, clipped to a global norm
        {"name": "adamw_ragged_clip", "op": "adamw", "bits": 32, "kind": "ragged", "width": 2000003, "layers": 1, "many": 300, "type": "fp32", "clip": True},
        # the widest configuration of the framework (300 channels, 30 layers) with 8-bit states
        {"name": "adamw8_gcn_h300", "op": "adamw", "bits": 8, "kind": "gcn", "width": 300, "layers": 30, "many": 50, "type": "fp32", "clip": True},
        # the wide blocks with 8-bit states: the largest training step
        {"name": "adamw8_blocks_bf16", "op": "adamw", "bits": 8, "kind": "blocks", "width": 1280, "layers": 6, "many": 32000, "type": "bf16", "clip": False},
        # one request being decoded, one token
        {"name": "logits_one_row", "op": "logits", "rows": 1, "vocab": 32000, "inner": 1, "history": 64, "type": "fp32", "mask": "none", "bias": "shared", "train": False, "pad": 0},
        # a batch of requests being decoded, each with its own penalties and grammar mask
        {"name": "logits_batch_64", "op": "logits", "rows": 64, "vocab": 131072, "inner": 1, "history": 2048, "type": "fp32", "mask": "bits", "bias": "shared", "train": False, "pad": 0},
        # few requests with long contexts, an odd vocabulary, rows of a padded buffer
        {"name": "logits_long_history", "op": "logits", "rows": 16, "vocab": 50021, "inner": 1, "history": 32768, "type": "bf16", "mask": "bits", "bias": "none", "train": False, "pad": 27},
        # the largest decoding batch
        {"name": "logits_batch_512", "op": "logits", "rows": 512, "vocab": 131072, "inner": 1, "history": 512, "type": "bf16", "mask": "bits", "bias": "none", "train": False, "pad": 0},
        # link scores of 20 graphs with 14 nodes and 10 commodities, with the gradient
        {"name": "links_train_14", "op": "logits", "rows": 280, "vocab": 14, "inner": 10, "history": 10, "type": "fp32", "mask": "bool", "bias": "period", "train": True, "pad": 0},
        # link scores of 4 graphs with 200 nodes and 100 commodities, with the gradient
        {"name": "links_train_200", "op": "logits", "rows": 800, "vocab": 200, "inner": 100, "history": 100, "type": "fp32", "mask": "bool", "bias": "period", "train": True, "pad": 0},
        # training on sampled tokens: every position of a few sequences, a learned bias shared by all rows
        {"name": "logits_train_tokens", "op": "logits", "rows": 2048, "vocab": 32000, "inner": 1, "history": 256, "type": "bf16", "mask": "bits", "bias": "shared", "train": True, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        kind = rng.choice(["gcn", "blocks", "ragged"])
        case = {"op": "adamw", "bits": rng.choice([32, 8]), "kind": kind, "type": rng.choice(["fp32", "bf16", "fp16"]), "clip": rng.random() < 0.5}
        if kind == "gcn":
            return {**case, "width": 4 * _log(rng, 2, 80), "layers": _log(rng, 2, 30), "many": _log(rng, 2, 100)}
        if kind == "blocks":
            return {**case, "width": _log(rng, 64, 1000), "layers": _log(rng, 1, 6), "many": _log(rng, 1000, 32000)}
        return {**case, "width": _log(rng, 100, 2000000), "layers": 1, "many": _log(rng, 1, 300)}
    if rng.random() < 0.4:
        graphs, nodes, flows = _log(rng, 1, 20), _log(rng, 3, 200), _log(rng, 1, 100)
        while graphs * nodes * nodes * flows > 16e6:
            graphs, flows = max(1, graphs // 2), max(1, flows // 2)
        return {"op": "logits", "rows": graphs * nodes, "vocab": nodes, "inner": flows, "history": flows, "type": "fp32",
                "mask": rng.choice(["none", "bool", "bits"]), "bias": rng.choice(["none", "shared", "period", "rows"]), "train": rng.random() < 0.7, "pad": 0}
    vocab = _log(rng, 500, 200000)
    train = rng.random() < 0.4
    rows = _log(rng, 1, max(2, min(2048, (60e6 if train else 64e6) // vocab)))
    return {"op": "logits", "rows": rows, "vocab": vocab, "inner": 1, "history": _log(rng, 1, 32768 if rows <= 32 else 2048), "type": rng.choice(["fp32", "bf16", "fp16"]),
            "mask": rng.choice(["none", "bool", "bits"]), "bias": rng.choice(["none", "shared", "rows"]), "train": train, "pad": rng.choice([0, 0, 3, 64])}


def _shapes(c):
    """The parameter tensors of a case."""
    w, n = c["width"], c["many"]
    if c["kind"] == "gcn":
        layer = [(w, w), (w,)] * 4 + [(w,)] * 4
        return [(3 * n, w // 2), (w // 2, 1), (w, 1)] + layer * c["layers"] + [(w, w), (w,), (2, w), (2,)]
    if c["kind"] == "blocks":
        return [(n, w)] + [(3 * w, w), (w, w), (4 * w, w), (w, 4 * w), (w,), (w,)] * c["layers"] + [(w,)]
    r = random.Random(n * 7919 + w)
    return [(max(1, int(round(math.exp(r.uniform(0.0, math.log(w)))))),) for _ in range(n)]


def _sizes(c):
    return [math.prod(s) for s in _shapes(c)]


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    return (_prepare_adamw if case["op"] == "adamw" else _prepare_logits)(case, seed)


def _flat(c, values, kind):
    """One buffer for all tensors of a case, each of them from a multiple of BLOCK elements on, and the tensors in it."""
    return _views(c, values.to(kind))


def _views(c, flat):
    starts = _starts(_sizes(c))
    return flat, [flat[o:o + math.prod(s)].view(s) for o, s in zip(starts, _shapes(c))]


def _starts(sizes):
    return list(itertools.accumulate((n + -n % BLOCK for n in sizes), initial=0))[:-1]


def _prepare_adamw(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    sizes, kind = _sizes(c), TYPES[c["type"]]
    padded = torch.tensor([n + -n % BLOCK for n in sizes], device=dev)
    total = int(padded.sum())
    place = torch.arange(total, device=dev) - torch.repeat_interleave(padded.cumsum(0) - padded, padded)
    inside = place < torch.repeat_interleave(torch.tensor(sizes, device=dev), padded)
    noise = lambda: torch.randn(total, device=dev, generator=gen) * inside  # noqa: E731
    # gradients of very different sizes, one in a hundred exactly zero (a unit that did not fire), weights of about 0.02
    size = torch.exp2(2 * noise() - 12)
    grad = noise() * size * (torch.rand(total, device=dev, generator=gen) > 0.01)
    weight, first, second = 0.02 * noise(), 0.3 * size * noise(), torch.square(size) * torch.exp2(0.5 * noise()) * inside
    s = {"case": c, "step": FIRST_STEP, "inside": inside}
    s["grad"], s["grads"] = _flat(c, grad, kind)
    s["param"], s["params"] = _flat(c, weight, kind)
    s["master"], s["masters"] = (None, None) if kind == torch.float32 else _flat(c, weight, torch.float32)
    if c["bits"] == 32:
        s["exp_avg"], s["exp_avgs"] = _flat(c, first, torch.float32)
        s["exp_avg_sq"], s["exp_avg_sqs"] = _flat(c, second, torch.float32)
        return s
    blocks = [-(-n // BLOCK) for n in sizes]
    for name, x in (("exp_avg", first), ("exp_avg_sq", second.sqrt())):
        codes, exps = _encode(x.view(-1, BLOCK), torch.zeros((), dtype=torch.int64, device=dev), name == "exp_avg_sq")
        s[name], s[name + "s"] = _views(c, codes.view(-1))
        s[name + "_exp"] = exps.view(-1)
        s[name + "_exps"] = list(s[name + "_exp"].split(blocks))
    return s


def _prepare_logits(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    rows, vocab, inner, length, kind = c["rows"], c["vocab"], c["inner"], c["history"], TYPES[c["type"]]
    rand = lambda *n: torch.rand(*n, device=dev, generator=gen)  # noqa: E731
    logits = 3 * torch.randn(rows, vocab, inner, device=dev, generator=gen)
    s = {"case": c, "masked": -1e9 if inner > 1 else -math.inf}
    if inner == 1:
        # common tokens come often; requests have contexts of their own lengths, a quarter of each is the prompt
        s["history"] = (vocab * rand(rows, length) ** 4).long().clamp_(0, vocab - 1)
        s["lens"] = (rand(rows) * (length + 1)).long().clamp_(0, length)
        s["prompts"] = s["lens"] // 4
        s["repetition"], s["presence"] = 1.0 + 0.5 * rand(rows), rand(rows) - 0.2
        s["frequency"], s["temperature"] = 0.4 * rand(rows), 0.5 + rand(rows)
    else:
        # the hops that earlier paths made from each node, -1 where a path did not pass
        s["history"] = torch.where(rand(rows, length) < 0.3, (vocab * rand(rows, length)).long().clamp_(0, vocab - 1), -1)
        s["lens"] = s["prompts"] = None
        s["repetition"], s["presence"], s["frequency"], s["temperature"] = 1.2, 0.1, 0.25, 0.9
    logits = logits.to(kind).view((rows, vocab) if inner == 1 else (rows, vocab, inner))
    if c["pad"]:
        logits = torch.nn.functional.pad(logits, (0, c["pad"]))[:, :vocab]
    s["logits"] = logits
    bias_rows = {"none": 0, "shared": 1, "period": vocab, "rows": rows}[c["bias"]]
    s["bias"] = torch.randn(bias_rows, vocab, device=dev, generator=gen) if bias_rows else None
    s["mask"] = None
    if c["mask"] != "none":
        # some rows allow a handful of tokens, some almost all, and one in sixteen nothing
        share = rand(rows, 1) ** 3
        share = torch.where(rand(rows, 1) < 1 / 16, torch.zeros_like(share), share)
        allowed = rand(rows, vocab) < share
        s["mask"] = allowed if c["mask"] == "bool" else _bits_of(allowed)
    s["grad"] = torch.randn(rows, vocab, inner, device=dev, generator=gen).to(kind).view(logits.shape) * 2.0 ** -8 if c["train"] else None
    return s


def _bits_of(allowed):
    """Truth values as 32-bit words, the lowest bit first."""
    rows, vocab = allowed.shape
    padded = torch.nn.functional.pad(allowed, (0, -vocab % 32)).view(rows, -1, 32).long()
    words = (padded << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _truth_of(mask, vocab):
    if mask.dtype == torch.bool:
        return mask
    bits = mask.long().unsqueeze(-1) >> torch.arange(32, device=mask.device)
    return (bits & 1).view(mask.shape[0], -1)[:, :vocab].bool()


# ---------------------------------------------------------------------------------------------------- 8-bit states, plain
def _blocks(tensors):
    """Tensors as rows of BLOCK elements, each tensor from a row of its own on, filled up with zeros."""
    sizes = [t.numel() for t in tensors]
    rows = torch.zeros(sum(n + -n % BLOCK for n in sizes), dtype=tensors[0].dtype, device=tensors[0].device)
    torch._foreach_copy_(_parts(rows, sizes), [t.view(-1) for t in tensors])
    return rows.view(-1, BLOCK)


def _parts(rows, sizes):
    return [p[:n] for p, n in zip(rows.view(-1).split([n + -n % BLOCK for n in sizes]), sizes)]


def _encode(x, random16, never_zero):
    """e4m3 codes and exponent bytes of rows of float32 values: x is about (the code's value) * 2^(byte - 127), and a row's
    largest value lands in [128, 256).  Stochastic rounding: random bits are added below the three mantissa bits that stay."""
    size = x.abs()
    bits = size.view(torch.int32)
    exps = ((torch.where(bits < 0x7F800000, bits, 0).amax(1, keepdim=True) >> 23) - 7).clamp(min=1)
    scaled = size * ((254 - exps) << 23).view(torch.float32)
    small = scaled < 2.0 ** -6                     # there the steps are 2^-9, those of the binade above 2^-6
    bits = torch.where(small, scaled + 2.0 ** -6, scaled).view(torch.int32).long()
    codes = (((bits + (random16 << 4)) >> 20) - torch.where(small, 968, 960)).clamp(0, 126)
    codes = torch.where((codes == 0) & (x > 0), 1, codes) if never_zero else torch.where(x < 0, codes + 128, codes)
    return codes.to(torch.uint8), exps.to(torch.uint8)


def _decode(codes, exps):
    return codes.view(torch.float8_e4m3fn).float() * (exps.int() << 23).view(torch.float32).view(-1, 1)


def _mix(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(sizes, step, device):
    """32 bits for each element of the padded rows: a hash of the seed, the step, the tensor's number and the element's."""
    key = _mix(_mix(_mix(_mix((SEED & 0xFFFFFFFF) ^ 0x9E3779B9) ^ (SEED >> 32)) ^ (step & 0xFFFFFFFF)) ^ (step >> 32))
    padded = torch.tensor([n + -n % BLOCK for n in sizes], device=device)
    keys = _mix(key ^ ((torch.arange(len(sizes), device=device) * 0x85EBCA6B) & 0xFFFFFFFF))
    total = sum(n + -n % BLOCK for n in sizes)
    place = torch.arange(total, device=device) - torch.repeat_interleave(padded.cumsum(0) - padded, padded, output_size=total)
    return _mix(torch.repeat_interleave(keys, padded, output_size=total) ^ place).view(-1, BLOCK)


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if state["case"]["op"] == "adamw":
        state["step"] += 1
        norm = (_own_adamw if own else _plain_adamw)(state)
        out = {k: state[k] for k in ("param", "master", "exp_avg", "exp_avg_sq") if state[k] is not None}
        if state["case"]["bits"] == 8:     # the values of the codes, and those of the scales
            out |= {k: state[k].view(torch.float8_e4m3fn) for k in ("exp_avg", "exp_avg_sq")}
            out |= {k: state[k].view(torch.float8_e8m0fnu) for k in ("exp_avg_exp", "exp_avg_sq_exp")}
        return out if norm is None else {**out, "norm": norm}
    return (_own_logits if own else _plain_logits)(state)


def _own_adamw(s):
    adamw, _ = _package()
    norm, coef = adamw.grad_norm(s["grads"], max_norm=MAX_NORM) if s["case"]["clip"] else (None, None)
    adamw.adamw_step_(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                      weight_decay=DECAY, masters=s["masters"], clip_coef=coef, exp_avg_exps=s.get("exp_avg_exps"),
                      exp_avg_sq_exps=s.get("exp_avg_sq_exps"), seed=SEED)
    return norm


def _plain_adamw(s):
    grads, norm = [g.float() for g in s["grads"]], None
    if s["case"]["clip"]:
        norm = torch.stack(torch._foreach_norm(grads)).square().sum().sqrt()
        grads = torch._foreach_mul(grads, (MAX_NORM / (norm + 1e-6)).clamp(max=1.0))
    weights = s["masters"] or s["params"]
    if s["case"]["bits"] == 32:
        first, second = s["exp_avgs"], s["exp_avg_sqs"]
    else:
        first = [_decode(_blocks(s["exp_avgs"]), torch.cat(s["exp_avg_exps"]))]
        second = [_decode(_blocks(s["exp_avg_sqs"]), torch.cat(s["exp_avg_sq_exps"])).square()]
        grads = [_blocks(grads)]
    torch._foreach_mul_(first, BETA1)
    torch._foreach_add_(first, torch._foreach_mul(grads, 1 - BETA1))
    torch._foreach_mul_(second, BETA2)
    squares = torch._foreach_mul(grads, grads)
    torch._foreach_mul_(squares, 1 - BETA2)
    torch._foreach_add_(second, squares)
    roots = torch._foreach_sqrt(second)
    below = torch._foreach_mul(roots, 1 / math.sqrt(1 - BETA2 ** s["step"]))
    torch._foreach_add_(below, EPS)
    change = torch._foreach_div(first, below)
    torch._foreach_mul_(change, -LR / (1 - BETA1 ** s["step"]))
    if s["case"]["bits"] == 8:
        bits = _random_bits([p.numel() for p in weights], s["step"], weights[0].device)
        for x, low, name in ((first[0], bits & 0xFFFF, "exp_avg"), (roots[0], bits >> 16, "exp_avg_sq")):
            codes, exps = _encode(x, low, name == "exp_avg_sq")
            torch._foreach_copy_([t.view(-1) for t in s[name + "s"]], _parts(codes, [t.numel() for t in s[name + "s"]]))
            torch._foreach_copy_(s[name + "_exps"], exps.view(-1).split([e.numel() for e in s[name + "_exps"]]))
        change = [x.view(p.shape) for x, p in zip(_parts(change[0], [p.numel() for p in weights]), weights)]
    torch._foreach_mul_(weights, 1 - LR * DECAY)
    torch._foreach_add_(weights, change)
    if s["masters"] is not None:
        torch._foreach_copy_(s["params"], weights)
    return norm


def _own_logits(s):
    _, logits = _package()
    rules = dict(dim=1, history=s["history"], history_lens=s["lens"], prompt_lens=s["prompts"], repetition_penalty=s["repetition"],
                 presence_penalty=s["presence"], frequency_penalty=s["frequency"], mask=s["mask"], temperature=s["temperature"], masked_value=s["masked"])
    if s["grad"] is None:
        return logits.process_logits(s["logits"], bias=s["bias"], **rules)
    x, b = s["logits"].detach().requires_grad_(), None if s["bias"] is None else s["bias"].detach().requires_grad_()
    out = logits.process_logits(x, bias=b, **rules)
    return [out.detach(), *torch.autograd.grad(out, [x] if b is None else [x, b], s["grad"])]


def _column(value):
    """A number, or one for each row, against [rows, vocabulary, inner]."""
    return value.view(-1, 1, 1) if isinstance(value, torch.Tensor) else value


def _counts(s, rows, vocab):
    """How often each token stands in each row's history: anywhere, and behind the prompt."""
    ids, place = s["history"], torch.arange(s["history"].shape[1], device=s["history"].device)
    valid = (ids >= 0) & (ids < vocab)
    valid = valid if s["lens"] is None else valid & (place < s["lens"].view(-1, 1))
    after = valid if s["prompts"] is None else valid & (place >= s["prompts"].view(-1, 1))
    ids, zero = torch.where(valid, ids, 0), torch.zeros(rows, vocab, device=ids.device)
    return zero.scatter_add(1, ids, valid.float()).unsqueeze(2), zero.scatter_add(1, ids, after.float()).unsqueeze(2)


def _plain_logits(s):
    c = s["case"]
    rows, vocab, inner = c["rows"], c["vocab"], c["inner"]
    x = s["logits"].view(rows, vocab, -1).float() if inner == 1 else s["logits"].float()
    rho, tau = _column(s["repetition"]), _column(s["temperature"])
    every, new = _counts(s, rows, vocab)
    seen, up = every > 0, x > 0
    y = torch.where(seen, torch.where(up, x / rho, x * rho), x)
    y = y - new * _column(s["frequency"]) - (new > 0) * _column(s["presence"])
    if s["bias"] is not None:
        y = y + s["bias"].repeat(rows // s["bias"].shape[0], 1).unsqueeze(2)
    y = y / tau
    allowed = None if s["mask"] is None else _truth_of(s["mask"], vocab).unsqueeze(2)
    if allowed is not None:
        y = torch.where(allowed, y, s["masked"])
    y = y.to(s["logits"].dtype).view(s["logits"].shape)
    if s["grad"] is None:
        return y
    g = s["grad"].view(rows, vocab, inner).float() / tau
    g = g if allowed is None else torch.where(allowed, g, 0.0)
    dx = torch.where(seen, torch.where(up, g / rho, g * rho), g).to(s["logits"].dtype).view(s["logits"].shape)
    if s["bias"] is None:
        return [y, dx]
    return [y, dx, g.view(-1, s["bias"].shape[0], vocab, inner).sum((0, 3))]


def work(case):
    c = case
    if c["op"] == "adamw":
        n, half = sum(_sizes(c)), TYPES[c["type"]].itemsize == 2
        state = 2 * (4 if c["bits"] == 32 else 1 + 1 / BLOCK)
        # the weights (in 16 bits: the master copy, and the parameter that is written), the gradient, both states in and out
        return {"bytes": n * ((4 + 4 + 2 + 2 if half else 4 + 4 + 4) + 2 * state), "flops": n * 16}
    n, size = c["rows"] * c["vocab"] * c["inner"], TYPES[c["type"]].itemsize
    more = c["rows"] * c["history"] * 8 + c["rows"] * c["vocab"] * {"none": 0, "bool": 1, "bits": 1 / 8}[c["mask"]]
    more += {"none": 0, "shared": 1, "period": c["vocab"], "rows": c["rows"]}[c["bias"]] * c["vocab"] * 4
    return {"bytes": (2 if c["train"] else 1) * (2 * n * size + more), "flops": n * (12 if c["train"] else 6)}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    return (_exact_adamw if case["op"] == "adamw" else _exact_logits)(case, seed)


def _exact_codes(x, random16, never_zero):
    """The codes' values and the scales by the definition: a value between two neighbours goes to the upper one if its
    distance from the lower one and the random number, in steps between them, together reach a step."""
    largest = x.abs().amax(1, keepdim=True)
    top = torch.where(largest > 0, torch.floor(torch.log2(largest)), -200.0).clamp(min=-119.0)
    scaled = x.abs() * torch.exp2(7 - top)
    step = torch.exp2(torch.floor(torch.log2(scaled.clamp(min=2.0 ** -6))) - 3)
    low = torch.floor(scaled / step)
    value = (low + ((scaled / step - low) + random16 / 65536 >= 1)) * step
    value = torch.where((value == 0) & (x > 0), 2.0 ** -9, value) if never_zero else value * torch.sign(x)
    return value.view(-1), torch.exp2(top - 7).view(-1)


def _exact_adamw(c, seed):
    s, kept = _prepare_adamw(c, seed), {}
    step, g = s["step"] + 1, s["grad"].double()
    if c["clip"]:
        kept["norm"] = (g * g).sum().sqrt()
        g = g * min(1.0, MAX_NORM / (float(kept["norm"]) + 1e-6))
    if c["bits"] == 32:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        e4m3 = torch.tensor([(-1.0) ** (k >> 7) * (2.0 ** ((k >> 3 & 15) - 10) * (8 + (k & 7)) if k & 0x78 else 2.0 ** -9 * (k & 7)) for k in range(256)],
                            dtype=torch.float64, device=g.device)
        value = lambda name: (e4m3[s[name].int()].view(-1, BLOCK) * torch.exp2(s[name + "_exp"].double() - 127).view(-1, 1)).view(-1)  # noqa: E731
        m, v = value("exp_avg"), value("exp_avg_sq") ** 2
    m, v = m + (1 - BETA1) * (g - m), v + (1 - BETA2) * (g * g - v)
    p = (s["param"] if s["master"] is None else s["master"]).double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** step)) / ((v / (1 - BETA2 ** step)).sqrt() + EPS)
    p = torch.where(s["inside"], p, 0.0)
    kept |= {"param": p, "exp_avg": m, "exp_avg_sq": v}
    if s["master"] is not None:
        kept["master"] = p
    if c["bits"] == 8:
        bits = _random_bits(_sizes(c), step, g.device)
        for name, x, low in (("exp_avg", m, bits & 0xFFFF), ("exp_avg_sq", v.sqrt(), bits >> 16)):
            kept[name], kept[name + "_exp"] = _exact_codes(x.view(-1, BLOCK), low, name == "exp_avg_sq")
    return kept


def _exact_logits(c, seed):
    s = _prepare_logits(c, seed)
    rows, vocab, inner = c["rows"], c["vocab"], c["inner"]
    x = s["logits"].double().reshape(rows, vocab, inner)
    number = lambda v: v.double().view(-1, 1, 1) if isinstance(v, torch.Tensor) else v  # noqa: E731
    rho, tau = number(s["repetition"]), number(s["temperature"])
    ids, length = s["history"], c["history"]
    place = torch.arange(length, device=ids.device).expand(rows, length)
    used = ids >= 0 if s["lens"] is None else place < s["lens"].unsqueeze(1)
    after = used if s["prompts"] is None else used & (place >= s["prompts"].unsqueeze(1))
    cell = ids + vocab * torch.arange(rows, device=ids.device).unsqueeze(1)
    seen = torch.bincount(cell[used], minlength=rows * vocab).view(rows, vocab, 1) > 0
    new = torch.bincount(cell[after], minlength=rows * vocab).view(rows, vocab, 1)
    slope = torch.where(seen, torch.where(x > 0, 1.0 / rho, 1.0 * rho), 1.0 + 0.0 * x) / tau
    y = x * slope
    y -= (number(s["frequency"]) * new + number(s["presence"]) * (new > 0).double()) / tau
    if s["bias"] is not None:
        y += (s["bias"].double().repeat(rows // s["bias"].shape[0], 1).unsqueeze(2)) / tau
    off = torch.zeros(rows, vocab, 1, dtype=torch.bool, device=x.device) if s["mask"] is None else ~_truth_of(s["mask"], vocab).unsqueeze(2)
    y = y.masked_fill(off, s["masked"]).view(s["logits"].shape)
    if s["grad"] is None:
        return y
    g = s["grad"].double().view(rows, vocab, inner).masked_fill(off, 0.0)
    dx = (g * slope).view(s["logits"].shape)
    if s["bias"] is None:
        return [y, dx]
    dbias = (g / tau).view(-1, s["bias"].shape[0], vocab, inner).sum(3).sum(0)
    return [y, dx, dbias]
