"""Rules on logits and their gradient in double precision (numpy, row by row), from the formulas in include/gcn_uelb_hip.h."""
import numpy as np


def _pick(value, o):
    a = np.asarray(value, dtype=np.float64).reshape(-1)
    return a[o % a.size]


def process(x, history=None, lens=None, prompts=None, rho=1.0, alpha_p=0.0, alpha_f=0.0, bias=None, mask=None, tau=1.0, masked=-np.inf):
    """x [rows, vocab, inner]; history [R, L], lens / prompts [R], bias [R, vocab], mask bool [R, vocab], numbers or [R].
    Returns (y, slope dy/dx, dy/dbias [rows, vocab], bound): bound adds the magnitudes that enter y, for error estimates."""
    x = np.asarray(x, dtype=np.float64)
    rows, vocab, inner = x.shape
    y, slope, slope_b, bound = np.empty_like(x), np.empty_like(x), np.empty((rows, vocab)), np.empty_like(x)
    for o in range(rows):
        n, seen = np.zeros(vocab), np.zeros(vocab, dtype=bool)
        if history is not None:
            r = o % history.shape[0]
            length = history.shape[1] if lens is None else min(max(int(lens[r]), 0), history.shape[1])
            start = 0 if prompts is None else int(prompts[r])
            for place in range(length):
                v = int(history[r, place])
                if 0 <= v < vocab:
                    seen[v] = True
                    n[v] += place >= start
        p, f, t, c = _pick(alpha_p, o), _pick(alpha_f, o), _pick(tau, o), _pick(rho, o)
        s = np.where(seen[:, None], np.where(x[o] > 0, 1 / c, c), 1.0)
        cut = (n * f + (n > 0) * p)[:, None]
        b = 0.0 if bias is None else np.asarray(bias, dtype=np.float64)[o % len(bias)][:, None]
        with np.errstate(invalid="ignore"):
            y[o] = (x[o] * s - cut + b) / t
            bound[o] = (np.abs(x[o] * s) + np.abs(n * f)[:, None] + np.abs(p) * (n > 0)[:, None] + np.abs(b)) / t
        slope[o], slope_b[o] = s / t, 1 / t
        if mask is not None:
            off = ~mask[o % len(mask)]
            y[o][off], slope[o][off], slope_b[o][off], bound[o][off] = masked, 0, 0, 0
    return y, slope, slope_b, bound


def gradient(dy, slope, slope_b, bias_rows):
    """(dx, dbias, magnitude of dbias' terms)."""
    rows, vocab, inner = dy.shape
    with np.errstate(invalid="ignore"):
        dx = np.where(slope == 0, 0.0, dy * slope)
        terms = np.where(slope_b[:, :, None] == 0, 0.0, dy * slope_b[:, :, None])
    per = terms.reshape(rows // bias_rows, bias_rows, vocab, inner)
    return dx, per.sum((0, 3)), np.abs(per).sum((0, 3))
