"""Plain numpy / float64 restatement of the operators on logits and gradients, and how far an f32 evaluation may be from it -- TEST
INFRASTRUCTURE of test_policy_ops_cpu.py and test_gpu_policy_ops.py."""
import numpy as np

E32 = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}     # finfo.eps / 2
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}       # below it a rounding (or a flush of the exponential) is absolute


def legal(mask, rows, width):
    """bits [rows or 1, nb] -> bool [rows, width]; None: everything"""
    if mask is None:
        return np.ones((rows, width), bool)
    m = np.asarray(mask)
    m = m.reshape(-1, m.shape[-1])
    v = np.arange(width)
    return np.broadcast_to((m[:, v >> 3] >> (v & 7)) & 1 == 1, (rows, width))


def pack(keep):
    keep = np.asarray(keep, bool)
    return np.packbits(keep, axis=1, bitorder="little")


def process(x, mask=None, bias=None, history=None, history_len=None, penalties=None):
    """-> (y, tol): tol bounds an f32 evaluation before its last rounding -- every one of the <= 6 operations is off by at most half a
    step of its own result, and no intermediate is larger than the sum of the terms' magnitudes"""
    x = np.asarray(x, np.float64)
    rows, width = x.shape
    ok = legal(mask, rows, width)
    y = np.where(ok, x, 0.0)
    mag = np.abs(y)
    if history is not None:
        h = np.asarray(history)
        h = np.broadcast_to(h if h.ndim == 2 else h[None], (rows, h.shape[-1]))
        p = np.broadcast_to(np.asarray(penalties, np.float64).reshape(-1, 3), (rows, 3))
        for r in range(rows):
            n = h.shape[1] if history_len is None else min(max(int(history_len[r]), 0), h.shape[1])
            ids = h[r, :n].astype(np.int64)
            ids = ids[(ids >= 0) & (ids < width)]
            c = np.bincount(ids, minlength=width).astype(np.float64)
            rep, freq, pres = p[r]
            hit = c > 0
            scaled = np.where(y[r] > 0, y[r] / rep, y[r] * rep)
            off = freq * c + pres
            mag[r] = np.where(hit, np.abs(scaled) + np.abs(freq * c) + np.abs(pres), mag[r])
            y[r] = np.where(hit, scaled - off, y[r])
    if bias is not None:
        b = np.asarray(bias, np.float64)
        y = y + b
        mag = mag + np.abs(b)
    with np.errstate(invalid="ignore"):
        return np.where(ok, y, -np.inf), np.where(ok, 6 * E32 * mag, 0.0)


def weights(targets, rows, width):
    t = np.asarray(targets)
    if t.ndim == 2:
        return t.astype(np.float64)
    w = np.zeros((rows, width))
    for r in range(rows):
        if 0 <= t[r] < width:
            w[r, int(t[r])] = 1.0
    return w


def loss(x, targets, mask=None, scale=1.0):
    """-> dict(loss, lse, total, grad) and their tolerances (f32, before the last rounding of the gradient).
    exp: the argument is off by <= 2 half steps of |x - m|, the function by <= 4; the sum of n terms, none negative, by <= (n / 64 + 16)
    half steps of itself (a lane's share one after the other, then a tree); so p by <= rel = (2 |x - m| + n / 64 + 24) half steps, log s by
    the same absolute amount with the weighted mean of |x - m| exp(x - m) <= 0.37 n / s <= 0.37 n in place of |x - m| ... bounded by the largest
    term's, 1 each: n / 64 + 24.  The loss is total * log s + sum t (m - x): terms >= 0, each off by <= 2 half steps, summed likewise."""
    x = np.asarray(x, np.float64)
    rows, width = x.shape
    ok = legal(mask, rows, width)
    w = np.where(ok, weights(targets, rows, width), 0.0)
    n = width / 64 + 24
    out = {k: np.zeros(rows) for k in ("loss", "lse", "total")}
    tol = {k: np.zeros(rows) for k in ("loss", "lse", "total")}
    out["grad"], tol["grad"] = np.zeros((rows, width)), np.zeros((rows, width))
    scale = np.broadcast_to(np.asarray(scale, np.float64), (rows,))
    with np.errstate(all="ignore"):
        for r in range(rows):
            y = x[r][ok[r]]
            if y.size == 0 or not (np.isnan(y).any() or y.max() > -np.inf):
                out["lse"][r] = -np.inf
                continue
            m = y.max()
            s = np.exp(y - m).sum()
            q = w[r][ok[r]]
            gap = np.where(q == 0, 0.0, q * (m - y))
            out["lse"][r] = m + np.log(s)
            out["total"][r] = q.sum()
            out["loss"][r] = q.sum() * np.log(s) + gap.sum()
            p = np.exp(y - m) / s
            out["grad"][r][ok[r]] = scale[r] * (q.sum() * p - q)
            tol["lse"][r] = E32 * (n + 4 * abs(m) + 4 * abs(np.log(s)))
            tol["total"][r] = E32 * n * q.sum()
            tol["loss"][r] = E32 * (n * (q.sum() * (1 + np.log(s)) + gap.sum()) + 4 * abs(out["loss"][r]))
            tol["grad"][r][ok[r]] = abs(scale[r]) * E32 * (q.sum() * p * (2 * np.where(p > 0, m - y, 0) + 2 * n) + 4 * q)
    return out, tol


def grad_from(x, targets, lse, total, dloss, mask=None):
    """the backward pass alone: lse and total are inputs as they stand (f32).  -> (grad, tol): exp's argument is off by <= 3 half steps of
    |x| + |lse|, the rest by <= 8"""
    x = np.asarray(x, np.float64)
    rows, width = x.shape
    lse, total = np.asarray(lse, np.float64), np.asarray(total, np.float64)
    dloss = np.broadcast_to(np.asarray(dloss, np.float64), (rows,))
    some = (lse > -np.inf) | np.isnan(lse)
    ok = legal(mask, rows, width) & some[:, None]
    w = np.where(ok, weights(targets, rows, width), 0.0)
    with np.errstate(all="ignore"):
        z = np.where(some, lse, 0.0)[:, None]
        p = np.where(ok, np.exp(x - z), 0.0)
        g = np.where(ok, dloss[:, None] * (total[:, None] * p - w), 0.0)
        t = np.abs(dloss)[:, None] * E32 * (total[:, None] * p * (3 * (np.where(p > 0, np.abs(x), 0) + np.abs(z)) + 8) + 4 * w)
    return g, np.where(ok, t, 0.0)


def near(got, want, tol, kind, what=""):
    """got (values of type `kind`) within tol plus the half step of its own rounding of want; infinities and NaN where they belong"""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    big = {"f32": np.finfo(np.float32).max, "f16": 65504.0, "bf16": 3.3895e38}[kind]
    over = np.abs(want) > big * (1 - 2 * HALF_STEP[kind])        # may round to infinity
    fine = np.isfinite(want) & ~over
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN", int(np.isnan(got).sum()), int(np.isnan(want).sum()))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), (what, "infinities")
    assert (np.abs(got[over & ~inf]) >= big * (1 - 4 * HALF_STEP[kind])).all(), what
    assert np.isfinite(got[fine]).all(), (what, "not finite")
    tol = np.broadcast_to(tol, want.shape)[fine]
    err, lim = np.abs(got[fine] - want[fine]), tol + HALF_STEP[kind] * (np.abs(want[fine]) + tol) + TINY[kind]
    if err.size:
        k = int(np.argmax(err / lim))
        assert err[k] <= lim[k], (what, float(err[k]), float(lim[k]), float(got[fine][k]), float(want[fine][k]))
