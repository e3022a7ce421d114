"""Plain 64-bit forms of the training operators (numpy), with bounds on what
fp32 arithmetic may be off by, used by the tests of boa_b200.training.

The bounds are running error bounds: each is evaluated next to the value, from
the documented errors of what the kernels call (u = 2^-24, half a step of
fp32): ex2.approx 2 steps of 2^-23 and rcp.approx 1, logf 1 step, one u for
each product and sum.  exp(x) is ex2 of x times log2 e, whose constant and
product are off by one u each: |x| (2 u) more, below the 1.173 |x| steps of
2^-23 that are allowed for.  They hold for any order of the sums and any grouping of the
recurrence.  What an open gate leaves of the state is bounded more closely in
test_gpu_training_gates.py."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
# half the spacing of the smallest numbers: what rounding costs below the normal range
FLOOR = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def stored(ref, err, dtype):
    """Bound on a stored value: the error before rounding, and half a step."""
    return err + HALF_STEP[dtype] * (np.abs(ref) + err) + FLOOR[dtype]


def sigmoid(x):
    with np.errstate(over="ignore"):
        return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def exp_err(x):
    x = np.abs(np.where(np.isfinite(x), x, 0.0))
    return (2 + 1.173 * x) * 2 * U


def embed(tok, table, scale):
    ok = (tok >= 0) & (tok < len(table))
    out = np.where(ok[:, None], table[np.where(ok, tok, 0)] * scale, 0.0)
    return out, U * np.abs(out)


def embed_grad(tok, dout, vocab, scale):
    ok = (tok >= 0) & (tok < vocab)
    out, size = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1]))
    np.add.at(out, tok[ok], dout[ok])
    np.add.at(size, tok[ok], np.abs(dout[ok]))
    # at most 768 additions one after the other in fp32: the rows of a piece (128 in calls of this size), the
    # groups of a block and the pieces of a token (at most 256 each)
    return out * scale, (768 * U) * size * abs(scale) + 2 * U * np.abs(out * scale)


def _cell(zh, live):
    d = zh.shape[2] // 2
    zl, hr = np.where(live, zh[..., :d], 0.0), np.where(live, zh[..., d:], 0.0)
    z, a = sigmoid(zl), sigmoid(-zl)
    c = np.where(hr >= 0, hr + 0.5, sigmoid(hr))
    k = exp_err(zl) * 2 + exp_err(np.where(hr >= 0, 0.0, hr)) + 20 * U  # z, a and c together, and four roundings
    return np.where(live, z, 0.0), np.where(live, a, 1.0), c, hr, k


def mingru(zh, h0, lengths, dh=None, dlast=None):
    """-> dict of (value, bound) of h, last and, with dh, of dzh and dh0."""
    B, T, w = zh.shape
    d = w // 2
    n = np.full(B, T) if lengths is None else np.clip(lengths, 0, T)
    live = (np.arange(T)[None, :] < n[:, None])[:, :, None]
    z, a, c, hr, k = _cell(zh, live)
    k = np.where(live, k, 0.0)
    h = np.zeros((T + 1, B, d))
    size, err = np.zeros_like(h), np.zeros_like(h)
    h[0], size[0] = h0, np.abs(h0)
    for t in range(T):
        h[t + 1] = a[:, t] * h[t] + z[:, t] * c[:, t]
        size[t + 1] = a[:, t] * size[t] + z[:, t] * np.abs(c[:, t])
        # a's error is taken as that of 1 - z, not relative to a
        err[t + 1] = a[:, t] * err[t] + k[:, t] * (size[t + 1] + z[:, t] * size[t])
    out = np.where(live, h[1:].transpose(1, 0, 2), 0.0)
    got = {"h": (out, np.where(live, err[1:].transpose(1, 0, 2), 0.0)), "last": (h[T], err[T])}
    if dh is None:
        return got
    g, gs, ge = dlast.astype(np.float64), np.abs(dlast).astype(np.float64), np.zeros((B, d))
    dzh, tol = np.zeros((B, T, 2 * d)), np.zeros((B, T, 2 * d))
    for t in range(T - 1, -1, -1):
        on = live[:, t]
        g = g + np.where(on, dh[:, t], 0.0)
        gs = gs + np.where(on, np.abs(dh[:, t]), 0.0)
        ge = ge + np.where(on, k[:, t] * gs, 0.0)
        cp = np.where(hr[:, t] >= 0, 1.0, c[:, t] * (1 - c[:, t]))
        near, zt, at = ge + 4 * k[:, t] * gs, z[:, t], a[:, t]
        dzh[:, t, :d] = np.where(on, g * zt * at * (c[:, t] - h[t]), 0.0)
        tol[:, t, :d] = np.where(on, zt * ((np.abs(c[:, t]) + size[t]) * (at * near + k[:, t] * gs) + at * gs * err[t]), 0.0)
        dzh[:, t, d:] = np.where(on, g * zt * cp, 0.0)
        tol[:, t, d:] = np.where(on, zt * cp * near, 0.0)
        g, gs, ge = at * g, at * gs, at * ge + k[:, t] * (at + np.where(on, zt, 0.0)) * gs
    return {**got, "dzh": (dzh, tol), "dh0": (g, ge)}


def token_loss(x, tok, inv_t, w):
    """-> (loss, bound), (gradient, bound); w = grad_scale * dloss per row."""
    rows, V = x.shape
    ok = (tok >= 0) & (tok < V)
    t = np.where(ok, tok, 0)
    x = np.where(ok[:, None], x, 0.0)
    m = x.max(axis=1, keepdims=True)
    none = np.isneginf(m)
    y = (x - np.where(none, 0.0, m)) * inv_t
    e = np.exp(y)
    s = e.sum(axis=1, keepdims=True)
    yf = np.where(np.isfinite(y), np.abs(y), 0.0)
    ke = exp_err(y) + 2 * U * yf
    ks = (np.where(e > 0, e * ke, 0.0).sum(axis=1, keepdims=True) / np.where(none, 1.0, s)) + 40 * U
    # an exponential below 2^-126 may come out as 0
    p = e / np.where(none, 1.0, s)
    yt = np.take_along_axis(y, t[:, None], 1)[:, 0]
    with np.errstate(divide="ignore", invalid="ignore"):
        loss = np.where(ok, np.where(none[:, 0], np.inf, np.log(s)[:, 0] - yt), 0.0)
    lerr = ks[:, 0] + 2 * U * np.abs(np.log(np.where(none, 1.0, s)))[:, 0] + 4 * U * np.where(np.isfinite(yt), np.abs(yt), 0.0)
    hot = np.zeros_like(p)
    hot[np.arange(rows), t] = 1.0
    c = (w * inv_t)[:, None]
    live = ok[:, None] & ~none
    grad = np.where(live, c * (p - hot), 0.0)
    gerr = np.where(live, np.abs(c) * (p * (ke + ks + 6 * U) + 4 * U * hot + 2.0 ** -125), 0.0)
    return (loss, np.where(ok, lerr + U * np.where(np.isfinite(loss), np.abs(loss), 0.0), 0.0)), (grad, gerr)
