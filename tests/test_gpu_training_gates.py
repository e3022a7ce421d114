"""Open gates of the minGRU recurrence (boa_b200.training): what is left of
the old state, a = 1 - z, and the gate's gradient, which is proportional to it,
against 64 bits within bounds that are relative to a.

With k the relative error of the gate and candidate of training_ref.py (twice
that of the exponentials, and 20 roundings): e = exp(-zl) has at most k / 2, and
so has z, so a = e z has k for zl >= 0; for zl < 0, a >= 1/2 >= z, and the
difference 1 - z has it too.  Below 2^-126 the exponential may come out as 0."""
import numpy as np
import pytest

import training_ref as R

pytestmark = pytest.mark.gpu

DT = ["float32", "float16", "bfloat16"]
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


def _bounds(zh, h0, dh, dlast):
    """Bounds on h, last, dzh and dh0; every position is a chunk's."""
    B, T, w = zh.shape
    d = w // 2
    z, a, c, hr, k = R._cell(zh, np.ones((B, T, 1), bool))
    h, size, err = np.zeros((T + 1, B, d)), np.zeros((T + 1, B, d)), np.zeros((T + 1, B, d))
    h[0], size[0] = h0, np.abs(h0)
    for t in range(T):
        h[t + 1] = a[:, t] * h[t] + z[:, t] * c[:, t]
        size[t + 1] = a[:, t] * size[t] + z[:, t] * np.abs(c[:, t])
        err[t + 1] = a[:, t] * err[t] + 2 * k[:, t] * size[t + 1] + TINY * size[t]
    g, gs, ge = dlast.copy(), np.abs(dlast), np.zeros((B, d))
    tol = np.zeros((B, T, w))
    for t in range(T - 1, -1, -1):
        kt, zt, at = k[:, t], z[:, t], a[:, t]
        gs = gs + np.abs(dh[:, t])
        ge = ge + kt * gs
        cp = np.where(hr[:, t] >= 0, 1.0, c[:, t] * (1 - c[:, t]))
        near = ge + 4 * kt * gs
        tol[:, t, :d] = zt * ((np.abs(c[:, t]) + size[t]) * ((at + TINY) * near + TINY * gs) + at * gs * err[t])
        tol[:, t, d:] = zt * cp * near
        gs, ge = at * gs, at * ge + kt * at * gs + TINY * gs
    return err[1:].transpose(1, 0, 2), err[T], tol, ge


def _close(got, ref, err, dtype, what):
    got = got.double().cpu().numpy()
    off, tol = np.abs(got - ref), R.stored(ref, err, dtype)
    assert (off <= tol).all(), f"{what}: {np.max(off / tol):.3g} times the bound, at {np.argwhere(off > tol)[0]}"


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lo,hi", [(0.0, 4.0), (8.0, 14.0), (14.0, 20.0), (20.0, 40.0), (60.0, 95.0), (-3.0, 20.0)])
@pytest.mark.parametrize("B,T,d", [(2, 1, 40), (3, 8, 33), (2, 300, 64), (150, 40, 64), (1, 2000, 24)])
def test_open_gates(tr, dtype, lo, hi, B, T, d):
    import torch
    rng = np.random.default_rng(T + int(hi))
    t = lambda x, k=dtype: torch.from_numpy(x.astype(np.float32)).cuda().to(getattr(torch, k))  # noqa: E731
    n = lambda x: x.double().cpu().numpy()  # noqa: E731
    zh = t(np.concatenate([rng.uniform(lo, hi, (B, T, d)), rng.normal(size=(B, T, d))], 2))
    dh, dl, h0 = t(rng.normal(size=(B, T, d)) * 64), t(rng.normal(size=(B, d)), "float32"), t(rng.normal(size=(B, d)), "float32")
    h, last, saved = tr.mingru_scan(zh, h0, save_states=True)
    dzh, dh0 = tr.mingru_scan_backward(zh, saved, dh, dl)
    ref = R.mingru(n(zh), n(h0), None, n(dh), n(dl))
    eh, el, ez, e0 = _bounds(n(zh), n(h0), n(dh), n(dl))
    _close(h, ref["h"][0], eh, dtype, "h")
    _close(last, ref["last"][0], el, "float32", "h_last")
    _close(dzh, ref["dzh"][0], ez, dtype, "dzh")
    _close(dh0, ref["dh0"][0], e0, "float32", "dh0")


def test_open_gates_have_a_gradient(tr):
    """One position, no state: dzl = z a c, which fp32 holds down to e^-87."""
    import torch
    zl = np.linspace(0.0, 80.0, 161)
    zh = torch.from_numpy(np.concatenate([zl, np.ones(161)]).astype(np.float32)).cuda().view(1, 1, -1)
    _, _, saved = tr.mingru_scan(zh, save_states=True)
    dzh, _ = tr.mingru_scan_backward(zh, saved, torch.ones(1, 1, 161, device="cuda"))
    got, want = dzh[0, 0, :161].double().cpu().numpy(), 1.5 * R.sigmoid(zl) * R.sigmoid(-zl)
    assert (np.abs(got - want) <= (4 * R.exp_err(zl) + 40 * R.U) * want).all()


@pytest.mark.parametrize("T", [5, 500])
def test_closed_gates_keep_the_state_exactly(tr, T):
    """Gates below -17 add nothing to a state of 1, position after position."""
    import torch
    zh = torch.cat((torch.linspace(-200, -20, 64, device="cuda"), torch.zeros(64, device="cuda"))).expand(2, T, 128)
    one = torch.ones(2, 64, device="cuda")
    h, last, saved = tr.mingru_scan(zh, one, save_states=True)
    _, dh0 = tr.mingru_scan_backward(zh, saved, torch.zeros(2, T, 64, device="cuda"), one)
    assert (dh0 == 1).all()  # the product of a: 1 - z rounds to 1
    assert (last - 1).abs().max().item() <= T * 2.1e-9 + 2.0 ** -23 and torch.equal(h[:, -1], last)
