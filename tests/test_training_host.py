"""Refusals of the training operators (no GPU: every check comes before the
launch), and the plain forms that their GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import training_ref as R

A = C.c_void_p(256)  # an aligned address; refused calls never read it


def _embed(L, tok_t=0, n=8, tab_t=0, ld_t=16, vocab=256, d=16, out_t=0, ld_o=16, p=(A, A, A)):
    return L.boa_embed(p[0], tok_t, n, p[1], tab_t, ld_t, vocab, d, 1.0, p[2], out_t, ld_o, None)


def _embed_bwd(L, tok_t=0, n=9000, g_t=0, ld_g=16, vocab=256, d=16, t_t=0, ld_t=16, p=(A, A, A, A), ws=None):
    ws = L.boa_embed_backward_workspace(n, vocab, d) if ws is None else ws
    return L.boa_embed_backward(p[0], tok_t, n, p[1], g_t, ld_g, vocab, d, 1.0, 0, p[2], t_t, ld_t, p[3], ws, None)


def _scan(L, t=0, zr=32, zc=320, B=4, T=10, d=16, hr=16, hc=160, zh=A, h=A, h0=None):
    return L.boa_mingru_scan(zh, t, zr, zc, B, T, d, None, h0, h, hr, hc, None, None, None)


def _scan_bwd(L, t=0, zr=32, zc=320, B=4, T=10, d=16, gr=16, gc=160, dr=32, dc=320, p=(A, A, A, A)):
    return L.boa_mingru_scan_backward(p[0], t, zr, zc, B, T, d, None, p[1], p[2], gr, gc, None, p[3], dr, dc, None,
                                      None)


def _loss(L, t=0, ld=256, rows=8, vocab=256, tok_t=0, inv=1.0, ld_g=256, p=(A, A, A, C.c_void_p(512))):
    return L.boa_token_loss(p[0], t, ld, rows, vocab, p[1], tok_t, inv, None, 1.0, p[2], p[3], ld_g, None)


odd = C.c_void_p(257)
REFUSED = [
    (_embed, dict(tok_t=3)), (_embed, dict(tab_t=-1)), (_embed, dict(out_t=3)), (_embed, dict(n=-1)),
    (_embed, dict(n=1 << 31)), (_embed, dict(vocab=0)), (_embed, dict(vocab=1025)), (_embed, dict(d=0)),
    (_embed, dict(d=65537, ld_t=70000, ld_o=70000)), (_embed, dict(ld_t=15)), (_embed, dict(ld_o=15)),
    (_embed, dict(ld_o=1 << 31)), (_embed, dict(p=(None, A, A))), (_embed, dict(p=(A, None, A))),
    (_embed, dict(p=(A, A, None))), (_embed, dict(tok_t=2, p=(C.c_void_p(260), A, A))),
    (_embed, dict(p=(A, odd, A))), (_embed, dict(out_t=2, p=(A, A, odd))),
    (_embed_bwd, dict(tok_t=-1)), (_embed_bwd, dict(g_t=7)), (_embed_bwd, dict(t_t=7)), (_embed_bwd, dict(n=-1)),
    (_embed_bwd, dict(vocab=1025)), (_embed_bwd, dict(d=0)), (_embed_bwd, dict(ld_g=15)), (_embed_bwd, dict(ld_t=15)),
    (_embed_bwd, dict(p=(None, A, A, A))), (_embed_bwd, dict(p=(A, None, A, A))),
    (_embed_bwd, dict(p=(A, A, None, A))), (_embed_bwd, dict(p=(A, A, A, None))),
    (_embed_bwd, dict(p=(A, A, A, C.c_void_p(264)))), (_embed_bwd, dict(ws=64)), (_embed_bwd, dict(n=0, p=(A, A, None, A))),
    (_scan, dict(t=3)), (_scan, dict(B=-1)), (_scan, dict(T=-1)), (_scan, dict(d=0)), (_scan, dict(d=65537)),
    (_scan, dict(B=1 << 20, d=4096)), (_scan, dict(zr=-1)), (_scan, dict(zc=1 << 60)), (_scan, dict(zr=1 << 30)), (_scan, dict(t=2, zr=1 << 31)), (_scan, dict(T=(1 << 30) + 1)), (_scan, dict(hr=15)),
    (_scan, dict(hc=150)), (_scan, dict(zh=None)), (_scan, dict(h=None)), (_scan, dict(zh=odd)),
    (_scan, dict(h0=C.c_void_p(258))),
    (_scan_bwd, dict(t=3)), (_scan_bwd, dict(dr=31)), (_scan_bwd, dict(dc=300)), (_scan_bwd, dict(gr=-16)),
    (_scan_bwd, dict(p=(A, None, A, A))), (_scan_bwd, dict(p=(A, A, None, A))), (_scan_bwd, dict(p=(A, A, A, None))),
    (_scan_bwd, dict(p=(A, C.c_void_p(258), A, A))),
    (_loss, dict(t=3)), (_loss, dict(tok_t=3)), (_loss, dict(rows=-1)), (_loss, dict(vocab=0)),
    (_loss, dict(vocab=1025, ld=1025)), (_loss, dict(ld=255)), (_loss, dict(ld_g=255)), (_loss, dict(inv=0.0)),
    (_loss, dict(inv=float("nan"))), (_loss, dict(inv=float("inf"))), (_loss, dict(p=(None, A, A, A))),
    (_loss, dict(p=(A, None, A, A))), (_loss, dict(p=(A, A, None, None))), (_loss, dict(p=(odd, A, A, None))),
    (_loss, dict(ld_g=300, p=(A, A, A, A))),
]


@pytest.mark.parametrize("call,args", REFUSED, ids=lambda x: x.__name__ if callable(x) else ",".join(x))
def test_refused_with_a_message(boa, call, args):
    L = boa.lib()
    assert call(L, **args) == boa.BOA_E_INVALID
    name = {"_embed": b"boa_embed:", "_embed_bwd": b"boa_embed_backward:", "_scan": b"boa_mingru_scan:",
            "_scan_bwd": b"boa_mingru_scan_backward:", "_loss": b"boa_token_loss:"}[call.__name__]
    assert L.boa_last_error(None).startswith(name)


def test_empty_calls_do_nothing(boa):
    """No rows: nothing is read, written or launched, whatever the buffers."""
    L = boa.lib()
    assert _embed(L, n=0, p=(None, None, None)) == 0
    assert _loss(L, rows=0, p=(None, None, None, None)) == 0
    assert _scan(L, B=0, zh=None, h=None) == 0
    assert _scan_bwd(L, B=0, p=(None, None, None, None)) == 0
    assert L.boa_embed_backward_workspace(0, 256, 64) == 0
    assert L.boa_embed_backward_workspace(-1, 256, 64) == 0
    assert L.boa_mingru_states_floats(3, 0, 64) == 0


def test_other_failures_keep_their_own_message(boa):
    """The last failed call of a thread is the one whose message is given."""
    L = boa.lib()
    assert _embed(L, vocab=0) == boa.BOA_E_INVALID and b"vocab" in L.boa_last_error(None)
    assert L.boa_rc_encoder_init(None, 4, None) == boa.BOA_E_INVALID
    assert L.boa_last_error(None).startswith(b"boa_rc_encoder_init")


def test_messages_of_threads_are_apart(boa):
    import threading
    L, seen = boa.lib(), {}

    def work(k):
        for _ in range(200):
            assert (_embed(L, vocab=0) if k else _loss(L, inv=0.0)) == boa.BOA_E_INVALID
            seen.setdefault(k, set()).add(bytes(L.boa_last_error(None)))
    ts = [threading.Thread(target=work, args=(k,)) for k in (0, 1)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert len(seen[0]) == len(seen[1]) == 1 and b"inv_temperature" in next(iter(seen[0]))


def test_python_refuses_tensors_off_the_gpu(boa):
    import torch
    from boa_b200 import training as tr
    x = torch.zeros(4, 8)
    for call in (lambda: tr.embed(torch.zeros(4, dtype=torch.uint8), x),
                 lambda: tr.embed_backward(torch.zeros(4, dtype=torch.int64), x, 8),
                 lambda: tr.mingru_scan(torch.zeros(1, 4, 8)),
                 lambda: tr.mingru_scan_backward(torch.zeros(1, 4, 8), x, x),
                 lambda: tr.token_loss(x, torch.zeros(4, dtype=torch.uint8)),
                 lambda: tr.token_loss(x, torch.zeros(5, dtype=torch.uint8))):
        with pytest.raises(boa.BoaError) as e:
            call()
        assert e.value.code == boa.BOA_E_INVALID


# The plain forms themselves: their gradients against differences.
def _diff(f, x, at, step=1e-6):
    hi, lo = x.copy(), x.copy()
    hi[at] += step
    lo[at] -= step
    return (f(hi) - f(lo)) / (2 * step)


def test_plain_mingru_gradient_against_differences():
    rng = np.random.default_rng(0)
    B, T, d = 3, 9, 4
    zh, h0 = rng.normal(size=(B, T, 2 * d)), rng.normal(size=(B, d))
    dh, dl, n = rng.normal(size=(B, T, d)), rng.normal(size=(B, d)), np.array([9, 4, 0])
    got = R.mingru(zh, h0, n, dh, dl)

    def f(z, s):
        r = R.mingru(z, s, n)
        return (r["h"][0] * dh).sum() + (r["last"][0] * dl).sum()
    for at in np.ndindex(zh.shape):
        if abs(zh[at]) > 1e-3:  # c has a kink at hr = 0
            assert abs(_diff(lambda z: f(z, h0), zh, at) - got["dzh"][0][at]) < 1e-7
    for at in np.ndindex(h0.shape):
        assert abs(_diff(lambda s: f(zh, s), h0, at) - got["dh0"][0][at]) < 1e-7


def test_plain_loss_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, t, w = rng.normal(size=(5, 7)), np.array([0, 6, 3, -1, 7]), rng.normal(size=5)
    _, (g, _) = R.token_loss(x, t, 1.3, w)
    for at in np.ndindex(x.shape):
        assert abs(_diff(lambda y: (R.token_loss(y, t, 1.3, w)[0][0] * w).sum(), x, at) - g[at]) < 1e-7


def test_plain_embedding_gradient_against_differences():
    rng = np.random.default_rng(2)
    E, t, u = rng.normal(size=(4, 3)), np.array([0, 3, 3, -1, 4, 0, 2]), rng.normal(size=(7, 3))
    g, _ = R.embed_grad(t, u, 4, 2.5)
    for at in np.ndindex(E.shape):
        assert abs(_diff(lambda e: (R.embed(t, e, 2.5)[0] * u).sum(), E, at) - g[at]) < 1e-7
