"""Refusals of the training operators' later entry points and calls (no GPU)."""
import ctypes as C

import numpy as np
import pytest


@pytest.mark.parametrize("args", [(-1, 4, 1, 1000), (4096, 4, 1, 1000), (0, 0, 1, 1000), (0, 65, 1, 1000),
                                  (0, 4, -1, 1000), (0, 4, 1, 0), (0, 4, 1, 1000001)])
def test_walk_selftest_refuses(boa, args):
    out = np.zeros((65, 128), np.float32).ctypes.data_as(C.POINTER(C.c_float))
    assert boa.lib().boa_selftest_walk_timeout(*args, out) == boa.BOA_E_INVALID
    assert boa.lib().boa_last_error(None).startswith(b"boa_selftest_walk_timeout")


def _calls(tr, torch):
    """name -> (call, the tensors through which a gradient could be lost)"""
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    tok = torch.zeros(4, dtype=torch.uint8)
    return {
        "embed": (lambda **k: tr.embed(tok, **k), dict(table=f(8, 4), out=f(4, 4))),
        "embed_backward": (lambda **k: tr.embed_backward(tok, vocab=8, **k), dict(dout=f(4, 4), out=f(8, 4))),
        "mingru_scan": (tr.mingru_scan, dict(zh=f(1, 3, 8), h0=f(1, 4), out=f(1, 3, 4), h_last=f(1, 4))),
        "mingru_scan_backward": (tr.mingru_scan_backward,
                                 dict(zh=f(1, 3, 8), states=f(4), dh=f(1, 3, 4), dh_last=f(1, 4), out=f(1, 3, 8))),
        "token_loss": (lambda **k: tr.token_loss(targets=tok, **k), dict(logits=f(4, 8), dloss=f(4), out=f(4, 8))),
    }


NAMES = [("embed", "table"), ("embed", "out"), ("embed_backward", "dout"), ("embed_backward", "out"),
         ("mingru_scan", "zh"), ("mingru_scan", "h0"), ("mingru_scan", "out"), ("mingru_scan", "h_last"),
         ("mingru_scan_backward", "zh"), ("mingru_scan_backward", "states"), ("mingru_scan_backward", "dh"),
         ("mingru_scan_backward", "dh_last"), ("mingru_scan_backward", "out"), ("token_loss", "logits"),
         ("token_loss", "dloss"), ("token_loss", "out")]


@pytest.mark.parametrize("op,name", NAMES)
def test_a_gradient_is_not_dropped_in_silence(boa, op, name):
    """Refused while torch records gradients; inside no_grad the same call goes
    on to the next check (here, that the tensors are on a GPU)."""
    import torch
    from boa_b200 import training as tr
    call, args = _calls(tr, torch)[op]
    args[name].requires_grad_()
    with pytest.raises(boa.BoaError, match=f"{name} requires a gradient") as e:
        call(**args)
    assert e.value.code == boa.BOA_E_INVALID
    with torch.no_grad(), pytest.raises(boa.BoaError, match="must be a CUDA tensor"):
        call(**args)


@pytest.mark.parametrize("op,name", NAMES)
def test_a_tangent_is_not_dropped_in_silence(boa, op, name):
    import torch
    from torch.autograd import forward_ad
    from boa_b200 import training as tr
    call, args = _calls(tr, torch)[op]
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with torch.no_grad(), pytest.raises(boa.BoaError, match=f"{name} is a forward-mode dual") as e:
            call(**args)
    assert e.value.code == boa.BOA_E_INVALID


def test_a_later_failure_of_the_probability_coder_is_the_last_one(boa):
    """boa_last_error(NULL) gives the last failed call without a handle, whichever kind it was."""
    L = boa.lib()
    assert L.boa_embed(None, 9, 0, None, 0, 0, 0, 0, 1.0, None, 0, 0, None) == boa.BOA_E_INVALID
    assert L.boa_last_error(None).startswith(b"boa_embed")
    h = C.c_void_p()
    assert L.boa_pyrc_create(0, 4, 4, 0, C.byref(h)) == boa.BOA_E_INVALID
    assert b"n_streams" in L.boa_last_error(None) and b"n_streams" in L.boa_pyrc_last_error(None)
