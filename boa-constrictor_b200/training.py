"""The operators a predictor is trained and stepped with, on torch tensors.

A thin binding of ``boa_embed``, ``boa_mingru_scan``, ``boa_token_loss`` and
their backward calls (``include/boa_b200.h``).  Inputs are CUDA tensors of one
device; work is enqueued on torch's current stream of that device, and
nothing synchronises, so every call can be captured into a CUDA graph.
Forward and backward are separate calls: what the backward pass needs is
returned by the forward call and kept by the caller.

``embed`` / ``embed_backward`` look tokens up and sum their gradients by
token; ``mingru_scan`` / ``mingru_scan_backward`` run the minGRU recurrence
over whole sequences (with one position, the decode step); ``token_loss``
gives the next-token loss and its gradient in one pass.  Wrong arguments
raise ``BoaError`` with ``BOA_E_INVALID``.
"""
from __future__ import annotations

import torch

from . import BOA_E_INVALID, BoaError, lib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TOKEN = {torch.uint8: 0, torch.int32: 1, torch.int64: 2}


def _bad(what: str):
    raise BoaError(BOA_E_INVALID, what)


def _call(fn, device, *args):
    """fn(*args, stream) with `device` current, on torch's current stream of it."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise BoaError(rc, (lib().boa_last_error(None) or b"").decode())


def _on(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _bad(f"{name} is on {t.device}, not on {device}")


def _type(t, name):
    k = _TYPE.get(t.dtype)
    return _bad(f"{name} must be float32, float16 or bfloat16, not {t.dtype}") if k is None else k


def _tokens(tokens, name="tokens"):
    """-> (contiguous tokens, their type code)"""
    if not tokens.is_cuda:
        _bad(f"{name} must be a CUDA tensor")
    k = _TOKEN.get(tokens.dtype)
    if k is None:
        _bad(f"{name} must be uint8, int32 or int64, not {tokens.dtype}")
    return tokens.contiguous(), k


def _rows(x, n, width, name, write=False):
    """x as n rows of `width` -> (tensor that holds them, elements between
    rows).  Rows that no single stride reaches are copied, unless they are
    written."""
    if x.dim() == 2 and x.shape[0] == n and x.shape[1] == width:
        rows = x
    elif x.dim() and x.shape[-1] == width and x.numel() == n * width:
        if write:
            try:
                rows = x.view(n, width)
            except RuntimeError:
                _bad(f"{name} must be a view of rows one stride apart")
        else:
            rows = x.reshape(n, width)
    else:
        _bad(f"{name} has shape {tuple(x.shape)}, not {n} rows of {width}")
    if n <= 1 and (width <= 1 or rows.stride(1) == 1):
        return rows, width
    s0, s1 = rows.stride()
    if (s1 == 1 or width == 1) and s0 >= width:
        return rows, s0
    if write:
        _bad(f"{name} must have rows that are contiguous and do not overlap")
    return rows.contiguous(), width


def _state(x, B, d, device, name, write=False):
    if x is None:
        return None
    if x.device != device or x.dtype != torch.float32 or x.shape != (B, d):
        _bad(f"{name} must be float32 of shape ({B}, {d}) on {device}")
    if x.is_contiguous():
        return x
    return _bad(f"{name} must be contiguous") if write else x.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def embed(tokens, table, scale: float = 1.0, dtype=None, out=None):
    """scale * table[tokens]: tokens of any shape (uint8, int32 or int64; one
    outside the table pads and gives a zero row), table [vocab <= 1024, d].
    -> tokens.shape + (d,) of `dtype` (the table's when not given)."""
    tokens, tok = _tokens(tokens)
    if table.dim() != 2:
        _bad("table must be [vocab, d]")
    vocab, d = table.shape
    n, device = tokens.numel(), tokens.device
    table, ld = _rows(table, vocab, d, "table")
    if out is None:
        out = torch.empty((*tokens.shape, d), dtype=dtype or table.dtype, device=device)
    elif out.shape != (*tokens.shape, d) or (dtype is not None and out.dtype != dtype):
        _bad(f"out must be of shape {(*tokens.shape, d)} and of dtype {dtype or out.dtype}")
    _on(device, table=table, out=out)
    rows, ld_out = _rows(out, n, d, "out", write=True)
    _call(lib().boa_embed, device, tokens.data_ptr(), tok, n, table.data_ptr(), _type(table, "table"), ld, vocab, d,
          scale, rows.data_ptr(), _type(out, "out"), ld_out)
    return out


def embed_backward(tokens, dout, vocab: int, scale: float = 1.0, dtype=torch.float32, out=None,
                   accumulate: bool = False):
    """Gradient of ``embed`` by its table, [vocab, d] of `dtype` (or in `out`,
    added to what it holds when `accumulate`)."""
    tokens, tok = _tokens(tokens)
    n, device = tokens.numel(), tokens.device
    if dout.dim() < 1 or dout.shape[-1] < 1 or dout.shape != (*tokens.shape, dout.shape[-1]):
        _bad(f"dout must be of shape {tuple(tokens.shape)} + (d,), not {tuple(dout.shape)}")
    d = dout.shape[-1]
    dout, ld = _rows(dout, n, d, "dout")
    if out is None:
        if accumulate:
            _bad("accumulate needs out")
        out = torch.empty((vocab, d), dtype=dtype, device=device)
    elif out.shape != (vocab, d):
        _bad(f"out must be of shape ({vocab}, {d})")
    _on(device, dout=dout, out=out)
    rows, ld_out = _rows(out, vocab, d, "out", write=True)
    L = lib()
    need = L.boa_embed_backward_workspace(n, vocab, d)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _call(L.boa_embed_backward, device, tokens.data_ptr(), tok, n, dout.data_ptr(), _type(dout, "dout"), ld, vocab, d,
          scale, int(accumulate), rows.data_ptr(), _type(out, "out"), ld_out, ws.data_ptr(), need)
    return out


def _gates(zh):
    if not zh.is_cuda or zh.dim() != 3 or zh.shape[2] < 2 or zh.shape[2] % 2:
        _bad("zh must be a CUDA tensor [chunks, positions, 2 d]")
    B, T, w = zh.shape
    return _steps(zh, "zh"), B, T, w // 2


def _steps(x, name, write=False):
    """x with contiguous rows; any strides between positions and chunks."""
    if x.stride(2) == 1 or x.shape[2] == 1:
        return x
    return _bad(f"{name} must have contiguous rows") if write else x.contiguous()


def _lengths(lengths, B, device):
    if lengths is None:
        return None
    if lengths.device != device or lengths.dtype != torch.int32 or lengths.shape != (B,):
        _bad(f"lengths must be int32 of shape ({B},) on {device}")
    return lengths.contiguous()


def mingru_scan(zh, h0=None, lengths=None, out=None, h_last=None, save_states: bool = False):
    """The minGRU recurrence over zh [chunks, positions, 2 d] (gate logits,
    then candidates) from the fp32 state h0 [chunks, d] (None = zeros).
    lengths: int32 positions of each chunk; rows past them are neither read
    nor part of the recurrence, and zero in h.  -> (h [chunks, positions, d],
    h_last fp32 [chunks, d]) and, with save_states, what
    ``mingru_scan_backward`` needs.  h_last may be h0 (updated in place)."""
    zh, B, T, d = _gates(zh)
    device = zh.device
    if out is None:
        out = torch.empty((B, T, d), dtype=zh.dtype, device=device)
    elif out.shape != (B, T, d) or out.dtype != zh.dtype:
        _bad(f"out must be {zh.dtype} of shape ({B}, {T}, {d})")
    _on(device, out=out)
    _steps(out, "out", write=True)
    h0 = _state(h0, B, d, device, "h0")
    if h_last is None:
        h_last = torch.empty((B, d), dtype=torch.float32, device=device)
    else:
        _state(h_last, B, d, device, "h_last", write=True)
    lengths = _lengths(lengths, B, device)
    L = lib()
    states = None
    if save_states:
        states = torch.empty(L.boa_mingru_states_floats(B, T, d), dtype=torch.float32, device=device)
    _call(L.boa_mingru_scan, device, zh.data_ptr(), _type(zh, "zh"), zh.stride(1), zh.stride(0), B, T, d,
          _ptr(lengths), _ptr(h0), out.data_ptr(), out.stride(1), out.stride(0), h_last.data_ptr(), _ptr(states))
    return (out, h_last, states) if save_states else (out, h_last)


def mingru_scan_backward(zh, states, dh, dh_last=None, lengths=None, out=None):
    """Gradient of ``mingru_scan`` from dh [chunks, positions, d] (zh's dtype)
    and dh_last fp32 [chunks, d] (None = zeros), with the states its forward
    call saved.  -> (dzh like zh, dh0 fp32 [chunks, d])"""
    zh, B, T, d = _gates(zh)
    device = zh.device
    if dh.shape != (B, T, d) or dh.dtype != zh.dtype:
        _bad(f"dh must be {zh.dtype} of shape ({B}, {T}, {d})")
    dh = _steps(dh, "dh")
    L = lib()
    if states.dtype != torch.float32 or states.numel() != L.boa_mingru_states_floats(B, T, d) or \
            not states.is_contiguous():
        _bad("states must be what mingru_scan(..., save_states=True) returned for these sizes")
    if out is None:
        out = torch.empty((B, T, 2 * d), dtype=zh.dtype, device=device)
    elif out.shape != (B, T, 2 * d) or out.dtype != zh.dtype:
        _bad(f"out must be {zh.dtype} of shape ({B}, {T}, {2 * d})")
    _on(device, dh=dh, states=states, out=out)
    _steps(out, "out", write=True)
    dh_last = _state(dh_last, B, d, device, "dh_last")
    dh0 = torch.empty((B, d), dtype=torch.float32, device=device)
    lengths = _lengths(lengths, B, device)
    _call(L.boa_mingru_scan_backward, device, zh.data_ptr(), _type(zh, "zh"), zh.stride(1), zh.stride(0), B, T, d,
          _ptr(lengths), states.data_ptr(), dh.data_ptr(), dh.stride(1), dh.stride(0), _ptr(dh_last),
          out.data_ptr(), out.stride(1), out.stride(0), dh0.data_ptr())
    return out, dh0


def token_loss(logits, targets, inv_temperature: float = 1.0, grad_scale: float | None = None, dloss=None, out=None):
    """Next-token cross entropy in nats of logits [..., vocab <= 1024] for
    targets [...] (uint8, int32 or int64; one outside the alphabet pads: loss
    and gradient 0).  -> (loss fp32 [...], gradient by the logits or None).

    The gradient is formed when grad_scale or dloss is given: that of
    sum(grad_scale * dloss * loss), with dloss fp32 [...] (None = ones), in the
    logits' dtype, in `out` when given (which may be `logits`)."""
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        _bad(f"logits {tuple(logits.shape)} do not match targets {tuple(targets.shape)}")
    targets, tok = _tokens(targets, "targets")
    n, vocab, device = targets.numel(), logits.shape[-1], targets.device
    rows, ld = _rows(logits, n, vocab, "logits")
    loss = torch.empty(targets.shape, dtype=torch.float32, device=device)
    grad, ld_grad = None, 0
    if dloss is not None:
        if dloss.dtype != torch.float32 or dloss.shape != targets.shape:
            _bad(f"dloss must be float32 of shape {tuple(targets.shape)}")
        dloss = dloss.contiguous()
    if grad_scale is not None or dloss is not None or out is not None:
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=device)
        elif out.shape != logits.shape or out.dtype != logits.dtype:
            _bad(f"out must be {logits.dtype} of shape {tuple(logits.shape)}")
        grad, ld_grad = _rows(out, n, vocab, "out", write=True)
        if grad.data_ptr() == logits.data_ptr() and grad.data_ptr() != rows.data_ptr():
            _bad("in place needs logits whose rows are contiguous")
    _on(device, logits=logits, dloss=dloss, out=out)
    _call(lib().boa_token_loss, device, rows.data_ptr(), _type(logits, "logits"), ld, n, vocab, targets.data_ptr(),
          tok, inv_temperature, _ptr(dloss), 1.0 if grad_scale is None else grad_scale, loss.data_ptr(), _ptr(grad),
          ld_grad)
    return loss, out
