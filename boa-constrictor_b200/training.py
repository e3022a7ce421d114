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

The results carry no autograd graph.  A tensor that requires a gradient is
refused where torch would record one (and so is a forward-mode dual), instead
of cutting the graph in silence: call these inside ``torch.no_grad()``, from a
``torch.autograd.Function`` whose backward is ``once_differentiable``, or on
detached tensors.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import BOA_E_INVALID, BoaError, lib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TOKEN = {torch.uint8: 0, torch.int32: 1, torch.int64: 2}
_FLOAT = torch.float32
_INT = 0x7FFFFFFF  # the largest C int: of a larger size ctypes would pass the low half


def _bad(what: str):
    raise BoaError(BOA_E_INVALID, what)


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same without the Stream object, which takes longer to make than a launch
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
# and the device without the check that CUDA is initialised: the tensors are on a GPU already
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _no_graph(names, *tensors):
    """Refuses tensors whose gradient would be lost."""
    for name, t in zip(names.split(), tensors):
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            _bad(f"{name} requires a gradient, which the result would not carry: call inside torch.no_grad(), "
                 f"from an autograd.Function (backward once_differentiable), or on {name}.detach()")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            _bad(f"{name} is a forward-mode dual, whose tangent the result would not carry")


def _call(fn, index, given, *args):
    """fn(*args, stream) with device `index` current, on torch's current stream
    of it.  `given`: the caller's tensor that it writes, or None; torch is told
    that it changed, so that a backward pass that saved it notices."""
    if index == _device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc != 0:
        raise BoaError(rc, (lib().boa_last_error(None) or b"").decode())
    if given is not None:
        increment_version(given)


def _same(index, t, name):
    if t.get_device() != index:
        _bad(f"{name} is on {t.device}, not on cuda:{index}")


def _type(t, name):
    k = _TYPE.get(t.dtype)
    return _bad(f"{name} must be float32, float16 or bfloat16, not {t.dtype}") if k is None else k


def _tokens(tokens, name="tokens"):
    """-> (contiguous tokens, their type code, their device)"""
    index = tokens.get_device()
    if index < 0:
        _bad(f"{name} must be a CUDA tensor")
    k = _TOKEN.get(tokens.dtype)
    if k is None:
        _bad(f"{name} must be uint8, int32 or int64, not {tokens.dtype}")
    return (tokens if tokens.is_contiguous() else tokens.contiguous()), k, index


def _sign(x, name, write=False):
    """A negative view (the imaginary part of a conjugate, whose sign torch
    keeps aside) as it reads in memory."""
    if write:
        _bad(f"{name} must not be a negative view")
    return x.resolve_neg()


def _rows(x, n, width, name, write=False):
    """x as n rows of `width` -> (tensor that holds them, elements between
    rows).  Rows that no single stride reaches are copied, unless they are
    written."""
    shape = x.shape
    if not shape or shape[-1] != width or x.numel() != n * width:
        _bad(f"{name} has shape {tuple(shape)}, not {n} rows of {width}")
    if x.is_neg():
        x = _sign(x, name, write)
    if x.is_contiguous():
        return x, width
    rows = x
    if len(shape) != 2:
        if write:
            try:
                rows = x.view(n, width)
            except RuntimeError:
                _bad(f"{name} must be a view of rows one stride apart")
        else:
            rows = x.reshape(n, width)
    s0, s1 = rows.stride()
    if s1 == 1 or width == 1:
        if n <= 1:
            return rows, width
        if s0 >= width:
            return rows, s0
    if write:
        _bad(f"{name} must have rows that are contiguous and do not overlap")
    return rows.contiguous(), width


def _state(x, shape, index, name, write=False):
    if x is None:
        return None
    if x.get_device() != index or x.dtype != _FLOAT or x.shape != shape:
        _bad(f"{name} must be float32 of shape {shape} on cuda:{index}")
    if x.is_neg():
        x = _sign(x, name, write)
    if x.is_contiguous():
        return x
    return _bad(f"{name} must be contiguous") if write else x.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def embed(tokens, table, scale: float = 1.0, dtype=None, out=None):
    """scale * table[tokens]: tokens of any shape (uint8, int32 or int64; one
    outside the table pads and gives a zero row), table [vocab <= 1024, d].
    -> tokens.shape + (d,) of `dtype` (the table's when not given)."""
    if table.requires_grad or (out is not None and out.requires_grad) or forward_ad._current_level >= 0:
        _no_graph("table out", table, out)
    tokens, tok, index = _tokens(tokens)
    if table.dim() != 2:
        _bad("table must be [vocab, d]")
    vocab, d = table.shape
    if vocab > _INT or d > _INT:
        _bad("the sides of table must be below 2^31")
    _same(index, table, "table")
    table, ld = _rows(table, vocab, d, "table")
    n, shape, given = tokens.numel(), tokens.shape + (d,), out
    if out is None:
        out = table.new_empty(shape, dtype=dtype)
        rows, ld_out = out, d
    else:
        if out.shape != shape or (dtype is not None and out.dtype != dtype):
            _bad(f"out must be of shape {tuple(shape)} and of dtype {dtype or out.dtype}")
        _same(index, out, "out")
        rows, ld_out = _rows(out, n, d, "out", write=True)
    _call(lib().boa_embed, index, given, tokens.data_ptr(), tok, n, table.data_ptr(), _type(table, "table"), ld, vocab,
          d, scale, rows.data_ptr(), _type(out, "out"), ld_out)
    return out


def embed_backward(tokens, dout, vocab: int, scale: float = 1.0, dtype=torch.float32, out=None,
                   accumulate: bool = False):
    """Gradient of ``embed`` by its table, [vocab, d] of `dtype` (or in `out`,
    added to what it holds when `accumulate`)."""
    if dout.requires_grad or (out is not None and out.requires_grad) or forward_ad._current_level >= 0:
        _no_graph("dout out", dout, out)
    tokens, tok, index = _tokens(tokens)
    n = tokens.numel()
    if dout.dim() < 1 or dout.shape[-1] < 1 or dout.shape[:-1] != tokens.shape:
        _bad(f"dout must be of shape {tuple(tokens.shape)} + (d,), not {tuple(dout.shape)}")
    d = dout.shape[-1]
    if vocab > _INT or d > _INT:
        _bad("vocab and d must be below 2^31")
    _same(index, dout, "dout")
    dout, ld = _rows(dout, n, d, "dout")
    given = out
    if out is None:
        if accumulate:
            _bad("accumulate needs out")
        if vocab < 1:
            _bad("vocab must be 1 .. 1024")
        out = dout.new_empty((vocab, d), dtype=dtype)
        rows, ld_out = out, d
    else:
        if out.shape != (vocab, d):
            _bad(f"out must be of shape ({vocab}, {d})")
        _same(index, out, "out")
        rows, ld_out = _rows(out, vocab, d, "out", write=True)
    L = lib()
    need = L.boa_embed_backward_workspace(n, vocab, d)
    ws = tokens.new_empty(need, dtype=torch.uint8) if need else None
    _call(L.boa_embed_backward, index, given, tokens.data_ptr(), tok, n, dout.data_ptr(), _type(dout, "dout"), ld,
          vocab, d, scale, int(accumulate), rows.data_ptr(), _type(out, "out"), ld_out, _ptr(ws), need)
    return out


def _gates(zh):
    """-> (zh with contiguous rows, chunks, positions, d, strides, device)"""
    index = zh.get_device()
    if index < 0 or zh.dim() != 3:
        _bad("zh must be a CUDA tensor [chunks, positions, 2 d]")
    B, T, w = zh.shape
    if w < 2 or w % 2:
        _bad("zh must be a CUDA tensor [chunks, positions, 2 d]")
    if B > _INT or T > _INT or w > _INT:
        _bad("chunks, positions and 2 d must be below 2^31")
    zh, row, chunk = _steps(zh, "zh")
    return zh, B, T, w // 2, row, chunk, index


def _steps(x, name, write=False):
    """x with contiguous rows -> (x, elements between positions, between chunks)"""
    if x.is_neg():
        x = _sign(x, name, write)
    chunk, row, one = x.stride()
    if one == 1 or x.shape[2] == 1:
        return x, row, chunk
    if write:
        _bad(f"{name} must have contiguous rows")
    x = x.contiguous()
    return x, x.stride(1), x.stride(0)


def _lengths(lengths, B, index):
    if lengths is None:
        return None
    if lengths.get_device() != index or lengths.dtype != torch.int32 or lengths.shape != (B,):
        _bad(f"lengths must be int32 of shape ({B},) on cuda:{index}")
    return lengths.contiguous()


def _result(x, like, shape, index, name):
    """-> (output tensor, elements between positions, between chunks)"""
    if x is None:
        return like.new_empty(shape), shape[2], shape[1] * shape[2]
    if x.shape != shape or x.dtype != like.dtype:
        _bad(f"{name} must be {like.dtype} of shape {shape}")
    _same(index, x, name)
    return _steps(x, name, write=True)


def mingru_scan(zh, h0=None, lengths=None, out=None, h_last=None, save_states: bool = False):
    """The minGRU recurrence over zh [chunks, positions, 2 d] (gate logits,
    then candidates) from the fp32 state h0 [chunks, d] (None = zeros).
    lengths: int32 positions of each chunk; rows past them are neither read
    nor part of the recurrence, and zero in h.  -> (h [chunks, positions, d],
    h_last fp32 [chunks, d]) and, with save_states, what
    ``mingru_scan_backward`` needs.  h_last may be h0 (updated in place).

    Calls of up to 8 positions give the same bits however a sequence is cut
    into them; a longer one agrees with them to rounding only.  An encoder and
    a decoder that must agree both step in calls of at most 8."""
    if (zh.requires_grad or (h0 is not None and h0.requires_grad) or (out is not None and out.requires_grad) or
            (h_last is not None and h_last.requires_grad) or forward_ad._current_level >= 0):
        _no_graph("zh h0 out h_last", zh, h0, out, h_last)
    zh, B, T, d, zr, zc, index = _gates(zh)
    given, state = out, h_last
    out, hr, hc = _result(out, zh, (B, T, d), index, "out")
    h0 = _state(h0, (B, d), index, "h0")
    if h_last is None:
        h_last = zh.new_empty((B, d), dtype=_FLOAT)
    else:
        _state(h_last, (B, d), index, "h_last", write=True)
    lengths = _lengths(lengths, B, index)
    L = lib()
    states = zh.new_empty(L.boa_mingru_states_floats(B, T, d), dtype=_FLOAT) if save_states else None
    _call(L.boa_mingru_scan, index, given, zh.data_ptr(), _type(zh, "zh"), zr, zc, B, T, d, _ptr(lengths), _ptr(h0),
          out.data_ptr(), hr, hc, h_last.data_ptr(), _ptr(states))
    if state is not None:
        increment_version(state)
    return (out, h_last, states) if save_states else (out, h_last)


def mingru_scan_backward(zh, states, dh, dh_last=None, lengths=None, out=None):
    """Gradient of ``mingru_scan`` from dh [chunks, positions, d] (zh's dtype)
    and dh_last fp32 [chunks, d] (None = zeros), with the states its forward
    call saved.  -> (dzh like zh, dh0 fp32 [chunks, d])"""
    if (zh.requires_grad or states.requires_grad or dh.requires_grad or
            (dh_last is not None and dh_last.requires_grad) or (out is not None and out.requires_grad) or
            forward_ad._current_level >= 0):
        _no_graph("zh states dh dh_last out", zh, states, dh, dh_last, out)
    zh, B, T, d, zr, zc, index = _gates(zh)
    if dh.shape != (B, T, d) or dh.dtype != zh.dtype:
        _bad(f"dh must be {zh.dtype} of shape ({B}, {T}, {d})")
    _same(index, dh, "dh")
    dh, gr, gc = _steps(dh, "dh")
    L = lib()
    if states.dtype != _FLOAT or states.numel() != L.boa_mingru_states_floats(B, T, d) or not states.is_contiguous():
        _bad("states must be what mingru_scan(..., save_states=True) returned for these sizes")
    _same(index, states, "states")
    given = out
    out, dr, dc = _result(out, zh, (B, T, 2 * d), index, "out")
    dh_last = _state(dh_last, (B, d), index, "dh_last")
    dh0 = zh.new_empty((B, d), dtype=_FLOAT)
    lengths = _lengths(lengths, B, index)
    _call(L.boa_mingru_scan_backward, index, given, zh.data_ptr(), _type(zh, "zh"), zr, zc, B, T, d, _ptr(lengths),
          states.data_ptr(), dh.data_ptr(), gr, gc, _ptr(dh_last), out.data_ptr(), dr, dc, dh0.data_ptr())
    return out, dh0


def token_loss(logits, targets, inv_temperature: float = 1.0, grad_scale: float | None = None, dloss=None, out=None):
    """Next-token cross entropy in nats of logits [..., vocab <= 1024] for
    targets [...] (uint8, int32 or int64; one outside the alphabet pads: loss
    and gradient 0).  -> (loss fp32 [...], gradient by the logits or None).

    The gradient is formed when grad_scale, dloss or out is given: that of
    sum(grad_scale * dloss * loss), with dloss fp32 [...] (None = ones), in the
    logits' dtype, in `out` when given (which may be `logits`)."""
    if (logits.requires_grad or (dloss is not None and dloss.requires_grad) or
            (out is not None and out.requires_grad) or forward_ad._current_level >= 0):
        _no_graph("logits dloss out", logits, dloss, out)
    targets, tok, index = _tokens(targets, "targets")
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        _bad(f"logits {tuple(logits.shape)} do not match targets {tuple(targets.shape)}")
    n, vocab = targets.numel(), logits.shape[-1]
    if vocab > _INT:
        _bad("vocab must be below 2^31")
    _same(index, logits, "logits")
    rows, ld = _rows(logits, n, vocab, "logits")
    loss = targets.new_empty(targets.shape, dtype=_FLOAT)
    grad, ld_grad, given = None, 0, out
    if dloss is not None:
        if dloss.get_device() != index or dloss.dtype != _FLOAT or dloss.shape != targets.shape:
            _bad(f"dloss must be float32 of shape {tuple(targets.shape)} on cuda:{index}")
        dloss = dloss.resolve_neg().contiguous()
    if out is not None:
        if out.shape != logits.shape or out.dtype != logits.dtype:
            _bad(f"out must be {logits.dtype} of shape {tuple(logits.shape)}")
        _same(index, out, "out")
        grad, ld_grad = _rows(out, n, vocab, "out", write=True)
        if grad.data_ptr() == logits.data_ptr() and grad.data_ptr() != rows.data_ptr():
            _bad("in place needs logits whose rows are contiguous")
    elif grad_scale is not None or dloss is not None:
        out = grad = logits.new_empty(logits.shape)
        ld_grad = vocab
    _call(lib().boa_token_loss, index, given, rows.data_ptr(), _type(logits, "logits"), ld, n, vocab,
          targets.data_ptr(), tok, inv_temperature, _ptr(dloss), 1.0 if grad_scale is None else grad_scale,
          loss.data_ptr(), _ptr(grad), ld_grad)
    return loss, out
