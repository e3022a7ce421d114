"""The training operators (boa_b200.training) against plain 64-bit forms, at
the sizes, types, strides and masks where they can go wrong.  Tolerances are
the running error bounds of training_ref.py plus half a step of the type that
a result is stored in."""
import numpy as np
import pytest

import training_ref as R

pytestmark = pytest.mark.gpu

DT = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


def _t(torch, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(getattr(torch, dtype))


def _n(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _close(got, ref, err, dtype, what=""):
    got, tol = _n(got), R.stored(ref, err, dtype)
    with np.errstate(invalid="ignore"):
        off = np.abs(got - ref)
    bad = ~(off <= tol) & ~(np.isnan(got) & np.isnan(ref)) & ~((got == ref) & np.isinf(ref))
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, first at {at}: got {got[at]!r}, "
                             f"want {ref[at]!r} within {tol[at]:.3g}")


def _strided(torch, x, gap=0, offset=0):
    """x in rows that are `gap` elements longer, `offset` elements into their buffer."""
    n, d = x.shape
    buf = torch.full((n * (d + gap) + offset,), float("nan") if x.is_floating_point() else 77, dtype=x.dtype,
                     device="cuda")
    v = buf[offset:].view(n, d + gap)[:, :d]
    v.copy_(x)
    return v


def _tokens(torch, rng, n, vocab, tok, pad=True, skew=False):
    t = rng.integers(0, vocab, n)
    if skew:
        t[rng.random(n) < 0.9] = vocab // 3
    if pad and tok != "uint8":
        t[rng.random(n) < 0.1] = -1
        t[rng.random(n) < 0.05] = vocab
        if tok == "int64":
            t[rng.random(n) < 0.05] = (1 << 32) + 1  # its low half is a token
    return t, _t(torch, t.astype(tok))


# ---------------------------------------------------------------- embedding
@pytest.mark.parametrize("tok", ["uint8", "int32", "int64"])
@pytest.mark.parametrize("table_t,out_t", [(a, b) for a in DT for b in DT])
@pytest.mark.parametrize("n,d,vocab", [(1, 1, 1), (1, 256, 256), (37, 80, 256), (3000, 64, 7), (513, 163, 256)])
def test_embed(tr, tok, table_t, out_t, n, d, vocab):
    import torch
    rng = np.random.default_rng(n + d)
    t, tt = _tokens(torch, rng, n, vocab, tok)
    E = _t(torch, rng.normal(size=(vocab, d)), table_t)
    out = tr.embed(tt, E, scale=3.7, dtype=getattr(torch, out_t))
    assert out.dtype == getattr(torch, out_t) and out.shape == (n, d)
    ref, err = R.embed(t, _n(E), float(np.float32(3.7)))
    _close(out, ref, err, out_t)


@pytest.mark.parametrize("gap,offset", [(0, 1), (3, 0), (8, 0), (8, 4)])
def test_embed_strides_and_alignment(tr, gap, offset):
    """Rows further apart than their width, and buffers off the 16-byte grid;
    what lies between the rows is left alone."""
    import torch
    rng = np.random.default_rng(5)
    t, tt = _tokens(torch, rng, 500, 200, "int32")
    E = _strided(torch, _t(torch, rng.normal(size=(200, 64)).astype(np.float32)), gap, offset)
    out = _strided(torch, torch.zeros(500, 64, dtype=torch.bfloat16, device="cuda"), gap, offset)
    ref, err = R.embed(t, _n(E), 0.5)
    got = tr.embed(tt, E, scale=0.5, out=out)
    assert got is out
    _close(out, ref, err, "bfloat16")
    if gap:
        buf = out.as_strided((499, gap), (64 + gap, 1), out.storage_offset() + 64)
        assert torch.isnan(buf).all()


def test_embed_takes_tokens_of_any_shape(tr):
    import torch
    E = torch.randn(256, 16, device="cuda")
    tok = torch.randint(0, 256, (5, 7, 3), device="cuda")
    assert torch.equal(tr.embed(tok, E), E[tok])
    assert torch.equal(tr.embed(tok.transpose(0, 2), E), E[tok.transpose(0, 2)])
    assert tr.embed(tok[:0], E).shape == (0, 7, 3, 16)
    assert torch.equal(tr.embed(tok[0, 0, 0], E), E[tok[0, 0, 0]])


@pytest.mark.parametrize("d", [4096, 65535, 65536])
def test_embed_widest_rows(tr, d):
    import torch
    tok, E = torch.tensor([3, 0, -1, 3], device="cuda"), torch.randn(4, d, device="cuda")
    out = tr.embed(tok, E, scale=2.0)
    assert torch.equal(out[[0, 1, 3]], 2 * E[[3, 0, 3]]) and (out[2] == 0).all()
    g = torch.randint(-8, 8, (4, d), device="cuda").float()
    ref = torch.zeros(4, d, device="cuda")
    ref[0], ref[3] = g[1], g[0] + g[3]
    assert torch.equal(tr.embed_backward(tok, g, 4), ref)
    many = torch.arange(6000, device="cuda") % 4
    g = torch.ones((), device="cuda").expand(6000, d // 16)
    assert (tr.embed_backward(many, g, 4) == 1500).all()


def test_embed_padding_reads_nothing(tr):
    """NaN in the table does not reach padded rows."""
    import torch
    E = torch.full((4, 8), float("nan"), device="cuda")
    out = tr.embed(torch.tensor([-1, 4, 1 << 40, -(1 << 40)], device="cuda"), E)
    assert torch.equal(out, torch.zeros_like(out))


@pytest.mark.parametrize("dout_t,dtable_t", [("float32", "float32"), ("float16", "float32"), ("bfloat16", "float32"),
                                             ("bfloat16", "bfloat16"), ("float16", "float16")])
@pytest.mark.parametrize("n,d,vocab,tok,skew", [
    (1, 1, 1, "int32", False), (1, 64, 256, "uint8", False), (2, 3, 2, "int64", False), (511, 64, 1, "int32", False),
    (512, 80, 256, "uint8", True), (513, 65, 256, "uint8", False), (4096, 64, 256, "uint8", True),
    (4097, 160, 1000, "int64", False), (9001, 33, 1024, "int32", True), (20011, 300, 256, "uint8", True)])
def test_embed_backward(tr, dout_t, dtable_t, n, d, vocab, tok, skew):
    import torch
    rng = np.random.default_rng(n * d)
    t, tt = _tokens(torch, rng, n, vocab, tok, skew=skew)
    g = _t(torch, rng.normal(size=(n, d)) * 0.1, dout_t)
    out = tr.embed_backward(tt, g, vocab, scale=2.5, dtype=getattr(torch, dtable_t))
    ref, err = R.embed_grad(t, _n(g), vocab, 2.5)
    _close(out, ref, err, dtable_t)
    assert torch.equal(out, tr.embed_backward(tt, g, vocab, scale=2.5, dtype=getattr(torch, dtable_t)))


@pytest.mark.parametrize("n,d,vocab,dout_t,skew", [
    (9000, 5, 1, "float32", False),          # one token, 71 pieces
    (40000, 12, 3, "bfloat16", True),        # more pieces than are kept of one token
    (300000, 7, 3, "float32", True),         # pieces longer than a block lists at once
    (300000, 300, 2, "float16", True),       # and columns in two rounds
    (5000, 2052, 256, "float32", False), (49152, 20, 1024, "float32", True), (49153, 20, 1024, "float32", False),
    (4096, 300, 1024, "bfloat16", True), (4097, 8, 1024, "float16", False)])
def test_embed_backward_pieces(tr, n, d, vocab, dout_t, skew):
    """Long pieces, many pieces and wide rows; the sums in 64 bits by torch."""
    import torch
    rng = np.random.default_rng(n + d)
    t, tt = _tokens(torch, rng, n, vocab, "int32", skew=skew)
    g = torch.randn(n, d, generator=torch.Generator(device="cuda").manual_seed(d), device="cuda")
    g = g.to(getattr(torch, dout_t))
    got = tr.embed_backward(tt, g, vocab)
    ok = (tt >= 0) & (tt < vocab)
    ref, size = (torch.zeros(vocab, d, dtype=torch.float64, device="cuda") for _ in range(2))
    ref.index_add_(0, tt[ok].long(), g[ok].double())
    size.index_add_(0, tt[ok].long(), g[ok].double().abs())
    # a piece has at most n / 256 + 128 rows, a token at most 256 pieces, a block at most 256 partial sums
    err = (n // 256 + 128 + 512) * R.U * _n(size)
    _close(got, _n(ref), err, "float32")


@pytest.mark.parametrize("gap,offset", [(0, 1), (3, 0), (8, 4)])
def test_embed_backward_strides_and_accumulate(tr, gap, offset):
    import torch
    rng = np.random.default_rng(6)
    t, tt = _tokens(torch, rng, 3001, 100, "int64")
    g = _strided(torch, _t(torch, rng.normal(size=(3001, 64)).astype(np.float32)), gap, offset)
    old = _t(torch, rng.normal(size=(100, 64)).astype(np.float32))
    out = _strided(torch, old, gap, offset)
    assert tr.embed_backward(tt, g, 100, scale=0.25, out=out, accumulate=True) is out
    ref, err = R.embed_grad(t, _n(g), 100, 0.25)
    ref = ref + _n(old)
    _close(out, ref, err + R.U * np.abs(ref), "float32")
    if gap:
        assert torch.isnan(out.as_strided((99, gap), (64 + gap, 1), out.storage_offset() + 64)).all()


def test_embed_backward_nothing_to_sum(tr):
    """No tokens, padding alone, and tokens that never occur: zeros, or with
    accumulate what was there; NaN in padded rows is not read."""
    import torch
    e = torch.empty(0, dtype=torch.uint8, device="cuda")
    z = torch.zeros(256, 24, device="cuda")
    assert torch.equal(tr.embed_backward(e, torch.empty(0, 24, device="cuda"), 256), z)
    old = torch.randn(256, 24, device="cuda")
    got = tr.embed_backward(e, torch.empty(0, 24, device="cuda"), 256, out=old.clone(), accumulate=True)
    assert torch.equal(got, old)
    nan = torch.full((700, 24), float("nan"), device="cuda")
    pad = torch.full((700,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(tr.embed_backward(pad, nan, 256), z)
    got = tr.embed_backward(pad, nan, 256, out=old.clone(), accumulate=True)
    assert torch.equal(got, old)


def test_embed_backward_takes_an_expanded_gradient(tr):
    """The gradient of a sum is one value expanded, with strides of 0."""
    import torch
    tok = torch.randint(0, 256, (4, 300), device="cuda", dtype=torch.uint8)
    got = tr.embed_backward(tok, torch.ones((), device="cuda").expand(4, 300, 48), 256)
    ref = torch.bincount(tok.flatten().long(), minlength=256).float()[:, None].expand(256, 48)
    assert torch.equal(got, ref)


# --------------------------------------------------------------- recurrence
def _case(torch, rng, B, T, d, dtype, lengths=None, gate=-1.0, layout="chunks"):
    """-> numpy inputs (rounded to dtype) and their tensors"""
    zh = np.concatenate([rng.normal(gate, 1.5, (B, T, d)), rng.normal(size=(B, T, d))], 2)
    zh, dh = _t(torch, zh, dtype), _t(torch, rng.normal(size=(B, T, d)) * 0.1, dtype)
    if layout == "time":  # [T][B] in memory
        zh, dh = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (zh, dh))
    elif layout == "wide":  # parts of wider rows, off the 16-byte grid
        zh = torch.nn.functional.pad(zh, (3, 6), value=float("nan"))[:, :, 3:3 + 2 * d]
        dh = torch.nn.functional.pad(dh, (1, 4), value=float("nan"))[:, :, 1:1 + d]
    h0 = _t(torch, rng.normal(size=(B, d)).astype(np.float32))
    dl = _t(torch, (rng.normal(size=(B, d)) * 0.1).astype(np.float32))
    n = None if lengths is None else _t(torch, np.asarray(lengths, np.int32))
    return zh, h0, n, dh, dl


def _check_scan(tr, torch, zh, h0, n, dh, dl, dtype):
    B, T, w = zh.shape
    d = w // 2
    h, last, states = tr.mingru_scan(zh, h0, n, save_states=True)
    dzh, dh0 = tr.mingru_scan_backward(zh, states, dh, dl, n)
    ref = R.mingru(_n(zh), 0.0 if h0 is None else _n(h0), None if n is None else _n(n), _n(dh),
                   np.zeros((B, d)) if dl is None else _n(dl))
    _close(h, *ref["h"], dtype, "h")
    _close(last, *ref["last"], "float32", "h_last")
    _close(dzh, *ref["dzh"], dtype, "dzh")
    _close(dh0, *ref["dh0"], "float32", "dh0")
    # without the states for a backward pass, and again: the same bits
    h2, last2 = tr.mingru_scan(zh, h0, n)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    again = tr.mingru_scan_backward(zh, states, dh, dl, n)
    assert torch.equal(dzh, again[0]) and torch.equal(dh0, again[1])
    return h, last, dzh, dh0


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,d", [
    (1, 1, 1), (3, 1, 80), (700, 1, 64), (2, 2, 33), (5, 7, 64), (3, 16, 160), (2, 31, 128), (1, 64, 256), (40, 65, 48),
    (2, 127, 65), (3, 128, 64), (1, 129, 512), (4, 255, 31), (2, 257, 64), (1, 1000, 7), (2, 2049, 40), (1, 9000, 3),
    (9, 515, 160)])
def test_mingru(tr, dtype, B, T, d):
    import torch
    _check_scan(tr, torch, *_case(torch, np.random.default_rng(B * T + d), B, T, d, dtype), dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,d", [(150, 70, 64), (150, 9, 66), (80, 200, 130), (40, 140, 256), (300, 33, 33)])
def test_mingru_many_chains(tr, dtype, B, T, d):
    """Enough chains for several blocks per SM, aligned and not."""
    import torch
    lengths = np.random.default_rng(B).integers(0, T + 1, B)
    lengths[: B // 2] = T
    _check_scan(tr, torch, *_case(torch, np.random.default_rng(T), B, T, d, dtype, lengths), dtype)


def test_mingru_shared_gates(tr):
    """One chunk's gates expanded over the batch (a stride of 0)."""
    import torch
    zh, _, _, dh, dl = _case(torch, np.random.default_rng(12), 1, 300, 32, "float32")
    zh, dh, dl = zh.expand(5, 300, 64), dh.expand(5, 300, 32), dl.expand(5, 32)
    h0 = torch.randn(5, 32, device="cuda")
    _check_scan(tr, torch, zh, h0, None, dh, dl, "float32")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("layout", ["time", "wide"])
@pytest.mark.parametrize("B,T,d", [(3, 1, 64), (5, 40, 64), (3, 300, 80), (2, 700, 33)])
def test_mingru_layouts(tr, dtype, layout, B, T, d):
    import torch
    _check_scan(tr, torch, *_case(torch, np.random.default_rng(T), B, T, d, dtype, layout=layout), dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,d", [(1, 64), (12, 80), (130, 64), (600, 33), (1500, 20)])
def test_mingru_ragged(tr, dtype, T, d):
    """Lengths of 0, 1, T, past T and below 0; NaN and infinities past a
    chunk's length reach nothing, and rows there are zero."""
    import torch
    lengths = [0, 1, T, T + 9, -3, T // 2, max(T - 1, 0), min(T, 128), min(T, 129)]
    zh, h0, n, dh, dl = _case(torch, np.random.default_rng(T + d), len(lengths), T, d, dtype, lengths)
    past = torch.arange(T, device="cuda")[None, :] >= n[:, None]
    zh[past], dh[past] = float("nan"), float("inf")
    h, last, dzh, dh0 = _check_scan(tr, torch, zh, h0, n, dh, dl, dtype)
    assert (h[past] == 0).all() and (dzh[past] == 0).all()
    assert torch.equal(last[0], h0[0]) and torch.equal(dh0[0], dl[0])


@pytest.mark.parametrize("gate", [-12.0, 8.0])
def test_mingru_gates_that_keep_or_forget(tr, gate):
    import torch
    _check_scan(tr, torch, *_case(torch, np.random.default_rng(3), 2, 1400, 40, "float32", gate=gate), "float32")


def test_mingru_without_states_at_the_ends(tr):
    import torch
    zh, _, n, dh, _ = _case(torch, np.random.default_rng(4), 3, 200, 24, "float32", [200, 7, 0])
    _check_scan(tr, torch, zh, None, n, dh, None, "float32")


def test_mingru_extreme_gates(tr):
    """Gates and candidates of either infinity, the type's range and NaN."""
    import torch
    inf = float("inf")
    vals = [(-inf, 1.0), (inf, 1.0), (200.0, -200.0), (-200.0, 3.0), (0.0, -inf), (inf, -inf), (3e38, -3e38), (-3e38, 0.0)]
    zh = torch.tensor([[list(v) for v in vals]], device="cuda")  # one chunk, d = 1
    h0 = torch.full((1, 1), 0.25, device="cuda")
    dh, dl = torch.full((1, 8, 1), 0.5, device="cuda"), torch.ones(1, 1, device="cuda")
    _check_scan(tr, torch, zh, h0, None, dh, dl, "float32")
    zh[0, 3, 0] = float("nan")
    h, last = tr.mingru_scan(zh, h0)
    # NaN stays until a gate of 1 forgets the state; it forgets as 0 * NaN does not: NaN
    assert torch.isfinite(h[0, :3]).all() and torch.isnan(h[0, 3:]).all() and torch.isnan(last).all()


def test_mingru_no_positions(tr):
    import torch
    h0, dl = torch.randn(3, 16, device="cuda"), torch.randn(3, 16, device="cuda")
    zh = torch.empty(3, 0, 32, device="cuda")
    h, last, states = tr.mingru_scan(zh, h0, save_states=True)
    assert h.shape == (3, 0, 16) and torch.equal(last, h0)
    dzh, dh0 = tr.mingru_scan_backward(zh, states, torch.empty(3, 0, 16, device="cuda"), dl)
    assert dzh.shape == zh.shape and torch.equal(dh0, dl)
    h, last = tr.mingru_scan(torch.empty(0, 5, 32, device="cuda"))
    assert h.shape == (0, 5, 16) and last.shape == (0, 16)


@pytest.mark.parametrize("T", [1, 20, 400])
def test_mingru_state_in_place_over_steps(tr, T):
    """A sequence in parts, its state updated in place, equals it in one call
    within the bound of the whole."""
    import torch
    zh, h0, _, _, _ = _case(torch, np.random.default_rng(8), 6, 3 * T, 32, "float32")
    ref = R.mingru(_n(zh), _n(h0), None)
    state, parts = h0.clone(), []
    for k in range(3):
        h, last = tr.mingru_scan(zh[:, k * T:(k + 1) * T], state, h_last=state)
        assert last is state
        parts.append(h)
    _close(torch.cat(parts, 1), *ref["h"], "float32")
    _close(state, *ref["last"], "float32")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,d", [(1, 700, 64), (1, 2000, 160), (2, 2049, 32), (3, 900, 33), (300, 40, 64)])
def test_mingru_states_in_place_both_ways(tr, dtype, B, T, d):
    """The state and its gradient updated in their own buffers give the bits
    of separate ones, with one block a group of chains and with several (which
    all read the buffer that one of them writes)."""
    import torch
    L = tr.lib()
    torch.manual_seed(T + d)
    r = lambda *s: torch.randn(*s, device="cuda")
    zh, dh = r(B, T, 2 * d).to(getattr(torch, dtype)), r(B, T, d).to(getattr(torch, dtype))
    h0, dl = r(B, d), r(B, d)
    h, last, saved = tr.mingru_scan(zh, h0, save_states=True)
    dzh, dh0 = tr.mingru_scan_backward(zh, saved, dh, dl)
    kind = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(20):
        s = h0.clone()
        h2, _ = tr.mingru_scan(zh, s, h_last=s)
        assert torch.equal(s, last) and torch.equal(h2, h)
        g, dzh2 = dl.clone(), torch.empty_like(dzh)
        assert L.boa_mingru_scan_backward(zh.data_ptr(), kind, 2 * d, T * 2 * d, B, T, d, None, saved.data_ptr(),
                                          dh.data_ptr(), d, T * d, g.data_ptr(), dzh2.data_ptr(), 2 * d, T * 2 * d,
                                          g.data_ptr(), stream) == 0
        assert torch.equal(g, dh0) and torch.equal(dzh2, dzh)


def test_mingru_takes_an_expanded_gradient(tr):
    import torch
    zh, h0, _, _, _ = _case(torch, np.random.default_rng(9), 4, 150, 32, "float32")
    _, _, states = tr.mingru_scan(zh, h0, save_states=True)
    one = torch.ones((), device="cuda").expand(4, 150, 32)
    a, b = tr.mingru_scan_backward(zh, states, one), tr.mingru_scan_backward(zh, states, one.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,T,d", [(3, 200, 24), (1, 1200, 160), (9, 515, 160), (3, 900, 64), (40, 77, 33), (2, 2049, 32),
                                   (200, 97, 96), (200, 300, 64)])
def test_mingru_writes_only_its_rows(tr, dtype, B, T, d):
    """Sequences that end inside a step of the kernels' walk: what lies before,
    behind and beside the rows is left alone."""
    import torch
    lengths = [T, T // 2, 0, T - 1][:B] + [T] * (B - 4)
    zh, h0, n, dh, dl = _case(torch, np.random.default_rng(10), B, T, d, dtype, lengths)
    margin = 600  # rows; more than a step of the walk may reach beyond the end
    out = torch.full((B, T + 2 * margin, d + 6), 7.0, dtype=zh.dtype, device="cuda")
    _, _, states = tr.mingru_scan(zh, h0, n, out=out[:, margin:margin + T, 3:3 + d], save_states=True)
    grad = torch.full((B, T + 2 * margin, 2 * d + 2), 7.0, dtype=zh.dtype, device="cuda")
    tr.mingru_scan_backward(zh, states, dh, dl, n, out=grad[:, margin:margin + T, 1:1 + 2 * d])
    for x, lo, hi in ((out, 3, 3 + d), (grad, 1, 1 + 2 * d)):
        assert not (x[:, margin:margin + T, lo:hi] == 7.0).all(-1).any()
        x[:, margin:margin + T, lo:hi] = 7.0
        assert (x == 7.0).all()


# --------------------------------------------------------------------- loss
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab,tok", [
    (1, 1, "int32"), (1, 256, "uint8"), (9, 256, "int64"), (1000, 256, "uint8"), (77, 255, "int32"),
    (33, 7, "int64"), (50, 264, "int32"), (64, 1000, "int64"), (129, 1024, "int32"), (5, 1023, "int32")])
def test_token_loss(tr, dtype, rows, vocab, tok):
    import torch
    rng = np.random.default_rng(rows + vocab)
    t, tt = _tokens(torch, rng, rows, vocab, tok)
    x = _t(torch, rng.normal(size=(rows, vocab)) * 4, dtype)
    w = rng.normal(size=rows).astype(np.float32)
    loss, grad = tr.token_loss(x, tt, inv_temperature=1.25, grad_scale=0.5, dloss=_t(torch, w))
    (rl, el), (rg, eg) = R.token_loss(_n(x), t, 1.25, 0.5 * w.astype(np.float64))
    assert loss.dtype == torch.float32 and grad.dtype == x.dtype
    _close(loss, rl, el, "float32", "loss")
    _close(grad, rg, eg, dtype, "gradient")
    only, none = tr.token_loss(x, tt, inv_temperature=1.25)
    assert none is None and torch.equal(only, loss)
    # in place: the gradient over the logits
    y = x.clone()
    _, inplace = tr.token_loss(y, tt, inv_temperature=1.25, grad_scale=0.5, dloss=_t(torch, w), out=y)
    assert inplace is y and torch.equal(y, grad)


@pytest.mark.parametrize("gap,offset", [(0, 1), (3, 0), (8, 0), (8, 4)])
@pytest.mark.parametrize("vocab", [256, 600])
def test_token_loss_strides_and_alignment(tr, gap, offset, vocab):
    import torch
    rng = np.random.default_rng(gap)
    t, tt = _tokens(torch, rng, 100, vocab, "int64")
    x = _strided(torch, _t(torch, rng.normal(size=(100, vocab)), "bfloat16"), gap, offset)
    out = _strided(torch, torch.zeros(100, vocab, dtype=torch.bfloat16, device="cuda"), gap, offset)
    loss, grad = tr.token_loss(x, tt, grad_scale=1.0, out=out)
    (rl, el), (rg, eg) = R.token_loss(_n(x), t, 1.0, np.ones(100))
    _close(loss, rl, el, "float32", "loss")
    _close(grad, rg, eg, "bfloat16", "gradient")
    if gap:
        assert torch.isnan(out.as_strided((99, gap), (vocab + gap, 1), out.storage_offset() + vocab)).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [256, 37])
def test_token_loss_masked_logits(tr, dtype, vocab):
    """Logits masked with -inf and with the type's lowest value; a masked
    target; a row of which nothing is left; a row of the lowest value alone."""
    import torch
    rng = np.random.default_rng(11)
    x = _t(torch, rng.normal(size=(6, vocab)), dtype)
    low = torch.finfo(x.dtype).min
    x[0, 5:] = -float("inf")
    x[1, ::2] = low
    x[2, 3] = -float("inf")          # the target itself
    x[3] = -float("inf")             # nothing is left
    x[4] = low                       # uniform
    x[5, :-1] = -float("inf")        # one symbol is left
    t = np.array([2, 1, 3, 0, 4, vocab - 1])
    for inv in (1.0, 3.0):
        loss, grad = tr.token_loss(x, _t(torch, t), inv_temperature=inv, grad_scale=1.0)
        (rl, el), (rg, eg) = R.token_loss(_n(x), t, inv, np.ones(6))
        _close(loss, rl, el, "float32", "loss")
        _close(grad, rg, eg, dtype, "gradient")
        assert loss[2] == float("inf") and loss[3] == float("inf") and (grad[3] == 0).all()
        assert loss[5] == 0 and (grad[5] == 0).all()


def test_token_loss_nan_and_padding(tr):
    import torch
    x = torch.randn(5, 256, device="cuda")
    x[1, 7], x[2, 9], x[3] = float("nan"), float("inf"), float("nan")
    t = torch.tensor([0, 1, 2, -1, 256], device="cuda")
    loss, grad = tr.token_loss(x, t, grad_scale=1.0)
    assert torch.isfinite(loss[0]) and torch.isfinite(grad[0]).all()
    assert torch.isnan(loss[1:3]).all() and torch.isnan(grad[1:3]).all()
    assert (loss[3:] == 0).all() and (grad[3:] == 0).all()


def test_token_loss_of_one_row_and_of_any_shape(tr):
    import torch
    x, t = torch.randn(2, 3, 256, device="cuda"), torch.randint(0, 256, (2, 3), device="cuda")
    loss, grad = tr.token_loss(x, t, grad_scale=2.0)
    flat = tr.token_loss(x.view(6, 256), t.view(6), grad_scale=2.0)
    assert torch.equal(loss.view(6), flat[0]) and torch.equal(grad.view(6, 256), flat[1])
    one = tr.token_loss(x[0, 0], t[0, 0], grad_scale=2.0)
    assert one[0].shape == () and torch.equal(one[0], loss[0, 0]) and torch.equal(one[1], grad[0, 0])
    # logits whose rows no stride reaches are copied; dloss expanded
    tt = tr.token_loss(x.transpose(0, 1), t.transpose(0, 1), grad_scale=2.0)
    assert torch.equal(tt[0], loss.t()) and torch.equal(tt[1], grad.transpose(0, 1))
    half = tr.token_loss(x, t, dloss=torch.full((), 2.0, device="cuda").expand(2, 3))
    assert torch.equal(half[1], grad)


def test_token_loss_empty(tr):
    import torch
    loss, grad = tr.token_loss(torch.empty(0, 3, 256, device="cuda"),
                               torch.empty(0, 3, dtype=torch.uint8, device="cuda"), grad_scale=1.0)
    assert loss.shape == (0, 3) and grad.shape == (0, 3, 256)


# ------------------------------------------------- streams, graphs, offsets
def _all_ops(tr, torch, s):
    x = tr.embed(s["tok"], s["E"], scale=2.0)
    h, last, states = tr.mingru_scan(s["zh"], s["h0"], s["n"], save_states=True)
    dzh, dh0 = tr.mingru_scan_backward(s["zh"], states, s["dh"], last, s["n"])
    loss, dx = tr.token_loss(s["x"], s["tok"], grad_scale=1.0)
    return [x, h, last, dzh, dh0, loss, dx, tr.embed_backward(s["tok"], x, 256)]


def _inputs(torch, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(tok=torch.randint(0, 256, (3, 700), generator=g, device="cuda", dtype=torch.uint8), E=r(256, 48),
                zh=r(3, 700, 96), h0=r(3, 48), n=torch.tensor([700, 300, 0], dtype=torch.int32, device="cuda"),
                dh=r(3, 700, 48), x=r(3, 700, 256))


def test_on_two_streams_at_once(tr):
    import torch
    ins = [_inputs(torch, k) for k in range(2)]
    want = [_all_ops(tr, torch, s) for s in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = _all_ops(tr, torch, ins[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_captured_and_replayed(tr):
    """Two graphs of the same calls, replayed with new contents in turn."""
    import torch
    ins = [_inputs(torch, k) for k in range(2)]
    other = [_inputs(torch, 10 + k) for k in range(2)]
    want = [_all_ops(tr, torch, s) for s in other]
    for s in ins:
        _all_ops(tr, torch, s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_ops(tr, torch, s))
        graphs.append(g)
    for s, o in zip(ins, other):
        for k in s:
            s[k].copy_(o[k])
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_offsets_past_32_bits(tr):
    """Rows whose element offsets pass 2^31 (and 2^32 bytes)."""
    import torch
    n, d = (1 << 31) // 512 + 1000, 512
    tok = torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda")
    E = torch.randn(256, d, device="cuda", dtype=torch.bfloat16)
    out = tr.embed(tok, E)
    assert torch.equal(out[-1200:], E[tok[-1200:].long()]) and torch.equal(out[:64], E[tok[:64].long()])
    tok[:-1000] = 255
    tok[-1000:] = torch.arange(1000, device="cuda") % 200
    got = tr.embed_backward(tok, out, 256)
    ref, err = R.embed_grad(_n(tok[-1000:]).astype(np.int64), _n(out[-1000:]), 256, 1.0)
    _close(got[:200], ref[:200], err[:200], "float32")
    # chunks further apart than 2^31 elements, and positions almost 2^32 bytes
    far = out.view(-1)
    for T, where in ((16, ((1 << 31) + 8, 512)), (2, (512, (1 << 31) - 8))):
        zh, h0, _, dh, dl = _case(torch, np.random.default_rng(1), 2, T, 256, "bfloat16")
        v = far.as_strided((2, T, 512), (*where, 1))
        v.copy_(zh)
        h, last, states = tr.mingru_scan(v, h0, save_states=True)
        a = tr.mingru_scan(zh, h0, save_states=True)
        assert torch.equal(h, a[0]) and torch.equal(last, a[1])
        b, c = tr.mingru_scan_backward(v, states, dh, dl), tr.mingru_scan_backward(zh, a[2], dh, dl)
        assert torch.equal(b[0], c[0]) and torch.equal(b[1], c[1])
    rows = n * d // 256
    x, t = out.view(rows, 256), torch.zeros(rows, dtype=torch.uint8, device="cuda")
    loss, grad = tr.token_loss(x, t, grad_scale=1.0)
    tail = tr.token_loss(x[-100:].clone(), t[-100:], grad_scale=1.0)
    assert torch.equal(loss[-100:], tail[0]) and torch.equal(grad[-100:], tail[1])


def test_on_another_device(tr):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two or more GPUs")
    s = _inputs(torch, 1)
    want = _all_ops(tr, torch, s)
    got = _all_ops(tr, torch, {k: v.to("cuda:1") for k, v in s.items()})
    assert torch.cuda.current_device() == 0
    for x, y in zip(want, got):
        assert torch.equal(x, y.to("cuda:0"))


def test_refused_on_the_gpu(tr, boa):
    import torch
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    tok = z(4, dtype=torch.uint8)
    zh, st = z(2, 5, 8), z(int(boa.lib().boa_mingru_states_floats(2, 5, 4)))
    for call in (
            lambda: tr.embed(tok, z(256, 8, dtype=torch.float64)), lambda: tr.embed(tok, z(1025, 8)),
            lambda: tr.embed(tok.short(), z(256, 8)), lambda: tr.embed(tok, z(256, 8).cpu()),
            lambda: tr.embed(tok, z(256, 8), out=z(4, 9)), lambda: tr.embed(tok, z(256, 8), out=z(8, 4).t()),
            lambda: tr.embed(tok, z(256, 8), out=z(1, 8).expand(4, 8)),
            lambda: tr.embed_backward(tok, z(5, 8), 256), lambda: tr.embed_backward(tok, z(4, 8), 256, accumulate=True),
            lambda: tr.embed_backward(tok, z(4, 8), 0), lambda: tr.embed_backward(tok, z(4, 8), 256, out=z(255, 8)),
            lambda: tr.mingru_scan(z(2, 5, 7)), lambda: tr.mingru_scan(zh, z(2, 5)),
            lambda: tr.mingru_scan(zh, z(2, 4, dtype=torch.float64)),
            lambda: tr.mingru_scan(zh, lengths=z(2, dtype=torch.int64)),
            lambda: tr.mingru_scan(zh, h_last=z(4, 2).t()), lambda: tr.mingru_scan(zh, out=z(2, 4, 5).transpose(1, 2)),
            lambda: tr.mingru_scan(zh, out=z(2, 1, 4).expand(2, 5, 4)),
            lambda: tr.mingru_scan_backward(zh, st[:-1], z(2, 5, 4)),
            lambda: tr.mingru_scan_backward(zh, st, z(2, 5, 4, dtype=torch.bfloat16)),
            lambda: tr.mingru_scan_backward(zh, st, z(2, 4, 4)),
            lambda: tr.token_loss(z(4, 1025), tok), lambda: tr.token_loss(z(4, 256), tok, inv_temperature=-1.0),
            lambda: tr.token_loss(z(4, 256), tok, dloss=z(5)), lambda: tr.token_loss(z(4, 256), tok, out=z(4, 255)),
            lambda: tr.token_loss(z(4, 256), tok, out=z(1, 256).expand(4, 256))):
        with pytest.raises(boa.BoaError) as e:
            call()
        assert e.value.code == boa.BOA_E_INVALID
    torch.cuda.synchronize()


# ------------------------------------------------------ the operators together
def _read_weights(torch, path, boa, d, L):
    raw = np.fromfile(path, np.float32, offset=4)
    w, o = {}, 0
    for name, shape, _ in boa.synth.weight_tensors("mingru", d, L):
        k = int(np.prod(shape))
        w[name], o = _t(torch, raw[o:o + k].reshape(shape)), o + k
    assert o == raw.size
    return w


def _predictor(torch, w, L, tok, embed, cell):
    """The framework's minGRU predictor around the given embedding and cell."""
    F = torch.nn.functional
    x = embed(tok, w["embedding.weight"])
    d = x.shape[-1]
    for i in range(L):
        p = f"blocks.{i}."
        y = F.layer_norm(x, (d,), w[p + "ln1.weight"], w[p + "ln1.bias"])
        zh = torch.cat((F.linear(y, w[p + "mingru.linear_z.weight"], w[p + "mingru.linear_z.bias"]),
                        F.linear(y, w[p + "mingru.linear_h.weight"], w[p + "mingru.linear_h.bias"])), -1)
        x = x + cell(zh)
        y = F.layer_norm(x, (d,), w[p + "ln2.weight"], w[p + "ln2.bias"])
        y = F.gelu(F.linear(y, w[p + "ff.0.weight"], w[p + "ff.0.bias"]), approximate="tanh")
        x = x + F.linear(y, w[p + "ff.2.weight"], w[p + "ff.2.bias"])
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w["final_norm.weight"]
    y = F.silu(F.linear(x, w["head.0.weight"], w["head.0.bias"]))
    return F.linear(y, w["head.2.weight"], w["head.2.bias"])


def test_operators_together_are_the_frameworks_predictor(tr, boa, weights):
    """The minGRU backbone rebuilt from these operators and torch products:
    its logits are those of Model.logits on the same weight file, within the
    framework's gate for logits (1e-3 of the largest), in one call and step by
    step; and the loss is the log-probability the coder codes with."""
    import torch
    d, L = 64, 2
    path = weights("mingru", d, L, 3, 0.1)
    m = boa.Model(path, "mingru", d, L)
    tok = np.random.default_rng(2).integers(0, 256, (5, 200), dtype=np.uint8)
    want = m.logits(tok, 0)
    w, tt = _read_weights(torch, path, boa, d, L), _t(torch, tok)
    got = _predictor(torch, w, L, tt, tr.embed, lambda zh: tr.mingru_scan(zh)[0])
    assert np.abs(_n(got) - want).max() <= 1e-3 * np.abs(want).max()
    # decode form: one position at a time, the states kept and updated in place
    state = [torch.zeros(5, d, device="cuda") for _ in range(L)]
    steps = []
    for t in range(20):
        k = iter(state)

        def cell(zh):
            s = next(k)
            return tr.mingru_scan(zh, s, h_last=s)[0]
        steps.append(_predictor(torch, w, L, tt[:, t:t + 1], tr.embed, cell))
    assert np.abs(_n(torch.cat(steps, 1)) - want[:, :20]).max() <= 1e-3 * np.abs(want).max()
    # the next byte's loss against the coder's own CDF of the same logits
    loss, _ = tr.token_loss(got[:, :-1], tt[:, 1:])
    Q = m.cdf_from_logits(_n(got[:, :-1]).astype(np.float32)).astype(np.int64)
    s = tok[:, 1:].reshape(-1).astype(int)
    f = (Q[np.arange(s.size), s + 1] - Q[np.arange(s.size), s]) / float(1 << 24)
    # f = p (1 - 256 / 2^24) + 2^-24 up to one step of the quantiser: relative to p >= 2^-14 here, 2^-9
    assert f.min() > 2.0 ** -14
    assert np.abs(-np.log(f) - _n(loss).reshape(-1)).max() < 2.0 ** -8


def test_operators_together_gradients(tr, boa, weights):
    """One training step's gradients of every weight, through these operators'
    forward and backward calls, against torch's in 64 bits."""
    import torch
    d, L, B, T = 64, 2, 3, 150
    w = _read_weights(torch, weights("mingru", d, L, 3, 0.1), boa, d, L)
    tok = _t(torch, np.random.default_rng(4).integers(0, 256, (B, T + 1), dtype=np.uint8))

    class Embed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, tok, E):
            ctx.save_for_backward(tok)
            return tr.embed(tok, E)

        @staticmethod
        def backward(ctx, g):
            return None, tr.embed_backward(ctx.saved_tensors[0], g, 256)

    class Cell(torch.autograd.Function):
        @staticmethod
        def forward(ctx, zh):
            h, _, states = tr.mingru_scan(zh, save_states=True)
            ctx.save_for_backward(zh, states)
            return h

        @staticmethod
        def backward(ctx, g):
            return tr.mingru_scan_backward(*ctx.saved_tensors, g)[0]

    def plain_cell(zh):
        zl, hr = zh.chunk(2, -1)
        z, c = torch.sigmoid(zl), torch.where(hr >= 0, hr + 0.5, torch.sigmoid(hr))
        h, out = torch.zeros_like(z[:, 0]), []
        for t in range(z.shape[1]):
            h = (1 - z[:, t]) * h + z[:, t] * c[:, t]
            out.append(h)
        return torch.stack(out, 1)

    a = {k: v.clone().requires_grad_() for k, v in w.items()}
    logits = _predictor(torch, a, L, tok[:, :-1], Embed.apply, Cell.apply)
    loss, dx = tr.token_loss(logits.detach(), tok[:, 1:], grad_scale=1.0 / (B * T))
    logits.backward(dx)
    b = {k: v.double().requires_grad_() for k, v in w.items()}
    ref = _predictor(torch, b, L, tok[:, :-1].long(), lambda t, E: E[t], plain_cell)
    mean = torch.nn.functional.cross_entropy(ref.flatten(0, 1), tok[:, 1:].long().flatten())
    mean.backward()
    assert abs(loss.double().mean().item() - mean.item()) < 1e-5 * mean.item()
    for k in w:
        x, y = a[k].grad.double(), b[k].grad
        # products of up to 4 d = 256 terms a layer in fp32 (torch's), ten of them in a row
        assert (x - y).norm() <= 10 * 256 * R.U * 16 * y.norm(), k
