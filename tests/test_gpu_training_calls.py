"""How the training operators (boa_b200.training) are called: from several
threads at once, in one captured graph, after a call that failed."""
import ctypes as C
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

KIND = {"float32": 0, "float16": 1, "bfloat16": 2}


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


def _scan_call(tr, torch, B, T, d, dtype, back, seed=0):
    """-> (call(stream) -> status, the tensors that it writes)"""
    L, g = tr.lib(), torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    zh, dh = r(B, T, 2 * d).to(getattr(torch, dtype)), r(B, T, d).to(getattr(torch, dtype))
    h, saved = torch.empty_like(dh), torch.empty(L.boa_mingru_states_floats(B, T, d), device="cuda")
    last, dzh, dh0 = r(B, d), torch.empty_like(zh), r(B, d)
    k, w = KIND[dtype], 2 * d

    def forward(st):
        return L.boa_mingru_scan(zh.data_ptr(), k, w, T * w, B, T, d, None, None, h.data_ptr(), d, T * d,
                                 last.data_ptr(), saved.data_ptr(), st)

    def backward(st):
        return L.boa_mingru_scan_backward(zh.data_ptr(), k, w, T * w, B, T, d, None, saved.data_ptr(), dh.data_ptr(),
                                          d, T * d, None, dzh.data_ptr(), w, T * w, dh0.data_ptr(), st)
    assert forward(torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return (backward, [dzh, dh0]) if back else (forward, [h, last, saved])


def _grad_call(tr, torch, n, vocab, d, seed=0):
    L, g = tr.lib(), torch.Generator(device="cuda").manual_seed(seed)
    tok = torch.randint(0, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    dout = torch.randn(n, d, generator=g, device="cuda")
    out = torch.empty(vocab, d, device="cuda")
    ws = torch.empty(L.boa_embed_backward_workspace(n, vocab, d), dtype=torch.uint8, device="cuda")

    def call(st):
        return L.boa_embed_backward(tok.data_ptr(), 1, n, dout.data_ptr(), 0, d, vocab, d, 1.0, 0, out.data_ptr(), 0, d,
                                    ws.data_ptr(), ws.numel(), st)
    return call, [out]


# two shapes of one kernel that need different amounts of shared memory
PAIRS = {
    "scan_f32": lambda tr, t: (_scan_call(tr, t, 8, 700, 256, "float32", False), _scan_call(tr, t, 75, 64, 64, "float32", False)),
    "scan_bf16": lambda tr, t: (_scan_call(tr, t, 16, 700, 256, "bfloat16", False), _scan_call(tr, t, 150, 64, 64, "bfloat16", False)),
    "back_f32": lambda tr, t: (_scan_call(tr, t, 8, 700, 256, "float32", True), _scan_call(tr, t, 75, 64, 64, "float32", True)),
    "back_bf16": lambda tr, t: (_scan_call(tr, t, 16, 700, 256, "bfloat16", True), _scan_call(tr, t, 150, 64, 64, "bfloat16", True)),
    "narrow_f32": lambda tr, t: (_scan_call(tr, t, 1, 3000, 64, "float32", False), _scan_call(tr, t, 1, 20, 64, "float32", False)),
    "table": lambda tr, t: (_grad_call(tr, t, 5000, 1024, 8), _grad_call(tr, t, 5000, 16, 8)),
}


@pytest.mark.parametrize("pair", PAIRS)
def test_two_threads_launch_different_shapes(tr, boa, pair):
    """Calls of one kernel with much and with little shared memory, from two
    threads at once: neither fails, and both give what they give alone."""
    import torch
    calls = PAIRS[pair](tr, torch)
    main = torch.cuda.current_stream().cuda_stream
    want = []
    for call, outs in calls:
        assert call(main) == 0
        torch.cuda.synchronize()
        want.append([x.clone() for x in outs])
    streams, failed = [torch.cuda.Stream() for _ in calls], []
    torch.cuda.synchronize()
    ready = threading.Barrier(len(calls))

    def work(k):
        torch.cuda.set_device(0)
        call, st = calls[k][0], streams[k].cuda_stream
        ready.wait()
        for i in range(3000):
            rc = call(st)
            if rc != 0:
                failed.append((k, i, rc, tr.lib().boa_last_error(None)))
                break
            if i % 256 == 255:
                streams[k].synchronize()
    ts = [threading.Thread(target=work, args=(k,)) for k in range(len(calls))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert not failed, failed
    for (_, outs), ref in zip(calls, want):
        for x, y in zip(outs, ref):
            assert torch.equal(x, y)


@pytest.mark.parametrize("pair", PAIRS)
def test_different_shapes_in_one_graph(tr, pair):
    """A graph that holds a launch with much shared memory, then one with
    little, is instantiated after both."""
    import torch
    calls = PAIRS[pair](tr, torch)
    s = torch.cuda.Stream()
    for call, _ in calls:
        assert call(s.cuda_stream) == 0
    s.synchronize()
    want = [[x.clone() for x in outs] for _, outs in calls]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for call, _ in calls:
            assert call(s.cuda_stream) == 0
    for _, outs in calls:
        [x.zero_() for x in outs]
    g.replay()
    torch.cuda.synchronize()
    for (_, outs), ref in zip(calls, want):
        for x, y in zip(outs, ref):
            assert torch.equal(x, y)


class _Driver:
    """The few driver calls that a stream capture needs, on a stream of its own."""

    def __init__(self):
        self.cu = C.CDLL("libcuda.so.1")
        self.stream = C.c_void_p()
        assert self.cu.cuStreamCreate(C.byref(self.stream), 0) == 0  # waits on the legacy stream, and it on this one

    def begin(self):
        assert self.cu.cuStreamBeginCapture_v2(self.stream, 0) == 0

    def end(self):
        graph = C.c_void_p()
        rc = self.cu.cuStreamEndCapture(self.stream, C.byref(graph))
        if graph.value:
            self.cu.cuGraphDestroy(graph)
        return rc


@pytest.mark.parametrize("failing", ["scan", "back", "table", "small_table", "step"])
@pytest.mark.parametrize("then", ["scan", "table", "step"])
def test_a_failed_launch_is_not_a_later_calls_error(tr, boa, failing, then):
    """A launch into the legacy stream while another stream that waits on it is
    captured is refused by the driver; the next call is sound again."""
    import torch
    make = {"scan": lambda: _scan_call(tr, torch, 2, 100, 32, "float32", False),
            "back": lambda: _scan_call(tr, torch, 2, 100, 32, "float32", True),
            "step": lambda: _scan_call(tr, torch, 2, 1, 32, "float32", False),
            "table": lambda: _grad_call(tr, torch, 5000, 64, 8), "small_table": lambda: _grad_call(tr, torch, 50, 64, 8)}
    bad, (good, outs) = make[failing]()[0], make[then]()
    main = torch.cuda.current_stream().cuda_stream
    assert good(main) == 0
    torch.cuda.synchronize()
    want = [x.clone() for x in outs]
    torch.cuda.synchronize()
    drv = _Driver()
    drv.begin()
    rc = bad(None)
    ended = drv.end()
    assert rc == boa.BOA_E_CUDA and ended != 0, (rc, ended)
    assert b"captur" in tr.lib().boa_last_error(None)
    for _ in range(2):
        assert good(main) == 0, tr.lib().boa_last_error(None)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_an_earlier_failure_elsewhere_is_not_this_calls_error(tr, boa):
    import torch
    call, _ = _scan_call(tr, torch, 2, 1, 32, "float32", False)
    with pytest.raises(boa.BoaError):
        boa.Model("/nonexistent.bin", "mingru", 64, 2, device=99)
    assert call(torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("silent", [0, 1, 2, 3, 5, 8])
def test_a_wait_that_runs_out_gives_nan_and_nothing_else(tr, boa, silent):
    """One of two blocks falls silent: from then on every state is NaN, before
    it every state is right, the kernel ends soon and the context goes on."""
    import time
    import torch
    call, outs = _scan_call(tr, torch, 1, 700, 64, "float32", False)  # by clusters
    torch.cuda.synchronize()
    want = [x.clone() for x in outs]
    got = np.zeros((8, 2, 2, 32), np.float32)
    t0 = time.monotonic()
    rc = tr.lib().boa_selftest_walk_timeout(0, 8, silent, 20000, got.ctypes.data_as(C.POINTER(C.c_float)))
    assert rc == 0 and time.monotonic() - t0 < 5
    step, block, team, _ = np.indices(got.shape)
    assert np.isnan(got[silent:]).all()
    assert (got[:silent] == (4 * step + 2 * block + team)[:silent]).all()
    assert call(torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_wrapped_in_an_autograd_function(tr, boa):
    """The recurrence as a differentiable function: its first derivative is
    that of the calls, a second one is refused, not silently zero."""
    import torch
    from torch.autograd.function import once_differentiable

    class Cell(torch.autograd.Function):
        @staticmethod
        def forward(ctx, zh):
            h, _, saved = tr.mingru_scan(zh, save_states=True)
            ctx.save_for_backward(zh, saved)
            return h

        @staticmethod
        @once_differentiable
        def backward(ctx, dh):
            return tr.mingru_scan_backward(*ctx.saved_tensors, dh)[0]

    class Unmarked(Cell):
        @staticmethod
        def backward(ctx, dh):
            return tr.mingru_scan_backward(*ctx.saved_tensors, dh)[0]
    zh = torch.randn(2, 50, 32, device="cuda", requires_grad=True)
    dh = torch.randn(2, 50, 16, device="cuda")
    with torch.no_grad():
        _, _, saved = tr.mingru_scan(zh, save_states=True)
        want = tr.mingru_scan_backward(zh, saved, dh)[0]
    assert torch.equal(torch.autograd.grad(Cell.apply(zh), zh, dh)[0], want)
    g, = torch.autograd.grad(Cell.apply(zh), zh, dh, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), zh)
    with pytest.raises(boa.BoaError, match="zh requires a gradient"):
        torch.autograd.grad(Unmarked.apply(zh), zh, dh, create_graph=True)
    with pytest.raises(boa.BoaError, match="zh requires a gradient"):
        tr.mingru_scan(zh)


def _writers(tr, torch):
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    tok = torch.randint(0, 8, (6,), device="cuda")
    zh, h0 = r(2, 5, 8), r(2, 4)
    saved = tr.mingru_scan(zh, h0, save_states=True)[2]
    return {
        "embed": ((6, 4), lambda y: tr.embed(tok, r(8, 4), out=y)),
        "embed_backward": ((8, 4), lambda y: tr.embed_backward(tok, r(6, 4), 8, out=y)),
        "accumulate": ((8, 4), lambda y: tr.embed_backward(tok, r(6, 4), 8, out=y, accumulate=True)),
        "scan": ((2, 5, 4), lambda y: tr.mingru_scan(zh, h0, out=y)),
        "state": ((2, 4), lambda y: tr.mingru_scan(zh, y, h_last=y)),
        "scan_backward": ((2, 5, 8), lambda y: tr.mingru_scan_backward(zh, saved, r(2, 5, 4), out=y)),
        "loss": ((6, 8), lambda y: tr.token_loss(y, tok, out=y)),
    }


@pytest.mark.parametrize("name", ["embed", "embed_backward", "accumulate", "scan", "state", "scan_backward", "loss"])
def test_a_saved_tensor_that_is_written_is_noticed(tr, name):
    """exp saves its result for its gradient: written over by one of these
    calls, torch refuses the backward pass, as after an in-place operation."""
    import torch
    shape, write = _writers(tr, torch)[name]
    a = torch.randn(shape, device="cuda", requires_grad=True)
    y = a.exp()
    write(y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():  # tensors without versions are written all the same
        z = torch.full(shape, 0.5, device="cuda")
        write(z)
        assert not (z == 0.5).all()


def _negative(torch, *shape):
    """A real view whose sign torch keeps aside, and the same values in memory."""
    x = torch.view_as_complex(torch.randn(*shape, 2, device="cuda")).conj().imag
    assert x.is_neg()
    return x, x.clone().resolve_neg()


def test_negative_views_keep_their_sign(tr, boa):
    import torch
    tok = torch.randint(0, 8, (6,), device="cuda")
    t, h0, dl, w = (_negative(torch, *s) for s in ((8, 4), (2, 4), (2, 4), (6,)))
    x, zh, dh, g = (_negative(torch, *s) for s in ((6, 8), (2, 5, 8), (2, 5, 4), (6, 4)))
    saved = tr.mingru_scan(zh[1], h0[1], save_states=True)[2]
    both = [[tr.embed(tok, t[k]), tr.embed_backward(tok, g[k], 8), *tr.mingru_scan(zh[k], h0[k]),
             *tr.mingru_scan_backward(zh[k], saved, dh[k], dl[k]), *tr.token_loss(x[k], tok, dloss=w[k])] for k in (0, 1)]
    for a, b in zip(*both):
        assert not a.is_neg() and torch.equal(a, b)
    for write in (lambda: tr.embed(tok, t[1], out=g[0]), lambda: tr.embed_backward(tok, g[1], 8, out=t[0]),
                  lambda: tr.mingru_scan(zh[1], out=dh[0]), lambda: tr.mingru_scan(zh[1], h_last=h0[0]),
                  lambda: tr.mingru_scan_backward(zh[1], saved, dh[1], out=zh[0]),
                  lambda: tr.token_loss(x[1], tok, out=x[0])):
        with pytest.raises(boa.BoaError, match="negative view"):
            write()


def test_sizes_past_a_c_int_are_refused(tr, boa):
    """Not taken by their low halves.  Views of one element, and of none."""
    import torch
    far = (1 << 32) + 8
    tok, one = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, device="cuda")
    none = torch.zeros(1, 0, 2, device="cuda")
    h0 = torch.zeros(1, 1, device="cuda")
    for call in (lambda: tr.embed(tok, one.expand(far, 1)), lambda: tr.embed(tok[:0], one.expand(1, far)),
                 lambda: tr.embed_backward(tok, torch.zeros(4, 1, device="cuda"), far),
                 lambda: tr.embed_backward(tok[:0], torch.zeros(0, 1, device="cuda").expand(0, far), 1),
                 lambda: tr.mingru_scan(none.expand(far, 0, 2)),
                 lambda: tr.mingru_scan(one[None].half().expand(1, far, 2)),
                 lambda: tr.mingru_scan_backward(none.expand(far, 0, 2), none, none.expand(far, 0, 2)[..., :1], h0),
                 lambda: tr.token_loss(torch.zeros(0, 1, device="cuda").expand(0, far), tok[:0])):
        before = torch.cuda.memory_allocated()
        with pytest.raises(boa.BoaError, match="below 2"):
            call()
        assert torch.cuda.memory_allocated() == before
