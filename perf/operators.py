"""The operators of a byte predictor's training and stepping, measured case by case.

Each case is one call (or one forward and backward pair) of
``boa_b200.training``: the embedding lookup and its gradient, the minGRU
recurrence and its gradient, and the next-token loss with its gradient.
``own`` selects the package's kernels; without it ``run`` computes the same in
elementary torch operations.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TOK = {"u8": torch.uint8, "i32": torch.int32, "i64": torch.int64}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "u8": 1, "i32": 4, "i64": 8}
_WIDTHS = (64, 80, 128, 160, 256, 512)  # the widths of the framework's models


def _training():
    """boa_b200.training, the package loaded by path as its docstring says (its folder's name has a hyphen)."""
    if "boa_b200" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "boa-constrictor_b200")
        spec = importlib.util.spec_from_file_location("boa_b200", os.path.join(at, "__init__.py"),
                                                      submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["boa_b200"] = mod
        spec.loader.exec_module(mod)
    from boa_b200 import training
    return training


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a full batch: one byte for each of 16384 chunks
        dict(name="embed_step", op="embed", n=16384, d=256, vocab=256, tok="u8", table="f32", out="f32", scale=1.0),
        # one 64-position tile of that batch, the widest model, mixed precision: a master table, bf16 activations
        dict(name="embed_tile_bf16", op="embed", n=16384 * 64, d=512, vocab=256, tok="u8", table="f32", out="bf16", scale=22.627417),
        # gradient of a small fine-tuning batch
        dict(name="embed_grad_small", op="embed_grad", n=4096, d=64, vocab=256, tok="u8", dout="f32", scale=1.0),
        # a wider alphabet with padding, an odd number of tokens
        dict(name="embed_grad_wide", op="embed_grad", n=100003, d=160, vocab=1000, tok="i64", dout="bf16", scale=12.649111),
        # gradient of a 64-position tile of a full batch
        dict(name="embed_grad_tile", op="embed_grad", n=16384 * 64, d=256, vocab=256, tok="u8", dout="f32", scale=1.0),
        # one decode step of a full batch: the state of every chunk is read and replaced
        dict(name="scan_step", op="scan", B=16384, T=1, d=256, dt="f32", ragged=False),
        # ordinary training batch, forward alone (evaluation)
        dict(name="scan_eval_bf16", op="scan", B=32, T=4096, d=256, dt="bf16", ragged=False),
        # one long stream: little parallelism beside the time axis
        dict(name="scan_long", op="scan", B=1, T=262144, d=512, dt="f32", ragged=False),
        # a small batch of the narrow width with ragged chunks, forward and backward
        dict(name="scan_train_ragged", op="scan_train", B=24, T=2047, d=160, dt="f32", ragged=True),
        # ordinary training batch, forward and backward
        dict(name="scan_train_bf16", op="scan_train", B=64, T=4096, d=256, dt="bf16", ragged=False),
        # loss of a small batch
        dict(name="loss_small", op="loss", rows=4096, vocab=256, tok="u8", dt="bf16", grad=True, inv_t=1.0),
        # loss and gradient of a 64-position tile of a full batch
        dict(name="loss_tile", op="loss", rows=16384 * 64, vocab=256, tok="u8", dt="f32", grad=True, inv_t=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("embed", "embed_grad", "scan", "scan", "scan_train", "scan_train", "loss"))
    if op in ("embed", "embed_grad"):
        vocab = rng.choice((256, 256, rng.randint(2, 1024)))
        tok = rng.choice(("u8", "i32", "i64")) if vocab == 256 else rng.choice(("i32", "i64"))
        d = rng.choice(_WIDTHS + (rng.randint(1, 600), rng.randint(1, 600)))
        n = min(_log(rng, 1, 1 << 20), int(1.0e9 // (4 * d)))
        scale = rng.choice((1.0, math.sqrt(d)))
        if op == "embed":
            return dict(op=op, n=n, d=d, vocab=vocab, tok=tok, table=rng.choice(tuple(_DT)), out=rng.choice(tuple(_DT)), scale=scale)
        return dict(op=op, n=n, d=d, vocab=vocab, tok=tok, dout=rng.choice(tuple(_DT)), scale=scale)
    if op in ("scan", "scan_train"):
        d = rng.choice(_WIDTHS + (rng.randint(1, 600),))
        dt = rng.choice(tuple(_DT))
        cells = _log(rng, 64, 1 << 18)  # positions of the batch
        T = min(_log(rng, 1, min(cells, 1 << 17)), (1 << 25) // d)
        B = min(max(1, cells // T), max(1, (1 << 25) // (T * d)))
        return dict(op=op, B=B, T=T, d=d, dt=dt, ragged=B > 3 and rng.random() < 0.5)
    vocab = rng.choice((256, 256, rng.randint(2, 1024)))
    tok = rng.choice(("u8", "i32", "i64")) if vocab == 256 else rng.choice(("i32", "i64"))
    rows = min(_log(rng, 1, 1 << 20), int(1.0e9 // (4 * vocab)))
    return dict(op=op, rows=rows, vocab=vocab, tok=tok, dt=rng.choice(tuple(_DT)), grad=rng.random() < 0.8,
                inv_t=rng.choice((1.0, 1.0, 1.25)))


def _lengths(case):
    """Positions of each chunk: all of them, or 0, 1 and the rest spread over [0, T]."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    return [(0, 1, T)[i] if i < 3 else (i * 2654435761 % 4294967296) * (T + 1) >> 32 for i in range(B)]


def work(case):
    op = case["op"]
    if op in ("embed", "embed_grad"):
        n, d, V = case["n"], case["d"], case["vocab"]
        if op == "embed":
            # tokens in, the rows of the table that can be named, rows out
            return {"bytes": n * _SIZE[case["tok"]] + min(n, V) * d * _SIZE[case["table"]] + n * d * _SIZE[case["out"]], "flops": n * d}
        return {"bytes": n * _SIZE[case["tok"]] + n * d * _SIZE[case["dout"]] + V * d * 4, "flops": n * d}
    if op in ("scan", "scan_train"):
        B, T, d, s = case["B"], case["T"], case["d"], _SIZE[case["dt"]]
        live, rows = sum(_lengths(case)) * d, B * T * d
        # forward: gates and candidates in, states out, the state before and after
        by, fl = (2 * live + rows) * s + 8 * B * d, 12 * live
        if op == "scan_train":
            # backward: gates, candidates and the states' gradient in, their gradients out, the state's gradients
            by, fl = by + (3 * live + 2 * rows) * s + 8 * B * d, fl + 24 * live
        return {"bytes": by, "flops": fl}
    rows, V, s = case["rows"], case["vocab"], _SIZE[case["dt"]]
    return {"bytes": rows * (V * s * (2 if case["grad"] else 1) + _SIZE[case["tok"]] + 4), "flops": rows * V * (6 if case["grad"] else 4)}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(g, n, vocab, tok, pad):
    if vocab == 256:  # bytes of binary records: exponent bytes few, mantissa bytes many
        x = torch.randn((n + 3) // 4, generator=g, device="cuda").view(torch.uint8)[:n]
        x = x if tok == "u8" else x.to(_TOK[tok])
    else:  # a wider alphabet, its low symbols more frequent
        x = (torch.rand(n, generator=g, device="cuda").square() * vocab).to(_TOK[tok]).clamp_(0, vocab - 1)
    if pad and tok != "u8":  # positions that pad a batch carry -1
        x = torch.where(torch.rand(n, generator=g, device="cuda") < 0.02, torch.full_like(x, -1), x)
    return x.clone()


def _normal(g, shape, dt, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(_DT[dt])


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("embed", "embed_grad"):
        s["tok"] = _tokens(g, case["n"], case["vocab"], case["tok"], True)
        if op == "embed":
            s["table"] = _normal(g, (case["vocab"], case["d"]), case["table"], 0.02)
        else:
            s["dout"] = _normal(g, (case["n"], case["d"]), case["dout"], 1e-2)
    elif op in ("scan", "scan_train"):
        B, T, d, dt = case["B"], case["T"], case["d"], case["dt"]
        # gates lean towards keeping the state, as trained ones do
        s["zh"] = torch.cat((_normal(g, (B, T, d), dt, 1.5) - 1.0, _normal(g, (B, T, d), dt)), dim=2)
        s["h0"] = torch.rand((B, d), generator=g, device="cuda")
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        if op == "scan_train":
            s["dh"] = _normal(g, (B, T, d), dt, 1e-2)
            s["dlast"] = torch.randn((B, d), generator=g, device="cuda") * 1e-2
    else:
        rows, V = case["rows"], case["vocab"]
        s["x"] = _normal(g, (rows, V), case["dt"], 2.0)
        s["tok"] = _tokens(g, rows, V, case["tok"], True)
        s["gscale"] = 1.0 if case["dt"] == "f16" else 1.0 / rows  # the mean; the sum in fp16, whose range ends early
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    ops, c = _training(), s["case"]
    op = c["op"]
    if op == "embed":
        return [ops.embed(s["tok"], s["table"], scale=c["scale"], dtype=_DT[c["out"]])]
    if op == "embed_grad":
        return [ops.embed_backward(s["tok"], s["dout"], c["vocab"], scale=c["scale"])]
    if op == "scan":
        return list(ops.mingru_scan(s["zh"], s["h0"], s["lengths"]))
    if op == "scan_train":
        h, last, states = ops.mingru_scan(s["zh"], s["h0"], s["lengths"], save_states=True)
        return [h, last, *ops.mingru_scan_backward(s["zh"], states, s["dh"], s["dlast"], s["lengths"])]
    loss, grad = ops.token_loss(s["x"], s["tok"], inv_temperature=c["inv_t"], grad_scale=s["gscale"] if c["grad"] else None)
    return [loss, grad] if c["grad"] else [loss]


def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 by doubling."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), dim=1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), dim=1)
        k *= 2
    return b


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "embed":
        t = s["tok"].long()
        ok = (t >= 0) & (t < c["vocab"])
        rows = s["table"].float()[torch.where(ok, t, 0)] * c["scale"]
        return [torch.where(ok[:, None], rows, 0.0).to(_DT[c["out"]])]
    if op == "embed_grad":
        t = s["tok"].long()
        ok = (t >= 0) & (t < c["vocab"])
        # long sums of values of either sign: in 64 bits
        total = torch.zeros(c["vocab"] + 1, c["d"], dtype=torch.float64, device="cuda")
        total.index_add_(0, torch.where(ok, t, c["vocab"]), s["dout"].double())
        return [(total[:-1] * c["scale"]).float()]
    if op in ("scan", "scan_train"):
        return _plain_scan(s)
    x = s["x"].float()
    t = s["tok"].long()
    ok = (t >= 0) & (t < c["vocab"])
    t = torch.where(ok, t, 0)
    x = (x - x.max(dim=1, keepdim=True).values) * c["inv_t"]
    e = torch.exp(x)
    total = e.sum(dim=1, keepdim=True)
    loss = torch.where(ok, (torch.log(total) - x.gather(1, t[:, None]))[:, 0], 0.0)
    if not c["grad"]:
        return [loss]
    grad = e / total
    grad.scatter_add_(1, t[:, None], torch.full_like(total, -1.0))
    grad = torch.where(ok[:, None], grad * (s["gscale"] * c["inv_t"]), 0.0)
    return [loss, grad.to(_DT[c["dt"]])]


def _plain_scan(s):
    c = s["case"]
    B, T, d, dt = c["B"], c["T"], c["d"], _DT[c["dt"]]
    zl, hr = s["zh"].float().split(d, dim=2)
    z = 1.0 / (1.0 + torch.exp(-zl))
    keep = 1.0 / (1.0 + torch.exp(zl))  # 1 - z
    ht = torch.where(hr >= 0, hr + 0.5, 1.0 / (1.0 + torch.exp(-hr)))
    a, b = keep, z * ht
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(T, device="cuda")[None, :] < s["lengths"][:, None])[:, :, None]
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    first = b[:, :1] + a[:, :1] * s["h0"][:, None]
    h = _linear_scan(a, torch.cat((first, b[:, 1:]), dim=1))
    last = h[:, -1].contiguous()
    out = h if live is None else torch.where(live, h, 0.0)
    if c["op"] == "scan":
        return [out.to(dt), last]
    dh = s["dh"].float()
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    # gradient that reaches each state: of its own output, and of the next state through its gate
    dh = torch.cat((dh[:, :-1], dh[:, -1:] + s["dlast"][:, None]), dim=1)
    nxt = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), dim=1)
    g = _linear_scan(nxt.flip(1), dh.flip(1)).flip(1)
    before = torch.cat((s["h0"][:, None], h[:, :-1]), dim=1)
    dz = g * (ht - before) * z * keep
    dr = g * z * torch.where(hr >= 0, 1.0, ht / (1.0 + torch.exp(hr)))
    if live is not None:
        dz, dr = torch.where(live, dz, 0.0), torch.where(live, dr, 0.0)
    return [out.to(dt), last, torch.cat((dz, dr), dim=2).to(dt), (a[:, 0] * g[:, 0]).contiguous()]


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f8, op = torch.float64, case["op"]
    if op == "embed":
        t, E = s["tok"].to(torch.int64), s["table"].to(f8)
        E = torch.cat((E * case["scale"], torch.zeros_like(E[:1])))  # the last row for tokens outside the alphabet
        t[(t < 0) | (t >= case["vocab"])] = case["vocab"]
        return [E.index_select(0, t)]
    if op == "embed_grad":
        # running sums over the rows in token order, and their differences at the tokens' borders, a few columns at a time
        t = s["tok"].to(torch.int64)
        t[(t < 0) | (t >= case["vocab"])] = case["vocab"]
        t, order = torch.sort(t, stable=True)
        cut = torch.searchsorted(t, torch.arange(case["vocab"] + 1, device="cuda"))
        cols = []
        for c0 in range(0, case["d"], 64):
            run_ = torch.cumsum(s["dout"][:, c0:c0 + 64].to(f8)[order], dim=0)
            run_ = torch.cat((torch.zeros_like(run_[:1]), run_))
            cols.append((run_[cut[1:]] - run_[cut[:-1]]) * case["scale"])
        return [torch.cat(cols, dim=1)]
    if op in ("scan", "scan_train"):
        return _exact_scan(case, s)
    x, t = s["x"].to(f8) * case["inv_t"], s["tok"].to(torch.int64)
    off = (t < 0) | (t >= case["vocab"])
    t[off] = 0
    logp = x - torch.logsumexp(x, dim=1, keepdim=True)
    loss = -logp[torch.arange(len(t), device="cuda"), t]
    loss[off] = 0
    if not case["grad"]:
        return [loss]
    grad = logp.exp_()
    grad[torch.arange(len(t), device="cuda"), t] -= 1
    grad[off] = 0
    return [loss, grad * (s["gscale"] * case["inv_t"])]


def _exact_scan(case, s):
    """Position by position, forward and then back; the gates of a block of positions at once."""
    f8, B, T, d, block = torch.float64, case["B"], case["T"], case["d"], 1024
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    past = torch.arange(T, device="cuda")[:, None] >= lengths[None, :]  # [T, B]

    def gates(t0, t1):
        z, r = (v.transpose(0, 1).to(f8).contiguous() for v in s["zh"][:, t0:t1].split(d, dim=2))
        z = torch.sigmoid(z)
        z[past[t0:t1]] = 0  # a gate of zero keeps the state
        return z, r, torch.where(r < 0, torch.sigmoid(r), r + 0.5)

    states = torch.empty(T + 1, B, d, dtype=f8, device="cuda")
    states[0] = s["h0"]
    for t0 in range(0, T, block):
        z, _, cand = gates(t0, min(T, t0 + block))
        for k in range(z.shape[0]):
            torch.lerp(states[t0 + k], cand[k], z[k], out=states[t0 + k + 1])
    out = states[1:].clone()
    out[past] = 0
    if case["op"] == "scan":
        return [out.transpose(0, 1).contiguous(), states[T]]
    g = s["dlast"].to(f8)
    grad = torch.empty(T, B, 2 * d, dtype=f8, device="cuda")
    for t0 in range((T - 1) // block * block, -1, -block):
        z, r, cand = gates(t0, min(T, t0 + block))
        dh = s["dh"][:, t0:t0 + block].transpose(0, 1).to(f8).contiguous()
        dh[past[t0:t0 + block]] = 0
        reach, keep = torch.empty_like(dh), 1 - z
        for k in range(z.shape[0] - 1, -1, -1):
            torch.add(g, dh[k], out=reach[k])
            g = reach[k] * keep[k]
        grad[t0:t0 + block, :, :d] = reach * (cand - states[t0:t0 + z.shape[0]]) * z * keep
        grad[t0:t0 + block, :, d:] = reach * z * torch.where(r < 0, cand * (1 - cand), 1.0)
    return [out.transpose(0, 1).contiguous(), states[T], grad.transpose(0, 1).contiguous(), g]
