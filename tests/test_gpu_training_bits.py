"""What a codec may rely on: calls of the minGRU recurrence (boa_b200.training)
of up to 8 positions agree bit by bit, however a sequence is cut into them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


def _run(tr, torch, zh, h0, cuts, lengths=None):
    """Sequential calls of cuts[0], cuts[1] .. positions, the state carried."""
    state, parts, at = h0.clone(), [], 0
    for k in cuts:
        left = None if lengths is None else (lengths - at).clamp(0, k).int()
        h, _ = tr.mingru_scan(zh[:, at:at + k], state, left, h_last=state)
        parts.append(h)
        at += k
    assert at == zh.shape[1]
    return torch.cat(parts, 1), state


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,d", [(1, 1), (3, 33), (2, 64), (700, 80), (5, 257)])
@pytest.mark.parametrize("ragged", [False, True])
def test_any_cut_into_short_calls_gives_the_same_bits(tr, dtype, B, d, ragged):
    import torch
    g = torch.Generator(device="cuda").manual_seed(B + d)
    T = 40
    zh = (torch.randn(B, T, 2 * d, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    h0 = torch.randn(B, d, generator=g, device="cuda")
    n = torch.randint(0, T + 1, (B,), generator=g, device="cuda") if ragged else None
    h, last = _run(tr, torch, zh, h0, [1] * T, n)
    rng = np.random.default_rng(B)
    for cuts in ([8] * 5, [2] * 20, [3, 8, 1, 7, 5, 8, 8], rng.multinomial(T - 16, np.ones(8) / 8).clip(0, 6)):
        cuts = [int(c) for c in cuts if c]
        while sum(cuts) < T:
            cuts.append(min(8, T - sum(cuts)))
        a, b = _run(tr, torch, zh, h0, cuts, n)
        assert torch.equal(a, h) and torch.equal(b, last), cuts
    # positions far apart, and rows off the 4- and 16-byte grid
    for wide in (torch.empty(B, T, 2 * d + 16, dtype=zh.dtype, device="cuda")[:, :, 8:8 + 2 * d],
                 torch.empty(B, T, 2 * d + 3, dtype=zh.dtype, device="cuda")[:, :, 1:1 + 2 * d],
                 torch.empty(T, B, 2 * d, dtype=zh.dtype, device="cuda").transpose(0, 1)):
        wide.copy_(zh)
        a, b = _run(tr, torch, wide, h0, [8] * 5, n)
        assert torch.equal(a, h) and torch.equal(b, last)
    # some of the chunks alone
    few = slice(B // 2, B // 2 + 1)
    a, b = _run(tr, torch, zh[few], h0[few], [5] * 8, None if n is None else n[few])
    assert torch.equal(a, h[few]) and torch.equal(b, last[few])
