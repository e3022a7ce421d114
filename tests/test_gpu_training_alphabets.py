"""The table gradient (boa_b200.training) with alphabets that end inside a
warp, at the sizes where one cluster of blocks sorts the tokens."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


@pytest.mark.parametrize("n", [4097, 20011, 49152])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 63, 100, 257, 1000, 1023])
def test_alphabets_that_end_inside_a_warp(tr, n, vocab):
    """Sums of small whole numbers, which fp32 holds exactly."""
    import torch
    rng = np.random.default_rng(n + vocab)
    tok = torch.from_numpy(rng.integers(-1, vocab + 1, n).astype(np.int32)).cuda()
    g = torch.from_numpy(rng.integers(-4, 5, (n, 3)).astype(np.float32)).cuda()
    ok = (tok >= 0) & (tok < vocab)
    want = torch.zeros(vocab, 3, dtype=torch.float64, device="cuda").index_add_(0, tok[ok].long(), g[ok].double())
    for _ in range(3):
        assert torch.equal(tr.embed_backward(tok, g, vocab).double(), want)
