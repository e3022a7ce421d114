"""The training operators (boa_b200.training) at the largest sizes that they take."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


@pytest.mark.parametrize("others", [0, 1000000])
def test_embed_backward_of_the_most_positions(tr, others):
    """2^31 - 1 positions, all but a few of one token: the sum of ones is their
    number.  fp32 holds every sum of fewer than 2^24 ones exactly, and a
    piece has 2^23 of them; up to 256 sums of pieces are then added in any
    order, each time off by at most half a step."""
    import torch
    n = 2 ** 31 - 1
    tok = torch.full((n,), 7, dtype=torch.uint8, device="cuda")
    tok[:others] = 9
    out = tr.embed_backward(tok, torch.ones(n, 1, dtype=torch.float16, device="cuda"), 16)
    torch.cuda.synchronize()
    got = out[:, 0].double().cpu()
    assert abs(got[7].item() - (n - others)) <= 256 * 2.0 ** -24 * n
    assert got[9].item() == others and got.sum().item() == got[7].item() + others
