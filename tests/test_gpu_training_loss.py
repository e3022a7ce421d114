"""The next-token loss (boa_b200.training): its gradient over the logits, and
the largest scales."""
import numpy as np
import pytest

import training_ref as R

pytestmark = pytest.mark.gpu

DT = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [1, 7, 32, 33, 255, 256, 257, 264, 1000, 1023, 1024])
def test_loss_in_place_equals_the_loss(tr, dtype, vocab):
    """Both results of a call that writes the gradient over its logits, for a
    target in every place of a row."""
    import torch
    rows = 4 * vocab + 37
    x = torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(vocab), device="cuda") * 3
    x = x.to(getattr(torch, dtype))
    t = torch.arange(rows, device="cuda") % vocab
    t[::11] = -1
    loss, grad = tr.token_loss(x, t, grad_scale=0.5)
    for _ in range(5):
        y = x.clone()
        loss2, grad2 = tr.token_loss(y, t, grad_scale=0.5, out=y)
        assert grad2 is y and torch.equal(y, grad) and torch.equal(loss2, loss)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [256, 37, 1024])
@pytest.mark.parametrize("inv", [1e30, 2.3e38, 2.4e38, 3.4e38, 1e-30, 1.5e-45])
def test_loss_at_the_ends_of_the_temperature(tr, dtype, vocab, inv):
    """The coldest distribution is the largest logit's symbol alone, the warmest is uniform."""
    import torch
    x = torch.randint(-8, 9, (6, vocab), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").float()
    x[:, 5] = 9.0
    x[2, 1::2] = -float("inf")
    x[2, 5] = 9.0
    t = torch.tensor([5, 5, 5, 0, 5, -1], device="cuda")
    scale = 1.0 / inv if inv > 1 else 1.0  # the gradient is in units of it
    loss, grad = tr.token_loss(x.to(getattr(torch, dtype)), t, inv_temperature=inv, grad_scale=scale)
    loss, grad = loss.double().cpu(), grad.double().cpu()
    if inv > 1:
        p = torch.zeros(6, vocab, dtype=torch.float64)
        p[:, 5] = 1.0
        # 9 - x[3, 0], times inv, where fp32 can hold it
        far = (9.0 - x[3, 0].item()) * inv
        assert abs(loss[3].item() - far) <= 4 * R.U * far if far < 3.402823e38 else loss[3] == float("inf")
        assert (loss[[0, 1, 2, 4, 5]] == 0).all()
        w = 1.0
    else:
        live = torch.isfinite(x).double().cpu()
        p = live / live.sum(1, keepdim=True)
        w = inv
        n = live.sum(1).log()
        assert (loss[:5] - n[:5]).abs().max() <= 4 * R.U * n.max() and loss[5] == 0
    hot = torch.zeros(6, vocab, dtype=torch.float64)
    hot[torch.arange(5), t[:5].cpu()] = 1.0
    want = w * (p - hot)
    want[5] = 0
    # exponential and sum 4 U each, the scale (below the normal range) 4 U, two products, a quotient, a difference
    tol = (16 * R.U + R.HALF_STEP[dtype]) * want.abs() + (2.0 ** -149 if dtype == "float32" else R.FLOOR[dtype])
    assert ((grad - want).abs() <= tol).all()
