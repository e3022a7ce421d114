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
