"""The minGRU recurrence (boa_b200.training) over long sequences, against 64 bits position by position."""
import numpy as np
import pytest

import training_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr(boa):
    from boa_b200 import training
    return training


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,T,d,lengths", [(1, 50001, 6, None), (2, 30011, 16, [30011, 12345]), (1, 20480, 64, None)])
def test_long_sequences(tr, dtype, B, T, d, lengths):
    import torch
    rng = np.random.default_rng(T)
    t = lambda x, k=dtype: torch.from_numpy(np.asarray(x, np.float32)).cuda().to(getattr(torch, k))  # noqa: E731
    n = lambda x: x.double().cpu().numpy()  # noqa: E731
    zh = t(np.concatenate([rng.normal(-3.0, 2.0, (B, T, d)), rng.normal(size=(B, T, d))], 2))
    dh, h0, dl = t(rng.normal(size=(B, T, d))), t(rng.normal(size=(B, d)), "float32"), t(rng.normal(size=(B, d)), "float32")
    left = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    h, last, saved = tr.mingru_scan(zh, h0, left, save_states=True)
    dzh, dh0 = tr.mingru_scan_backward(zh, saved, dh, dl, left)
    ref = R.mingru(n(zh), n(h0), lengths, n(dh), n(dl))
    for what, got, k in (("h", h, dtype), ("last", last, "float32"), ("dzh", dzh, dtype), ("dh0", dh0, "float32")):
        want, err = ref[what]
        off, tol = np.abs(n(got) - want), R.stored(want, err, k)
        assert (off <= tol).all(), f"{what}: {np.max(off / tol):.3g} times the bound"
