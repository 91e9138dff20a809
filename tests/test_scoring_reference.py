"""The scoring operators' 64-bit reference (tests/scoring_reference.py) against torch's own conversions and plain sums."""
import numpy as np
import pytest
import torch

import scoring_reference as R

TYPE = {R.E4M3: torch.float8_e4m3fn, R.E5M2: torch.float8_e5m2}


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2])
def test_decode_every_code(fmt):
    want = torch.arange(256, dtype=torch.uint8).view(TYPE[fmt]).double().numpy()
    assert np.array_equal(R.VALUES[fmt], want, equal_nan=True)


@pytest.mark.parametrize("fmt", [R.E4M3, R.E5M2])
def test_codes_of_power_of_two_scales_are_torchs(fmt):
    """With the scale a power of two the quotient is exact in float32 and torch's conversion rounds it."""
    x = (np.random.default_rng(fmt).standard_normal((50, 300)) * 8).astype(np.float32).clip(-30, 30)
    x[:, ::128] = R.MAX[fmt] / 8
    val, scale = R.quantize(x, fmt, 1)
    assert (scale == 0.125).all()
    want = torch.from_numpy(x / 0.125).to(TYPE[fmt]).double().numpy()
    assert np.array_equal(val, want)
    val, scale = R.quantize(x, fmt, 128)
    assert scale.shape == (1, 3) and np.array_equal(val, want)


def test_product_and_logprobs():
    rng = np.random.default_rng(0)
    a, b = rng.standard_normal((5, 300)), rng.standard_normal((140, 300))
    sa, sb = rng.random((5, 3)).astype(np.float32), rng.random((2, 3)).astype(np.float32)
    da = a * np.repeat(sa.astype(np.float64), 128, 1)[:, :300]
    db = b * np.repeat(np.repeat(sb.astype(np.float64), 128, 0)[:140], 128, 1)[:, :300]
    y, err = R.matmul(a, sa, b, sb)
    assert np.allclose(y, da @ db.T, rtol=1e-12) and (err > 0).all()
    x = (rng.standard_normal((6, 50)) * 5).astype(np.float32)
    x[2, 7], x[5, 0] = -np.inf, np.nan
    ids = np.array([0, 49, 7, -1, 50, 3])
    got = R.logprobs(x, ids, 4)
    ls = torch.log_softmax(torch.from_numpy(x).double(), -1)
    lp = [ls[0, 0], ls[1, 49], -np.inf, 0.0, np.nan, np.nan]
    assert np.allclose(got["lp"], lp, rtol=1e-12, equal_nan=True)
    p = ls.exp()
    h = -torch.xlogy(p, p).sum(-1).numpy()
    assert np.allclose(got["h"][:5], h[:5], rtol=1e-12) and np.isnan(got["h"][5])
    assert np.array_equal(got["top_ids"][:5], torch.sort(torch.from_numpy(x[:5]), descending=True, stable=True)[1][:, :4].numpy())
    assert 0 not in got["top_ids"][5]
