"""``top_logits``' log-sum-exp of rows far from zero.

The kernel works in powers of two, 2^(x k) with k = log2(e) / T rounded to fp32,
relative error up to 2^-24; times a mean of x / T of a thousand that alone would
be the rounding of the result once more.  With that taken out again, what is
left is the rounding of the fp32 result, half a step or 2^-24 of it, and the
bound of a log probability, 4e-6 (derived in ``test_gpu_token_losses``)."""
import pytest
import torch

import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import DTYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 4000, 30522, 70001])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.4, 2.8, 5.0, 5.3])   # k is off by 4.9e-8 of itself at 5, 1.3e-8 at 1
def test_far_from_zero(device, V, T, dtype):
    g = seeded(V)
    for mean in (-3000.0, -700.0, 60.0, 2500.0):
        x = (torch.randn(24, V, generator=g) * 2 * T + mean).to(dtype)
        want = torch.logsumexp(x.double() / T, -1)
        got = ta.top_logits(x.to(device), 5, T).logsumexp.cpu().double()
        assert ((got - want).abs() <= 4e-6 + 2.0 ** -24 * want.abs()).all(), (mean, (got - want).abs().max().item())
