"""Distillation with the other classes as one outcome where the student leaves
them next to nothing: their share of its probability underflows (beyond some 87
units of logits / T), the loss and the gradient, r times a softmax among them,
do not.  Bounds as in ``test_gpu_top_logits``."""
import pytest
import torch

import token_oracle as ref64
import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import DTYPES, LOGP_ABS, check_grad
from test_gpu_top_logits import teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k,T", [(5, 3, 1.0), (16, 12, 0.5), (300, 40, 1.0), (5000, 64, 2.0), (20001, 256, 1.0),
                                   (50257, 64, 1.0), (100001, 10, 1.0), (150001, 30, 1.5)])
def test_rest_far_below(device, V, k, T, dtype):
    g = seeded(1009 + V)
    rows = 8
    vals, idx, lse = teacher(rows, V, k, g, dtype, T)
    lse = lse + 0.2                                # leaves the others a fifth or more
    x = torch.randn(rows, V, generator=g)
    kept = torch.zeros(rows, V, dtype=torch.bool).scatter_(1, idx.long(), True)
    far = [0.0, -60.0 * T, -80.0 * T, -95.0 * T, -130.0 * T, -1e4, 0.0, 0.0]
    for r in range(rows):
        x[r] = torch.where(kept[r], x[r], x[r] + far[r])
    x[6] = torch.where(kept[6], x[6], torch.finfo(dtype).min)        # the others alike
    x[7] = torch.where(kept[7], x[7], float("-inf"))
    x[7, int((~kept[7]).nonzero()[0])] = -1e3 * T                    # one of them left
    x = x.to(dtype)
    weight = 64.0 * rows
    # What equal logits below all others are does not matter to the gradient, so the 64-bit statement takes
    # another value in row 6 (a + ln 2 is a again at 3.4e38, in 64 bits too).
    x64 = x.double()
    x64[6] = torch.where(kept[6], x64[6], -1e4)
    x64.requires_grad_()
    want = ref64.top_distil(x64, vals, idx, T, weight, None, lse)
    want.backward()
    xd = x.to(device).requires_grad_()
    args = (vals.to(device), idx.to(device), T, weight, None, lse.to(device))
    loss = ta.top_logits_distil_loss(xd, *args)
    loss.backward()
    if dtype == torch.float16:
        want = ref64.top_distil(x.double(), vals, idx, T, weight, None, lse)
        assert abs(loss.item() - want.item()) <= weight * T * T * 2 * LOGP_ABS + 2.0 ** -23 * abs(want.item())
    else:  # row 6: a tenth of 3.4e38, times 64 T, and more
        assert loss.item() == float("inf")
    check_grad(xd.grad, x64.grad, dtype, coef=weight * T / rows)
    assert (xd.grad.cpu() != 0)[~kept & (x64.grad.abs() > 1e-6)].all()
    with torch.no_grad():  # without a gradient: the same loss
        assert ta.top_logits_distil_loss(xd, *args).item() == loss.item()
