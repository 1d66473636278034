"""Sums over long rows of coarse logits, where every addition of a thread rounds
the same way: a thread adds up to 300 such terms at 150 thousand classes and 2000
at a million, and a sum of n is off by up to n 2^-25 of itself.  Taken 64 at a time
and those sums in turn it is (64 + 64) 2^-25 at most up to 2^20 classes, which the
bounds of the token losses cover: a log probability within 4e-6."""
import pytest
import torch

import token_oracle as ref64
import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import DTYPES, check_logp
from test_gpu_top_logits import check_top, run_case, teacher

pytestmark = pytest.mark.gpu


def coarse(rows, V, dtype, g, about=0.0):
    """Each row of three neighbouring logits, a sixteenth apart (or the type's step), about a number of its own."""
    step = max(2.0 ** -4, abs(about) * torch.finfo(dtype).eps)
    base = about + torch.arange(rows)[:, None] * (7 * step / 16)
    return ((base / step).round() * step + step * torch.randint(0, 3, (rows, V), generator=g)).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("about", [0.0, -300.0])
@pytest.mark.parametrize("V,T", [(30522, 1.0), (152717, 0.5), (1000003, 1.0), (1000003, 0.7)])
def test_log_probabilities(device, V, T, about, dtype):
    g = seeded(V)
    x = coarse(8, V, dtype, g, about)[None]
    x[0, 7] = x[0, 7, 0]                        # all equal
    labels = torch.randint(0, V, (1, 8), generator=g)
    want, _ = ref64.log_probs(x.double(), labels, T)
    xd, labels = x.to(device), labels.to(device)
    check_logp(ta.token_log_probs(xd, labels, T), want)
    zero = torch.zeros(1, 8, device=device)
    _, got = ta.clipped_policy_loss(xd, labels, zero, torch.ones(1, device=device), temperature=T, return_log_probs=True)
    # (the policy loss keeps k's rounding, times the distance from the row's mean: less than a step here)
    check_logp(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,T", [(30522, 1.0), (152717, 0.5), (1000003, 1.0)])
def test_log_sum_exp(device, V, T, dtype):
    g = seeded(V + 1)
    x = coarse(8, V, dtype, g)
    check_top(x, 40, device, T)                 # thousands of equal logits at the border
    for r in range(8):                          # some above all others, in the first piece
        x[r, torch.randperm(20000, generator=g)[:64]] += torch.linspace(1, 2, 64).to(dtype)
    check_top(x, 40, device, T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,T,below", [(152717, 0.5, 0.0), (1000003, 1.0, 0.0), (1000003, 1.0, 200.0)])
def test_distillation(device, V, T, below, tail, dtype):
    g = seeded(V + 2)
    vals, idx, lse = teacher(1, V, 30, g, dtype, T)
    for n in range(4):
        x = coarse(4, V, dtype, g)[n:n + 1] - below
        if below:                               # the others' share by their own maximum
            x.scatter_(1, idx.long(), torch.randn(1, 30, generator=g).to(dtype))
        run_case(device, x, vals, idx, T, 64.0, None, lse if tail else None)
