"""Distillation with the other classes as one outcome over a vocabulary of which
all but a few tokens are masked, for the teacher and the student alike: what the
teacher leaves to the others is then the rounding of its log-sum-exp, the student
leaves them nothing, and the loss is that over the tokens left.

Bounds, with e the teacher's log-sum-exp off by 4e-6 and half a step of fp32: its
probabilities are off by e of themselves, their sum by e, and a remainder of up to
4e-6 and a step is taken for none, so P by E = 2 (4e-6 + 2^-23 |lse|).  A term p
(ln p - ln q) moves by E p (1 + |ln p - ln q|) and p times a log probability's
error of 4e-6 each, a gradient q P - p by (E + 1e-5) (q + p) and its rounding."""
import pytest
import torch

import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import DTYPES, LOGP_ABS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fill", ["inf", "lowest", "10000"])
@pytest.mark.parametrize("V,k,left,T", [(300, 40, 1, 1.0), (1000, 64, 30, 1.0), (1000, 64, 64, 2.0), (30522, 64, 30, 2.0),
                                        (50257, 16, 16, 1.0), (100001, 64, 50, 1.0), (150001, 32, 20, 0.5)])
def test_all_but_a_few_tokens_masked(device, V, k, left, T, fill, dtype):
    g = seeded(V + left)
    rows = 32
    low = {"inf": float("-inf"), "lowest": torch.finfo(dtype).min, "10000": -1e4}[fill]
    at = torch.randperm(V, generator=g)[:left]
    t, s = torch.full((rows, V), low), torch.full((rows, V), low)
    t[:, at] = torch.randn(rows, left, generator=g) * 3 + torch.randn(rows, 1, generator=g) * 10
    s[:, at] = torch.randn(rows, left, generator=g) * 3
    t, s = t.to(dtype), s.to(dtype)
    p64, q64 = (x[:, at].double() / T for x in (t, s))
    lse = torch.logsumexp(p64, -1).abs()
    ratio = p64.log_softmax(-1) - q64.log_softmax(-1)
    p64, q64 = p64.softmax(-1), q64.softmax(-1)
    weight = 8.0 * rows
    want = weight * T * T * (p64 * ratio).sum(-1).mean()
    E = 2 * (LOGP_ABS + 2.0 ** -23 * lse)
    within = weight * T * T * ((E * (1 + (p64 * ratio.abs()).sum(-1))).mean() + 2 * LOGP_ABS) + 2.0 ** -23 * want.abs()

    x = s.to(device).requires_grad_()
    top = ta.top_logits(t.to(device), k, T)
    loss = ta.top_logits_distil_loss(x, top.values, top.indices, T, weight, t_logsumexp=top.logsumexp)
    loss.backward()
    assert abs(loss.item() - want.item()) <= within
    coef = weight * T / rows
    grad = x.grad.cpu().double()
    ideal = coef * (q64 - p64)
    fi = torch.finfo(dtype)
    tol = fi.eps / 2 * 1.001 * ideal.abs() + coef * (E[:, None] + 1e-5) * (q64 + p64) * (1 + fi.eps)
    tol = tol + 2.0 ** -22 * coef + (fi.smallest_normal * fi.eps if dtype == torch.float16 else fi.smallest_normal)
    assert ((grad[:, at] - ideal).abs() <= tol).all()
    masked = torch.ones(V, dtype=torch.bool)
    masked[at] = False
    assert (grad[:, masked] == 0).all()
    with torch.no_grad():
        assert ta.top_logits_distil_loss(x, top.values, top.indices, T, weight, t_logsumexp=top.logsumexp).item() == loss.item()


def test_remainder_the_student_cannot_reach(device):
    # a remainder that the teacher does leave stays one: infinite where the student has none of it
    x = torch.zeros(1, 50)
    x[0, 5:] = float("-inf")
    vals, idx = torch.zeros(1, 5), torch.arange(5, dtype=torch.int32)[None]
    for extra in (1e-4, 0.5):
        lse = torch.full((1,), 5.0).log() + extra
        loss = ta.top_logits_distil_loss(x.to(device), vals.to(device), idx.to(device), 1.0, t_logsumexp=lse.to(device))
        assert loss.item() == float("inf")
