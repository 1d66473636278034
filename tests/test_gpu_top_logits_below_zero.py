"""``top_logits`` of rows whose logits are mostly or all below zero, as language
models and log probabilities have them: the same values, places and sums as of
any row (exact; bounds of the log-sum-exp as in ``test_gpu_top_logits``), and in
one pass over the row like it.  The time is tested because nothing else tells
the pass from the slower walk that gives the same results: that walk reads a row
some fifty times, so a bound of three times the time of the same rows moved to
zero lies far from both."""
import pytest
import torch

import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import DTYPES
from test_gpu_top_logits import check_top

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(5, 3), (300, 40), (1000, 64), (1000, 128), (2063, 256), (4099, 64), (10001, 200),
                                 (30522, 64), (50257, 128), (140003, 31)])
def test_rows_below_zero(device, V, k, dtype):
    g = seeded(5 * V + k)
    x = torch.randn(10, V, generator=g) * 3
    x[0] = x[0] / 3 * 2.5 - 8
    x[1] -= 40
    x[2] -= 1000                                   # steps of 4 and 8 in bf16
    x[3] = x[3].log_softmax(-1)
    x[4] = x[4].clamp(max=0)                       # half of them zero
    x[5] = x[5].clamp(min=0)
    x[6] = -x[6].abs() - 1
    x[6, torch.randperm(V, generator=g)[:k - 1]] = 2.0       # one fewer above zero than asked for
    x[7] = -x[7].abs()
    x[7, torch.randperm(V, generator=g)[:k]] = 0.5
    x[8] = -x[8].abs() - 1
    x[8, torch.randperm(V, generator=g)[:k + 1]] = -0.0      # the border at zero, of either sign
    x[8, torch.randperm(V, generator=g)[:k // 2]] = 0.0
    x[9] = -x[9].abs() - 1
    x[9, -V // 8:] = x[9, -V // 8:].abs()          # what lies above zero stands at the end
    x = x.to(dtype)
    check_top(x, k, device)
    check_top(x[:, 1:].contiguous(), min(k, V - 1), device, 2.0, xd=x.to(device)[:, 1:])   # off a 16-byte boundary


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(1000, 64), (30522, 64), (70001, 100)])
def test_nan_and_infinities_below_zero(device, V, k, dtype):
    g = seeded(3 * V)
    x = torch.randn(4, V, generator=g) - 50
    x[1, [7, V - 2]] = float("nan")
    x[2, [3, V // 2]] = -float("nan")
    x[3, ::3] = float("-inf")
    x = x.to(dtype)
    top = ta.top_logits(x.to(device), k)
    check_top(x[::3].contiguous(), k, device)
    for r, places in ((1, [7, V - 2]), (2, [3, V // 2])):
        assert top.indices[r, :2].tolist() == places and top.logsumexp[r].isnan()
        rest = x[r].float().nan_to_num(float("-inf"))
        rest[places] = float("-inf")
        order = torch.argsort(rest, descending=True, stable=True)[:k - 2]
        assert torch.equal(top.indices[r, 2:].cpu().long(), order)


def _time(f):
    f()
    best = float("inf")
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("rows,V,k,dtype", [(4096, 30522, 64, torch.bfloat16), (1024, 131072, 128, torch.bfloat16),
                                            (8192, 1000, 64, torch.bfloat16), (2048, 30522, 64, torch.float32),
                                            (4096, 10000, 64, torch.float16), (8192, 4000, 256, torch.float16)])
def test_one_pass_below_zero(device, rows, V, k, dtype):
    x = torch.randn(rows, V, device=device, generator=torch.Generator(device=device).manual_seed(V)) * 3
    at_zero = x.to(dtype)
    want = _time(lambda: ta.top_logits(at_zero, k))
    for below in ((x - 40).to(dtype), (x / 3 * 2.5 - 8).to(dtype), x.log_softmax(-1).to(dtype)):
        assert _time(lambda: ta.top_logits(below, k)) < 3 * want
