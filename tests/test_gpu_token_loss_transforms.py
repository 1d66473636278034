"""Function transforms wrap tensors without memory of their own: every operator
on vocabulary rows refuses them before a launch, in the C++ nodes and in the
Python functions, and works on the same tensors afterwards."""
import pytest
import torch

import tspipe_amd as ta
from helpers import bits_equal, seeded
from test_gpu_token_losses import _both_ways

pytestmark = pytest.mark.gpu


def test_function_transforms_are_refused(device, monkeypatch):
    g = seeded(41)
    x = torch.randn(2, 3, 50, generator=g).to(device)
    lab = torch.randint(0, 50, (2, 3), generator=g).to(device)
    ref = torch.zeros(2, 3, device=device)
    top = ta.top_logits(x, 3)
    calls = [lambda y: ta.token_log_probs(y, lab).sum(), lambda y: ta.preference_loss(y, lab, ref),
             lambda y: ta.clipped_policy_loss(y, lab, ref, ref),
             lambda y: ta.top_logits_distil_loss(y, top.values, top.indices, 1.0), lambda y: ta.top_logits(y, 3).logsumexp.sum()]
    want = [f(x) for f in calls]
    batch = x.expand(4, 2, 3, 50).contiguous()
    labels, refs = torch.stack([lab, lab]), torch.stack([ref, ref])

    def refused():
        for f in calls:
            for transformed in (lambda: torch.func.grad(f)(x), lambda: torch.func.vmap(f)(batch),
                                lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.functionalize(f)(x)):
                with pytest.raises(RuntimeError):
                    transformed()
        for f, other in ((lambda t: ta.token_log_probs(x, t), labels), (lambda t: ta.preference_loss(x, lab, t), refs),
                         (lambda t: ta.clipped_policy_loss(x, lab, t, ref), refs),
                         (lambda t: ta.clipped_policy_loss(x, lab, ref, t), refs),
                         (lambda t: ta.token_log_probs(x, lab, row_mask=t), labels > 7)):
            with pytest.raises(RuntimeError):
                torch.func.vmap(f)(other)
        return all(bits_equal(f(x), w) for f, w in zip(calls, want))

    assert _both_ways(monkeypatch, refused) == (True, True)
