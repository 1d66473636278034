"""Vocabulary rows in more than three dimensions with nothing in them: outputs
of the rows' shape, gradients of the logits', a loss over no rows NaN."""
import pytest
import torch

import tspipe_amd as ta

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 3, 0, 10), (2, 0, 3, 10), (0, 2, 3, 10), (0, 0, 0, 10), (2, 1, 2, 0, 10)])
def test_nothing_in_four_dimensions(device, shape):
    x = torch.zeros(shape, device=device, requires_grad=True)
    out = ta.token_log_probs(x, torch.zeros(shape[:-1], dtype=torch.int64, device=device))
    assert out.shape == shape[:-1]
    out.sum().backward()
    assert x.grad.shape == shape
    top = ta.top_logits(x, 3, 2.0)
    assert top.values.shape == top.indices.shape == shape[:-1] + (3,) and top.logsumexp.shape == shape[:-1]
    for lse in (None, top.logsumexp):
        x.grad = None
        loss = ta.top_logits_distil_loss(x, top.values, top.indices, 2.0, t_logsumexp=lse)
        loss.backward()
        assert loss.isnan() and x.grad.shape == shape
