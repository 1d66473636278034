"""The ``loss_fn`` plug-ins of the post-training losses with fp16 logits: the
loss scale in ``params.weight`` reaches the gradient before its rounding.
Bounds of the gradient as derived in ``test_gpu_token_losses``."""
from types import SimpleNamespace

import pytest
import torch

import token_oracle as ref64
import tspipe_amd as ta
from helpers import seeded
from test_gpu_token_losses import check_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight", [None, 1.0, 4096.0])
@pytest.mark.parametrize("which", ["preference", "policy"])
def test_weight_of_half_precision_gradients(device, which, weight):
    n, L, V = 4, 6, 3001
    g = seeded(901)
    s, t = ((torch.randn(n, L, V, generator=g) * 2).half() for _ in range(2))
    tokens = torch.randint(0, V, (n, L), generator=g)
    mask = torch.ones(n, L, dtype=torch.bool)
    nxt = torch.full_like(tokens, -100)
    nxt[:, :-1] = tokens[:, 1:]
    s64 = s.double().requires_grad_()
    ref = ref64.log_probs(t.double(), nxt)[0]
    params = SimpleNamespace(beta=0.1, kl_weight=0.05, clip_low=0.2, clip_high=0.2)
    if weight is not None:
        params.weight = weight
    sd = s.to(device).requires_grad_()
    outs = {"logits": sd}, {"logits": t.to(device)}
    if which == "preference":
        want, _ = ref64.preference(s64, nxt, ref, 0.1)
        loss = ta.preference_loss_fn(*outs, (tokens.to(device), mask.to(device)), None, params, 0)
    else:
        old, adv = ref64.log_probs(s.double(), nxt)[0].float() - 0.01, torch.randn(n, generator=g)
        want, _ = ref64.policy(s64, nxt, old.double(), adv.double(), ref, 0.05)
        loss = ta.policy_loss_fn(*outs, (tokens.to(device), mask.to(device), old.to(device), adv.to(device)), None,
                                 params, 0)
    want.backward()
    loss.backward()
    scale = weight or 1.0
    assert abs(loss.item() - scale * want.item()) <= scale * (4 * L * 4e-6 + 1e-6)
    check_grad(sd.grad, scale * s64.grad, torch.float16, coef=scale)
    if scale > 1:  # small elements survive: those above half of fp16's least step
        seen = (scale * s64.grad).abs() > 2.0 ** -24
        assert (s64.grad != 0)[:, :-1].all() and seen[:, :-1].double().mean() > 0.9
        assert (sd.grad.cpu()[seen] != 0).all()
