"""Distillation with the other classes as one outcome over the widest rows it
takes, by one thread and by two at once on rows of different widths (whose marks
take different amounts of LDS): the bits one thread gives.  Bounds as in
``test_gpu_top_logits``."""
import threading

import pytest
import torch

import tspipe_amd as ta
from helpers import bits_equal, seeded
from test_gpu_top_logits import run_case, teacher

pytestmark = pytest.mark.gpu
MOST = 1 << 20


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widest_rows(device, dtype):
    g = seeded(77)
    vals, idx, lse = teacher(2, MOST, 64, g, dtype, 1.0)
    x = (torch.randn(2, MOST, generator=g) * 2).to(dtype)
    x.scatter_add_(1, idx.long(), (vals.float() * 0.6).to(dtype))
    run_case(device, x, vals, idx, 1.0, 8.0, None, lse)
    with pytest.raises((RuntimeError, ValueError)):
        wide = torch.zeros(1, MOST + 1, device=device)
        ta.top_logits_distil_loss(wide, *ta.top_logits(wide, 2)[:2], 1.0, t_logsumexp=torch.zeros(1, device=device))


def test_two_widths_at_once(device):
    g = seeded(79)
    inputs = []
    for V in (300001, MOST):
        t = (torch.randn(3, V, generator=g) * 2).bfloat16().to(device)
        s = (torch.randn(3, V, generator=g) * 2).bfloat16().to(device)
        inputs.append((s, ta.top_logits(t, 50)))

    def step(s, top):
        leaf = s.clone().requires_grad_()
        loss = ta.top_logits_distil_loss(leaf, top.values, top.indices, 1.0, t_logsumexp=top.logsumexp)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = step(*inputs[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for w, h in zip(want, got):
        for a, b in zip(w, h):
            assert bits_equal(a, b)
