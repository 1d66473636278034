"""GPU parity of the token losses (log probabilities, preference, clipped
policy) against 64-bit statements on the CPU.

Tolerances.  A row's sum z of 2^((x - m) k) has terms off by the exponent's
two roundings, relative |x - m| k ln2 2^-23 (the shares of terms with
|x - m| / T above 16 vanish, so 16 * 2^-23 = 1.9e-6), and v_exp_f32's unit in
the last place; adding them up in fp32, a few hundred to a thread at most,
stays below 2e-6.  So a log probability is off by at most 4e-6 besides the
rounding of the fp32 result, a probability q by 1e-5 q, and a gradient
c (onehot - q) by 1e-5 |c| q, the half step of its storage type and the
rounding of 1 - q at 2^-24 |c|.
"""
import pytest
import torch

import token_oracle as ref64
import tspipe_amd as ta
from helpers import bits_equal, seeded

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LOGP_ABS = 4e-6


def check_logp(got, want, extra=0.0):
    got, want = got.detach().cpu().double(), want.detach().double()
    assert got.shape == want.shape
    err = (got - want).abs()
    assert (err <= LOGP_ABS + extra + 2.0 ** -24 * want.abs()).all(), err.max().item()


def check_grad(got, want, dtype, coef=None):
    """`coef`: largest |c| of the rows, [...] against gradients [..., V]."""
    assert got.dtype == dtype and got.shape == want.shape
    g, w = got.detach().cpu().double(), want.double()
    fi = torch.finfo(dtype)
    c = w.abs().amax(-1, keepdim=True) if coef is None else coef
    # half a step of fp16's subnormals is felt; those of the wider types may be flushed
    least = fi.smallest_normal * fi.eps if dtype == torch.float16 else fi.smallest_normal
    # (the coefficient itself comes from sums of log probabilities: 1e-5 relative covers it)
    tol = (fi.eps / 2 * 1.001 + 2e-5) * w.abs() + 2.0 ** -22 * c + least
    bad = (g - w).abs() > tol
    assert not bad.any(), ((g - w).abs() / tol).max().item()


def make(shape, dtype, seed, std=2.5):
    g = seeded(seed)
    x = (torch.randn(*shape, generator=g) * std).to(dtype)
    labels = torch.randint(0, shape[-1], shape[:-1], generator=g)
    lift = torch.rand(*shape[:-1], 1, generator=g) * 8
    x.scatter_(-1, labels[..., None], lift.to(dtype))
    return x, labels, g


SIZES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (2, 5, 100), (3, 4, 255), (2, 2, 1000), (2, 3, 2049), (2, 7, 4099), (2, 2, 8193),
         (2, 3, 30522), (2, 2, 32001), (2, 2, 50257), (2, 1, 65537), (2, 1, 131072), (2, 1, 140003)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,L,V", SIZES)
def test_log_probs(device, n, L, V, dtype):
    x, labels, g = make((n, L, V), dtype, 10 + V)
    if n * L > 2:
        labels[0, 0] = -100
        labels[-1, -1] = V  # outside: does not count either
    T = 0.9 if V % 2 else 1.0
    x64 = x.double().requires_grad_()
    want, live = ref64.log_probs(x64, labels, T)
    go = torch.randn(n, L, generator=g)
    want.backward(go.double())
    xd = x.to(device).requires_grad_()
    got = ta.token_log_probs(xd, labels.to(device), T)
    assert got.dtype == torch.float32
    check_logp(got, want)
    got.backward(go.to(device))
    check_grad(xd.grad, x64.grad, dtype, coef=(go.abs() / T)[..., None])
    assert (xd.grad.cpu()[~live] == 0).all()
    with torch.no_grad():
        again = ta.token_log_probs(xd, labels.to(device), T)
    assert not again.requires_grad and bits_equal(again, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,cut", [(37, 1), (1000, 1), (4099, 2), (30522, 1)])
def test_log_probs_of_slices_and_shifted_bases(device, V, cut, dtype):
    # the logits without each sequence's last positions, a transposed batch, and rows off a 16-byte
    # boundary are read where they lie; where the rows start at the same distances from such a boundary
    # as a dense copy's (V a multiple of 8), the sums run in the same order and give the same bits
    x, labels, g = make((3, 6, V), dtype, 77 + V)
    go = torch.randn(3, 6 - cut, generator=g)
    lab = labels[:, cut:].contiguous()
    x64 = x[:, :-cut].double().requires_grad_()
    want, _ = ref64.log_probs(x64, lab)
    want.backward(go.double())
    xd, labd, god = x.to(device), lab.to(device), go.to(device)
    dense = xd[:, :-cut].contiguous().requires_grad_()
    plain = ta.token_log_probs(dense, labd)
    plain.backward(god)
    pad = torch.zeros(3 * 6 * V + 3, dtype=dtype, device=device)
    pad[3:] = xd.reshape(-1)
    views = {
        "slice": xd.clone(),
        "token major": xd.permute(1, 0, 2).contiguous().permute(1, 0, 2),
        "shifted": pad[3:].view(3, 6, V),
        "last dimension not dense": xd.transpose(1, 2).contiguous().transpose(1, 2),
    }
    for name, v in views.items():
        leaf = v.detach().requires_grad_()
        out = ta.token_log_probs(leaf[:, :-cut], labd)
        out.backward(god)
        check_logp(out, want)
        check_grad(leaf.grad[:, :-cut], x64.grad, dtype, coef=go.abs()[..., None])
        assert (leaf.grad[:, -cut:] == 0).all()
        if V % 8 == 0 and name != "shifted":
            assert bits_equal(out, plain) and bits_equal(leaf.grad[:, :-cut], dense.grad), name


def test_log_probs_row_mask_and_label_types(device):
    x, labels, g = make((4, 5, 501), torch.float32, 3)
    mask = torch.rand(4, 5, generator=g) < 0.5
    want, _ = ref64.log_probs(x.double(), labels.masked_fill(~mask, -100))
    for m in (mask, mask.to(torch.int32) * 3, mask.float()):
        for lab in (labels, labels.to(torch.int32)):
            check_logp(ta.token_log_probs(x.to(device), lab.to(device), row_mask=m.to(device)), want)
    odd = labels.clone()
    odd[0] = 7
    check_logp(ta.token_log_probs(x.to(device), odd.to(device), ignore_index=7),
               ref64.log_probs(x.double(), odd.masked_fill(odd == 7, -100))[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_extreme_logits(device, dtype):
    V = 3001
    x, labels, g = make((1, 8, V), dtype, 5)
    fi = torch.finfo(dtype)
    labels[:] = 0
    x[0, 0, 5:] = float("-inf")              # a masked vocabulary
    x[0, 1, 5:] = fi.min                     # masked by the type's lowest value
    x[0, 2, :] = fi.min                      # all of it: equal logits
    x[0, 3, :] = 0                           # equal logits
    x[0, 4, 1:] = float("-inf")              # one class left
    x[0, 5, 7] = 80.0                        # far from the label
    x[0, 6, 0], x[0, 6, 1] = 60.0, 59.5      # large, close
    x[0, 7, 9] = float("-inf")
    x64 = x.double().requires_grad_()
    want, _ = ref64.log_probs(x64, labels)
    go = torch.randn(1, 8, generator=g)
    want.backward(go.double())
    xd = x.to(device).requires_grad_()
    got = ta.token_log_probs(xd, labels.to(device))
    check_logp(got, want)
    got.backward(go.to(device))
    check_grad(xd.grad, x64.grad, dtype, coef=go.abs()[..., None])


def test_log_probs_nan_and_infinities(device):
    x, labels, _ = make((1, 6, 700), torch.float32, 6)
    x[0, 0, 13] = float("nan")
    x[0, 1, 13] = float("inf")
    x[0, 2, :] = float("-inf")
    x[0, 3, labels[0, 3]] = float("-inf")
    x[0, 4, :] = float("nan")
    labels[0, 4] = -100  # not read
    got = ta.token_log_probs(x.to(device), labels.to(device)).cpu()[0]
    assert torch.isnan(got[:3]).all() and got[3] == float("-inf") and got[4] == 0 and torch.isfinite(got[5])
    xd = x.to(device).requires_grad_()
    ta.token_log_probs(xd, labels.to(device)).sum().backward()
    assert (xd.grad[0, 4] == 0).all() and torch.isfinite(xd.grad[0, 5]).all()


def test_log_probs_empty(device):
    for shape in [(0, 4, 10), (3, 0, 10), (0, 10)]:
        x = torch.zeros(shape, device=device, requires_grad=True)
        out = ta.token_log_probs(x, torch.zeros(shape[:-1], dtype=torch.int64, device=device))
        assert out.shape == shape[:-1]
        out.sum().backward()
        assert x.grad.shape == shape
    x = torch.randn(10, device=device)
    out = ta.token_log_probs(x, torch.tensor(3, device=device))
    check_logp(out, x.cpu().double().log_softmax(-1)[3])


def test_log_probs_against_differences(device):
    x, labels, g = make((2, 4, 777), torch.float32, 8, std=1.0)
    d = torch.randn(x.shape, generator=g).to(device)
    go = torch.randn(2, 4, generator=g).to(device)
    xd = x.to(device).requires_grad_()
    lab = labels.to(device)
    ta.token_log_probs(xd, lab).backward(go)
    h = 1e-2
    up, down = (ta.token_log_probs((xd + s * h * d).detach(), lab) for s in (1, -1))
    numeric = ((up.double() - down.double()) * go).sum() / (2 * h)
    # eight log probabilities off by 4e-6 each over 2 h, and h^2 / 6 times third cumulants of order one
    tol = 8 * LOGP_ABS / h * go.abs().max().item() + 8 * h * h
    assert abs(numeric.item() - (xd.grad.double() * d).sum().item()) < tol


# ---- preference ------------------------------------------------------------------------

def ragged(labels, g, empty=()):
    L = labels.shape[1]
    for i in range(labels.shape[0]):
        a, b = sorted(torch.randint(0, L + 1, (2,), generator=g).tolist())
        labels[i, :a] = -100
        labels[i, max(b, a + 1):] = -100
        if i in empty:
            labels[i] = -100
    return labels


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.0, False), ("sigmoid", 0.2, True), ("hinge", 0.0, False),
                                                    ("ipo", 0.0, True), ("ipo", 0.0, False)])
@pytest.mark.parametrize("pairs,L,V", [(1, 1, 5), (1, 9, 4099), (3, 17, 1000), (5, 6, 30522), (2, 300, 131)])
def test_preference(device, pairs, L, V, kind, smoothing, average, dtype):
    x, labels, g = make((2 * pairs, L, V), dtype, 1000 + V + L)
    if L > 1:
        labels = ragged(labels, g, empty=(1,) if pairs > 1 else ())
    ref = ref64.log_probs(x.double(), labels)[0].float() + torch.randn(2 * pairs, L, generator=g) * 0.2
    beta, weight = 0.3, 64.0
    x64 = x.double().requires_grad_()
    want, rewards = ref64.preference(x64, labels, ref.double(), beta, kind, smoothing, average, weight)
    want.backward()
    xd = x.to(device).requires_grad_()
    loss, got_r = ta.preference_loss(xd, labels.to(device), ref.to(device), beta, kind, smoothing, average, weight,
                                     return_rewards=True)
    loss.backward()
    # an answer's sum is off by 4e-6 a token; its reward by beta times that, the loss by weight * |f'| times two
    n_tok = 1 if average else L
    slope = {"sigmoid": beta, "hinge": beta, "ipo": 2 * (rewards.abs().max().item() * 2 / beta + 1 / (2 * beta))}[kind]
    assert ((got_r.cpu().double() - rewards).abs() <= beta * n_tok * LOGP_ABS + 2.0 ** -24 * rewards.abs()).all()
    assert abs(loss.item() - want.item()) <= weight * slope * 2 * n_tok * LOGP_ABS + 2.0 ** -23 * abs(want.item())
    assert not got_r.requires_grad and loss.dtype == torch.float32
    # the factor c inherits the sums' error through f''
    curve = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kind] * weight / pairs * 2 * n_tok * LOGP_ABS
    check_grad(xd.grad, x64.grad, dtype, coef=x64.grad.abs().amax(-1, keepdim=True) + curve * 2 ** 22)
    # loss alone, and a reference summed per answer
    with torch.no_grad():
        assert bits_equal(ta.preference_loss(xd, labels.to(device), ref.to(device), beta, kind, smoothing, average, weight),
                          loss.detach())
    live = labels >= 0
    per = torch.where(live, ref, torch.zeros_like(ref)).double().sum(-1)
    if average:
        per = per / live.sum(-1).clamp_min(1)
    per = per.float()
    want2, r2 = ref64.preference(x.double(), labels, per.double(), beta, kind, smoothing, average, weight)
    loss2, got2 = ta.preference_loss(xd, labels.to(device), per.to(device), beta, kind, smoothing, average, weight,
                                     return_rewards=True)
    assert ((got2.cpu().double() - r2).abs() <= beta * n_tok * LOGP_ABS + 2.0 ** -24 * r2.abs()).all()
    slope2 = slope if kind != "ipo" else 2 * (r2.abs().max().item() * 2 / beta + 1 / (2 * beta))
    assert abs(loss2.item() - want2.item()) <= weight * slope2 * 2 * n_tok * LOGP_ABS + 2.0 ** -23 * abs(want2.item())


def test_preference_empty_and_extreme(device):
    x = torch.zeros(0, 4, 10, device=device, requires_grad=True)
    loss = ta.preference_loss(x, torch.zeros(0, 4, dtype=torch.int64, device=device), torch.zeros(0, 4, device=device))
    assert torch.isnan(loss)
    loss.backward()
    x = torch.zeros(2, 0, 10, device=device, requires_grad=True)
    loss = ta.preference_loss(x, torch.zeros(2, 0, dtype=torch.int64, device=device), torch.zeros(2, device=device))
    assert abs(loss.item() - 0.6931471805599453) < 1e-6
    loss.backward()
    # far apart: neither side overflows
    x, labels, g = make((2, 40, 300), torch.float32, 12)
    for sign in (1.0, -1.0):
        shift = torch.tensor([5000.0, -5000.0]) * sign
        want, _ = ref64.preference(x.double(), labels, shift.double(), 1.0)
        xd = x.to(device).requires_grad_()
        loss = ta.preference_loss(xd, labels.to(device), shift.to(device), 1.0)
        loss.backward()
        assert abs(loss.item() - want.item()) <= 1e-6 * abs(want.item()) + 1e-6
        assert torch.isfinite(xd.grad).all()
    # NaN logits in a row that does not count, and in one that does
    x[0, 3] = float("nan")
    labels[0, 3] = -100
    xd = x.to(device).requires_grad_()
    loss = ta.preference_loss(xd, labels.to(device), torch.zeros(2, device=device))
    loss.backward()
    assert torch.isfinite(loss) and torch.isfinite(xd.grad).all() and (xd.grad[0, 3] == 0).all()
    labels[0, 3] = 5
    assert torch.isnan(ta.preference_loss(xd, labels.to(device), torch.zeros(2, device=device)))


# ---- clipped policy loss -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("per_answer", [True, False])
@pytest.mark.parametrize("n,L,V,kl,T", [(1, 1, 3, 0.0, 1.0), (3, 7, 1000, 0.1, 0.7), (4, 9, 4099, 0.0, 1.0),
                                        (3, 5, 30522, 0.05, 1.0), (2, 3, 70001, 0.1, 1.5), (5, 200, 127, 0.3, 1.0)])
def test_policy(device, n, L, V, kl, T, per_answer, reduction, dtype):
    x, labels, g = make((n, L, V), dtype, 2000 + V + L)
    if L > 1:
        labels = ragged(labels, g, empty=(1,))
    base = ref64.log_probs(x.double(), labels, T)[0].float()
    drift = torch.randn(n, L, generator=g) * 0.25
    # ratios within 1e-4 of an end of the clipping range are moved: there the last bits decide
    ends = torch.minimum((torch.exp(-drift) - 0.9).abs(), (torch.exp(-drift) - 1.3).abs()) < 1e-4
    old = base + drift.masked_fill(ends, 0.0)
    rlp = base + torch.randn(n, L, generator=g) * 0.3
    adv = torch.randn(n, generator=g) if per_answer else torch.randn(n, L, generator=g)
    weight = 32.0 * n * L
    x64 = x.double().requires_grad_()
    want, lp = ref64.policy(x64, labels, old.double(), adv.double(), rlp.double(), kl, 0.1, 0.3, T, reduction, weight)
    want.backward()
    xd = x.to(device).requires_grad_()
    loss, got_lp = ta.clipped_policy_loss(xd, labels.to(device), old.to(device), adv.to(device),
                                          rlp.to(device) if kl else None, kl, 0.1, 0.3, T, reduction, weight,
                                          return_log_probs=True)
    loss.backward()
    check_logp(got_lp, lp)
    # a term moves by |A| r + kl e^d times its log probability's error
    steep = adv.abs().max().item() * 2 + 2 * kl
    assert abs(loss.item() - want.item()) <= weight * steep * LOGP_ABS + 2.0 ** -23 * abs(want.item())
    per_row = weight / (1 if reduction == "sequence" else max(1, int((labels >= 0).sum())))
    check_grad(xd.grad, x64.grad, dtype,
               coef=x64.grad.abs().amax(-1, keepdim=True) + per_row / T * (kl + steep) * LOGP_ABS * 2 ** 22)
    with torch.no_grad():
        assert bits_equal(ta.clipped_policy_loss(xd, labels.to(device), old.to(device), adv.to(device),
                                                 rlp.to(device) if kl else None, kl, 0.1, 0.3, T, reduction, weight),
                          loss.detach())


def test_policy_empty_and_nothing_counts(device):
    for n, L in [(0, 3), (2, 0), (2, 3)]:
        for reduction in ("token", "sequence"):
            x = torch.randn(n, L, 50, device=device).requires_grad_()
            labels = torch.full((n, L), -100, device=device)
            z = torch.zeros(n, L, device=device)
            loss = ta.clipped_policy_loss(x, labels, z, z, reduction=reduction)
            assert torch.isnan(loss)
            loss.backward()
            assert (x.grad == 0).all()


def test_policy_gradient_stops_at_the_clip(device):
    x, labels, g = make((1, 4, 64), torch.float32, 31)
    lp = ref64.log_probs(x.double(), labels)[0].float()
    old = lp - torch.tensor([[0.5, 0.5, -0.5, -0.5]])     # ratios e^.5, e^.5, e^-.5, e^-.5
    adv = torch.tensor([[1.0, -1.0, 1.0, -1.0]])
    xd = x.to(device).requires_grad_()
    ta.clipped_policy_loss(xd, labels.to(device), old.to(device), adv.to(device)).backward()
    moved = xd.grad.abs().amax(-1).cpu()[0] > 0
    assert moved.tolist() == [False, True, True, False]


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_losses_against_differences(device, which):
    x, labels, g = make((2, 5, 400), torch.float32, 41, std=1.0)
    base = ref64.log_probs(x.double(), labels)[0].float()
    rlp = (base + 0.3 * torch.randn(2, 5, generator=g)).to(device)
    old = (base + 0.05 * torch.randn(2, 5, generator=g)).to(device)
    adv = torch.randn(2, 5, generator=g).to(device)
    lab = labels.to(device)

    def f(t):
        if which == "preference":
            return ta.preference_loss(t, lab, rlp, 0.5)
        return ta.clipped_policy_loss(t, lab, old, adv, rlp, 0.2, clip_low=10.0, clip_high=10.0)

    d = torch.randn(x.shape, generator=g).to(device) * 0.3
    xd = x.to(device).requires_grad_()
    f(xd).backward()
    h = 1e-2
    with torch.no_grad():
        numeric = (f(xd + h * d).double() - f(xd - h * d).double()).item() / (2 * h)
    # losses of order one off by 1e-5 over 2 h, and h^2 / 6 times a third derivative of order ten along d
    assert abs(numeric - (xd.grad.double() * d).sum().item()) < 1e-5 / h + 20 * h * h


def test_scaled_backward_runs_once(device):
    x, labels, g = make((2, 4, 600), torch.float32, 51)
    ref = torch.zeros(2, 4, device=device)
    a, b = (x.to(device).requires_grad_() for _ in range(2))
    la = ta.preference_loss(a, labels.to(device), ref)
    la.backward()
    lb = ta.preference_loss(b, labels.to(device), ref)
    (lb * 3.0).backward()
    assert torch.allclose(b.grad, 3.0 * a.grad, rtol=1e-6, atol=0)
    with pytest.raises(RuntimeError):
        la.backward()
    # log probabilities keep their inputs and may go backward again
    c = x.to(device).requires_grad_()
    out = ta.token_log_probs(c, labels.to(device)).sum()
    g1, = torch.autograd.grad(out, c, retain_graph=True)
    g2, = torch.autograd.grad(out, c)
    assert bits_equal(g1, g2)


def test_other_stream_and_repeatability(device):
    x, labels, g = make((4, 50, 2000), torch.bfloat16, 61)
    lab, ref, adv = labels.to(device), torch.randn(4, 50, generator=g).to(device) - 8, torch.randn(4, generator=g).to(device)

    def step(xd):
        l1, r = ta.preference_loss(xd, lab, ref, return_rewards=True)
        l2, lp = ta.clipped_policy_loss(xd, lab, ref, adv, ref, 0.1, return_log_probs=True)
        return [l1.detach(), r, l2.detach(), lp, *torch.autograd.grad(l1 + l2, xd)]

    xd = x.to(device).requires_grad_()
    want = [t.clone() for t in step(xd)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xd)
    side.synchronize()
    for a, b in zip(want, got):
        assert bits_equal(a, b)


def test_graph_capture_replays(device):
    x, labels, g = make((2, 20, 3000), torch.bfloat16, 71)
    lab, ref, adv = labels.to(device), torch.randn(2, 20, generator=g).to(device) - 8, torch.randn(2, generator=g).to(device)
    static = x.to(device).requires_grad_()

    def step(xd):
        lp = ta.token_log_probs(xd, lab)
        l1 = ta.preference_loss(xd, lab, ref)
        l2 = ta.clipped_policy_loss(xd, lab, ref, adv, ref, 0.1)
        return [lp.detach(), l1.detach(), l2.detach(), torch.autograd.grad(lp, xd, torch.ones_like(lp))[0],
                torch.autograd.grad(l1, xd)[0], torch.autograd.grad(l2, xd)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for trial in range(4):
        fresh = (x.float() * (1 + 0.1 * trial)).to(torch.bfloat16).to(device)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = step(fresh.requires_grad_())
        for a, b in zip(outs, want):
            assert bits_equal(a, b), trial


# ---- used together ----------------------------------------------------------------------------

class _Params:
    beta, kl_weight, clip_low, clip_high = 0.2, 0.1, 0.2, 0.25


def test_plug_ins(device):
    g = seeded(81)
    n, L, V = 4, 12, 900
    s, t = (torch.randn(n, L, V, generator=g) * 2 for _ in range(2))
    tokens = torch.randint(0, V, (n, L), generator=g)
    mask = torch.rand(n, L, generator=g) < 0.6
    nxt = torch.full_like(tokens, -100)
    nxt[:, :-1] = tokens[:, 1:].masked_fill(~mask[:, 1:], -100)
    ref = ref64.log_probs(t.double(), nxt)[0]
    s64 = s.double().requires_grad_()
    want, _ = ref64.preference(s64, nxt, ref, _Params.beta)
    want.backward()
    sd = s.to(device).requires_grad_()
    loss = ta.preference_loss_fn({"logits": sd}, {"logits": t.to(device)}, (tokens.to(device), mask.to(device)), None,
                                 _Params(), 0)
    loss.backward()
    assert abs(loss.item() - want.item()) < 4 * L * LOGP_ABS + 1e-6
    check_grad(sd.grad, s64.grad, torch.float32, coef=1.0)
    old = ref64.log_probs(s.double(), nxt)[0].float() + 0.01
    adv = torch.randn(n, generator=g)
    s64 = s.double().requires_grad_()
    want, _ = ref64.policy(s64, nxt, old.double(), adv.double(), ref, 0.1, 0.2, 0.25)
    want.backward()
    sd = s.to(device).requires_grad_()
    loss = ta.policy_loss_fn({"logits": sd}, {"logits": t.to(device)},
                             (tokens.to(device), mask.to(device), old.to(device), adv.to(device)), None, _Params(), 0)
    loss.backward()
    # ref - log p reaches several units here, and its exponential multiplies the error
    big = (ref - ref64.log_probs(s.double(), nxt)[0]).abs().max().exp().item()
    assert abs(loss.item() - want.item()) < (3 + big) * LOGP_ABS * 2 + 1e-6 * abs(want.item())
    check_grad(sd.grad, s64.grad, torch.float32, coef=1.0 + 0.1 * big * 2 * LOGP_ABS * 2 ** 22)


def test_training_steps_with_the_plug_in(device):
    # a few optimizer steps of a linear head under the preference plug-in follow the same steps in 64 bits
    g = seeded(91)
    n, L, D, V = 4, 8, 16, 300
    h = torch.randn(n, L, D, generator=g)
    w0 = torch.randn(V, D, generator=g) * 0.3
    tokens = torch.randint(0, V, (n, L), generator=g)
    mask = torch.ones(n, L, dtype=torch.bool)
    nxt = torch.full_like(tokens, -100)
    nxt[:, :-1] = tokens[:, 1:]
    t = h @ w0.t()
    ref = ref64.log_probs(t.double(), nxt)[0]
    w64, wd = w0.double(), w0.to(device)
    for _ in range(3):
        w64 = w64.detach().requires_grad_()
        l64, _ = ref64.preference(h.double() @ w64.t(), nxt, ref, 0.2)
        l64.backward()
        wd = wd.detach().requires_grad_()
        loss = ta.preference_loss_fn({"logits": h.to(device) @ wd.t()}, {"logits": t.to(device)},
                                     (tokens.to(device), mask.to(device)), None, _Params(), 0)
        loss.backward()
        assert abs(loss.item() - l64.item()) < 1e-4
        assert (wd.grad.cpu().double() - w64.grad).abs().max() < 1e-4 * w64.grad.abs().max() + 1e-5
        w64, wd = w64.detach() - 0.5 * w64.grad, wd.detach() - 0.5 * wd.grad


# ---- the C++ node and the Python functions ----------------------------------------------------

def _both_ways(monkeypatch, f):
    from tspipe_amd import _vocab
    assert _vocab.host_for(torch.zeros(1, device="cuda")) is not None
    monkeypatch.setattr(_vocab, "_HOST_NODE", True)
    a = f()
    monkeypatch.setattr(_vocab, "_HOST_NODE", False)
    return a, f()


def test_host_node_and_python_functions_agree(device, monkeypatch):
    x, labels, g = make((4, 13, 1501), torch.bfloat16, 111)
    xd, lab = x.to(device), labels.to(device)
    mask = (torch.rand(4, 13, generator=g) < 0.7).to(device)
    ref = (torch.randn(4, 13, generator=g) - 8).to(device)
    adv = torch.randn(4, generator=g).to(device)
    top = ta.top_logits(xd, 20, 2.0)

    def everything():
        leaf = xd.clone().requires_grad_()
        outs = []
        for view in (leaf, leaf[:, :, :]):
            lp = ta.token_log_probs(view, lab, 0.9, row_mask=mask)
            l1, r = ta.preference_loss(view, lab, ref, 0.2, label_smoothing=0.1, row_mask=mask, return_rewards=True)
            l2, lp2 = ta.clipped_policy_loss(view, lab, ref, adv, ref, 0.1, reduction="sequence", row_mask=mask,
                                             return_log_probs=True)
            l3 = ta.top_logits_distil_loss(view, top.values, top.indices, 2.0, row_mask=mask, t_logsumexp=top.logsumexp)
            outs += [lp, l1, r, l2, lp2, l3, *ta.top_logits(view, 7)]
            for loss in (lp.sum(), l1, l2 * 2.0, l3):
                outs += torch.autograd.grad(loss, leaf)
        return [o.detach() for o in outs]

    a, b = _both_ways(monkeypatch, everything)
    assert len(a) == len(b)
    for i, (p, q) in enumerate(zip(a, b)):
        assert bits_equal(p, q), i


def test_both_refuse_alike(device, monkeypatch):
    x, labels, _ = make((2, 5, 300), torch.float32, 121)
    lab, ref = labels.to(device), torch.zeros(2, 5, device=device)

    def twice():
        leaf = x.to(device).requires_grad_()
        loss = ta.preference_loss(leaf, lab, ref)
        loss.backward()
        with pytest.raises(RuntimeError):
            loss.backward()
        # log probabilities read their logits again: a change in between is noticed
        mid = leaf * 1.0
        lp = ta.token_log_probs(mid, lab).sum()
        mid.add_(1.0)
        with pytest.raises(RuntimeError):
            lp.backward()
        # a second derivative is refused
        for make_loss in (lambda: ta.token_log_probs(leaf, lab).sum(), lambda: ta.preference_loss(leaf, lab, ref),
                          lambda: ta.clipped_policy_loss(leaf, lab, ref, ref),
                          lambda: ta.top_logits_distil_loss(leaf, *ta.top_logits(leaf, 3)[:2], 1.0)):
            with pytest.raises(RuntimeError):
                g, = torch.autograd.grad(make_loss(), leaf, create_graph=True)
                g.sum().backward()
        for call in (lambda: ta.preference_loss(leaf, lab[:, :4], ref), lambda: ta.preference_loss(leaf, lab, ref[:, :4]),
                     lambda: ta.clipped_policy_loss(leaf, lab, ref, ref[:1, 0]),
                     lambda: ta.token_log_probs(leaf, lab.cpu()),
                     lambda: ta.top_logits(leaf, 301), lambda: ta.top_logits(leaf, 0),
                     lambda: ta.top_logits_distil_loss(leaf, ref, lab.to(torch.int32), 1.0)):
            with pytest.raises(ValueError):
                call()
        for call in (lambda: ta.token_log_probs(leaf, lab.float()), lambda: ta.token_log_probs(leaf.double(), lab),
                     lambda: ta.preference_loss(leaf, lab, lab), lambda: ta.top_logits(leaf.long(), 2)):
            with pytest.raises(TypeError):
                call()
        return True

    assert _both_ways(monkeypatch, twice) == (True, True)
    # without gradients there is nothing to record
    with torch.no_grad():
        leaf = x.to(device).requires_grad_()
        assert not ta.preference_loss(leaf, lab, ref).requires_grad
    assert not ta.preference_loss(x.to(device), lab, ref).requires_grad


def test_two_threads_on_two_streams(device):
    import threading
    x, labels, g = make((4, 40, 3000), torch.bfloat16, 131)
    lab, ref = labels.to(device), (torch.randn(4, 40, generator=g) - 8).to(device)
    adv = torch.randn(4, generator=g).to(device)
    inputs = [(x.float() * s).to(torch.bfloat16).to(device) for s in (1.0, 0.7)]

    def step(xd):
        leaf = xd.clone().requires_grad_()
        l1 = ta.preference_loss(leaf, lab, ref)
        g1, = torch.autograd.grad(l1, leaf)
        l2 = ta.clipped_policy_loss(leaf, lab, ref, adv, ref, 0.1)
        g2, = torch.autograd.grad(l2, leaf)
        top = ta.top_logits(leaf, 11)
        l3 = ta.top_logits_distil_loss(leaf, top.values, top.indices, 2.0)
        g3, = torch.autograd.grad(l3, leaf)
        return [l1.detach(), g1, l2.detach(), g2, *top, l3.detach(), g3]

    want = [step(t) for t in inputs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = step(inputs[i])
            s.synchronize()
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


@pytest.mark.parametrize("V", [700, 9000, 40000, 90000, 150001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_stretches_and_lone_peaks(device, V, dtype):
    # stretches of vocabulary masked with -1e4, -1e9, -inf or the type's lowest value, wherever they fall among
    # the wavefronts' vectors; whole rows far from zero; one logit far above all others, at temperatures down to 0.2
    g = seeded(140 + V)
    fi = torch.finfo(dtype)
    fills = [-1e4, -6e4 if dtype == torch.float16 else -1e9, float("-inf"), fi.min]
    rows = []
    for fill in fills:
        for lo, hi in ((0, V // 2), (V // 2, V - 3), (5, V - 5)):
            r = torch.randn(V, generator=g) * 2
            r[lo:hi] = fill
            rows.append(r)
    for shift in (-3e4, 3e4):
        rows.append(torch.randn(V, generator=g) * 50 + shift)
    for at in (0, V // 3, V - 1):
        r = torch.randn(V, generator=g)
        r[at] = 60.0
        rows.append(r)
    x = torch.stack(rows).to(dtype)[None]
    n = x.shape[1]
    labels = torch.tensor([[int(x[0, i].float().argmax()) if i % 2 else V - 1 for i in range(n)]])
    go = torch.randn(1, n, generator=g)
    for T in (1.0, 0.2):
        x64 = x.double().requires_grad_()
        want, _ = ref64.log_probs(x64, labels, T)
        want.backward(go.double())
        xd = x.to(device).requires_grad_()
        got = ta.token_log_probs(xd, labels.to(device), T)
        got.backward(go.to(device))
        finite = torch.isfinite(want) & (want.abs() < 1e30)
        # exponents of rows far from zero carry the fp32 rounding of x k, at most 2^-24 |x| / T each way
        extra = 2.0 ** -23 * (x.double().abs().amin(-1) / T)
        err = (got.cpu().double() - want).abs()
        assert (err <= LOGP_ABS + extra + 2.0 ** -24 * want.abs())[finite].all()
        same = torch.isinf(want) & (got.cpu().double() == want)
        assert (finite | same | (want.abs() >= 1e30)).all()
        check_grad(xd.grad, x64.grad, dtype, coef=(go.abs() / T)[..., None] * (1 + extra[..., None] * 2 ** 22))
    adv, old = torch.randn(1, n, generator=g), want.float().clamp(-50, 0).detach()
    ok = (want > -50) & torch.isfinite(want)
    lab2 = labels.masked_fill(~ok, -100)
    x64 = x.double().requires_grad_()
    wl, wlp = ref64.policy(x64, lab2, old.double(), adv.double(), T=0.2, lo=10.0, hi=10.0)
    wl.backward()
    xd = x.to(device).requires_grad_()
    loss, lp = ta.clipped_policy_loss(xd, lab2.to(device), old.to(device), adv.to(device), temperature=0.2, clip_low=10.0,
                                      clip_high=10.0, return_log_probs=True)
    loss.backward()
    assert ((lp.cpu().double() - wlp).abs() <= LOGP_ABS + extra + 2.0 ** -24 * wlp.abs()).all()
    c = adv.abs()[..., None] / 0.2 / int(ok.sum())
    check_grad(xd.grad, x64.grad, dtype, coef=c * (1 + extra[..., None] * 2 ** 22 + LOGP_ABS * 2 ** 22))


# ---- where a loss is NaN, so is its gradient ---------------------------------------------------

def test_nan_losses_have_nan_gradients(device):
    x, labels, _ = make((2, 4, 600), torch.float32, 151)
    lab = labels.to(device)
    old = torch.full((2, 4), -5.0, device=device)
    adv = torch.ones(2, 4, device=device)
    adv[0, 1] = float("nan")
    leaf = x.to(device).requires_grad_()
    loss = ta.clipped_policy_loss(leaf, lab, old, adv)
    loss.backward()
    assert loss.isnan() and leaf.grad[0, 1].isnan().all() and leaf.grad[0, 0].isfinite().all()
    # an infinite ratio of no advantage: inf * 0
    old[1, 2], adv[0, 1], adv[1, 2] = float("-inf"), 1.0, 0.0
    leaf = x.to(device).requires_grad_()
    loss = ta.clipped_policy_loss(leaf, lab, old, adv)
    loss.backward()
    assert loss.isnan() and leaf.grad[1, 2].isnan().all() and leaf.grad[1, 1].isfinite().all()
    for kind in ("sigmoid", "hinge", "ipo"):
        ref = torch.zeros(2, device=device)
        ref[1] = float("nan")
        leaf = x.to(device).requires_grad_()
        loss = ta.preference_loss(leaf, lab, ref, loss_type=kind)
        loss.backward()
        assert loss.isnan() and leaf.grad.isnan().all(), kind


# ---- many short answers ------------------------------------------------------------------------

@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("n,L", [(5000, 1), (4099, 2), (1300, 3), (700, 17), (257, 33), (9, 64), (3, 65), (2, 1500)])
def test_policy_many_short_answers(device, n, L, reduction):
    x, labels, g = make((n, L, 11), torch.float32, 160 + n + L)
    labels[torch.rand(n, L, generator=g) < 0.4] = -100
    labels[n // 2] = -100
    adv = torch.randn(n, generator=g)
    x64 = x.double().requires_grad_()
    lp, live = ref64.log_probs(x64, labels)
    old = (lp.detach() + torch.randn(n, L, generator=g) * 0.05).float()
    want, _ = ref64.policy(x64, labels, old.double(), adv.double(), lo=0.5, hi=0.5, reduction=reduction, weight=n * L)
    want.backward()
    xd = x.to(device).requires_grad_()
    loss = ta.clipped_policy_loss(xd, labels.to(device), old.to(device), adv.to(device), clip_low=0.5, clip_high=0.5,
                                  reduction=reduction, weight=n * L)
    loss.backward()
    # a term is off by 1e-5 of itself at most (the ratio's exponential of a log probability), and the terms add up in 64 bits
    size = (n * L) * adv.abs().max().item() * 1.5
    assert abs(loss.item() - want.item()) <= 1e-5 * size + 2.0 ** -24 * abs(want.item())
    per = live.sum(-1)
    count = per.sum() if reduction == "token" else (per > 0).sum() * per.clamp_min(1)
    c = (adv.abs() * 1.5 * n * L / count).double()[:, None, None].expand(n, L, 1)
    check_grad(xd.grad, x64.grad, torch.float32, coef=c * (1 + 1e-5 * 2 ** 22))


# ---- a near-certain token behind the first piece of a long row ---------------------------------

@pytest.mark.parametrize("V", [50257, 150001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_log_probs_of_near_certain_tokens(device, V, dtype):
    # Sums are taken relative to an integer near the row's largest exponent, so that the exponent of a token
    # that holds nearly all of the probability is exact but for its last half unit below one: its log
    # probability carries an exponential's and a logarithm's errors, 1.2e-7 and 2e-7, and is within 1e-6.
    g = seeded(170 + V)
    peaks = torch.arange(24, 88).to(dtype) * 0.75
    x = torch.randn(1, peaks.numel(), V, generator=g).to(dtype)
    at = torch.randint(V * 3 // 4, V, (1, peaks.numel()), generator=g)
    x.scatter_(-1, at[..., None], peaks[None, :, None])
    want, _ = ref64.log_probs(x.double(), at)
    xd = x.to(device)
    got = ta.token_log_probs(xd, at.to(device))
    assert ((got.cpu().double() - want).abs() <= 1e-6 + 2.0 ** -24 * want.abs()).all()
    zero = torch.zeros(1, peaks.numel(), device=device)
    _, lp = ta.clipped_policy_loss(xd, at.to(device), zero, zero[:, 0] + 1, return_log_probs=True)
    assert ((lp.cpu().double() - want).abs() <= 1e-6 + 2.0 ** -24 * want.abs()).all()
    # one entry that the teacher is sure of: the row's loss is minus the student's log probability of it
    values = torch.zeros(1, peaks.numel(), 1, device=device)
    for lse in (None, zero):
        loss = ta.top_logits_distil_loss(xd, values, at[..., None].to(device).int(), 1.0, t_logsumexp=lse)
        assert abs(loss.item() + want.mean().item()) <= 1e-6


def test_forward_mode_is_refused(device, monkeypatch):
    import torch.autograd.forward_ad as fw
    x, labels, _ = make((2, 3, 40), torch.float32, 181)
    xd, lab, ref = x.to(device), labels.to(device), torch.zeros(2, 3, device=device)

    def refused():
        with fw.dual_level():
            dual = fw.make_dual(xd, torch.ones_like(xd))
            for call in (lambda: ta.token_log_probs(dual, lab), lambda: ta.preference_loss(dual, lab, ref),
                         lambda: ta.clipped_policy_loss(dual, lab, ref, ref),
                         lambda: ta.top_logits_distil_loss(dual, *ta.top_logits(xd, 3)[:2], 1.0)):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call()
        return True

    assert _both_ways(monkeypatch, refused) == (True, True)


def test_capture_while_an_eager_graph_holds_the_leaf(device, monkeypatch):
    from tspipe_amd import _lib
    x, labels, _ = make((2, 5, 700), torch.float32, 191)
    lab, ref = labels.to(device), torch.zeros(2, 5, device=device)
    leaf = x.to(device).requires_grad_()
    calls = [lambda: ta.token_log_probs(leaf, lab).sum(), lambda: ta.preference_loss(leaf, lab, ref),
             lambda: ta.clipped_policy_loss(leaf, lab, ref, ref),
             lambda: ta.top_logits_distil_loss(leaf, *ta.top_logits(leaf, 3)[:2], 1.0)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        calls[1]()  # (workspaces and code are there before the captures)
    side.synchronize()
    eager = calls[0]()
    want, = torch.autograd.grad(eager, leaf, retain_graph=True)
    host = _lib.host_helper()
    assert host.leaf_on_default_stream(leaf)
    with torch.cuda.stream(side):
        assert host.leaf_on_default_stream(leaf)
        calls[1]()  # outside a capture there is nothing to refuse
    side.synchronize()

    def refused():
        for call in calls:
            with pytest.raises(RuntimeError, match="captured"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    call()
        return True

    assert _both_ways(monkeypatch, refused) == (True, True)
    monkeypatch.undo()
    del eager
    assert not torch.cuda.is_current_stream_capturing()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert not host.leaf_on_default_stream(leaf)
        got, = torch.autograd.grad(calls[0](), leaf)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bits_equal(got, want)


@pytest.mark.parametrize("per_token", [True, False])
@pytest.mark.parametrize("pairs,L", [(3000, 1), (1025, 2), (257, 70), (5, 512), (3, 513), (300, 600)])
def test_preference_many_pairs(device, pairs, L, per_token):
    x, labels, g = make((2 * pairs, L, 7), torch.float32, 200 + pairs + L)
    labels[torch.rand(2 * pairs, L, generator=g) < 0.3] = -100
    labels[1] = -100
    lp, _ = ref64.log_probs(x.double(), labels)
    ref = ((lp if per_token else lp.sum(-1)) + torch.randn(lp.shape if per_token else (2 * pairs,), generator=g) * 0.1).float()
    for average in ((False, True) if per_token else (False,)):
        x64 = x.double().requires_grad_()
        want, wr = ref64.preference(x64, labels, ref.double(), 0.3, average=average, weight=2.0 * pairs)
        want.backward()
        xd = x.to(device).requires_grad_()
        loss, rewards = ta.preference_loss(xd, labels.to(device), ref.to(device), 0.3, length_average=average,
                                           weight=2.0 * pairs, return_rewards=True)
        loss.backward()
        # a sequence's sum is off by LOGP_ABS a token, and 2 sequences by 0.3 of that in a pair's loss, whose slope is below 1
        off = 2 * L * LOGP_ABS * 0.3
        assert abs(loss.item() - want.item()) <= 2 * pairs * off + 2.0 ** -23 * want.item()
        assert ((rewards.cpu().double() - wr).abs() <= off + 2.0 ** -23 * wr.abs()).all()
        # the factor of a row: 0.3 at most times the pair's weight, 2; off by what the slope's argument is
        check_grad(xd.grad, x64.grad, torch.float32, coef=0.6 * (1 + off * 2 ** 22))
