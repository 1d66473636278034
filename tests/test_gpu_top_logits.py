"""GPU parity of the sparse-teacher operators: ``top_logits`` (exact values and
places, equal ones by place) and ``top_logits_distil_loss``, against 64-bit
statements on the CPU.

Tolerances: those of the token losses for everything that goes through a row's
statistics (a log probability within 4e-6, a probability within 1e-5 of
itself); a row's loss adds its entries' with weights that sum to at most one.
"""
import pytest
import torch

import token_oracle as ref64
import tspipe_amd as ta
from helpers import bits_equal, rel_err, seeded
from test_gpu_token_losses import DTYPES, LOGP_ABS, check_grad

pytestmark = pytest.mark.gpu


def check_top(x, k, device, T=1.0, xd=None):
    want_v, want_i, want_l = ref64.top(x.float(), k, T)
    top = ta.top_logits(x.to(device) if xd is None else xd, k, T)
    assert top.values.dtype == x.dtype and top.indices.dtype == torch.int32 and top.logsumexp.dtype == torch.float32
    assert torch.equal(top.indices.cpu().long(), want_i)
    assert torch.equal(top.values.cpu().float(), want_v) or torch.isnan(want_v).any()
    ok = torch.isfinite(want_l)
    err = (top.logsumexp.cpu().double() - want_l).abs()[ok]
    assert (err <= LOGP_ABS + 2.0 ** -24 * want_l.abs()[ok]).all()
    return top


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 64, 64), (9, 100, 10), (3, 255, 255), (3, 256, 256),
                                      (4, 1000, 17), (3, 2049, 256), (5, 4099, 1), (3, 30522, 64), (2, 50257, 128),
                                      (2, 65537, 100), (2, 131072, 256), (2, 140003, 31)])
def test_top_logits(device, rows, V, k, dtype):
    g = seeded(V + k)
    check_top((torch.randn(rows, V, generator=g) * 3).to(dtype), k, device, 1.0 if V % 2 else 2.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(50, 20), (3000, 200), (30522, 64), (70001, 256)])
def test_top_logits_ties(device, V, k, dtype):
    g = seeded(7 * V)
    x = torch.randint(-2, 3, (6, V), generator=g).to(dtype)      # thousands of equal logits
    x[1] = 0                                                     # all equal
    x[2, ::2] = -0.0                                             # +0 and -0 are equal
    x[2, 1::2] = 0.0
    x[3] = torch.finfo(dtype).min                                # nothing but the lowest value
    x[4] = float("-inf")
    x[4, V - 1] = 1.0                                            # one finite logit, at the end
    x[5] = torch.arange(V).div(V / 100, rounding_mode="floor").to(dtype)  # rising in steps: the best lie together
    check_top(x, k, device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(300, 40), (30522, 64), (50257, 200)])
def test_top_logits_sorted_rows(device, V, k, dtype):
    # rows in falling and in rising order: the largest all lie in one place
    g = seeded(11 * V)
    x = (torch.randn(4, V, generator=g) * 3).to(dtype)
    x[0] = x[0].sort(descending=True).values
    x[1] = x[1].sort().values
    x[2, 1000 % V:] = x[2, 1000 % V:] - 100
    check_top(x, k, device)


def test_top_logits_nan_and_infinities(device):
    g = seeded(13)
    x = torch.randn(4, 5000, generator=g)
    x[0, 77] = float("inf")
    x[1, [5, 4000]] = float("nan")
    x[2] = float("-inf")
    x[3, 100:] = float("-inf")
    top = ta.top_logits(x.to(device), 120)
    i = top.indices.cpu()
    assert i[0, 0] == 77 and i[1, :2].tolist() == [5, 4000] and torch.isnan(top.values[1, :2]).all()
    assert i[2].tolist() == list(range(120)) and i[3, 100:].tolist() == list(range(100, 120))
    assert top.logsumexp[0].item() == float("inf") and torch.isnan(top.logsumexp[1]) and top.logsumexp[2].item() == float("-inf")


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logits_views(device, dtype):
    g = seeded(17)
    x = (torch.randn(3, 5, 4001, generator=g) * 3).to(dtype)
    xd = x.to(device)
    check_top(x[:, :-1].contiguous(), 33, device, xd=xd[:, :-1])
    check_top(x[:, 1::2].contiguous(), 33, device, xd=xd[:, 1::2])
    check_top(x.transpose(0, 1).contiguous(), 33, device, xd=xd.transpose(0, 1))
    check_top(x[..., 1:].contiguous(), 33, device, xd=xd[..., 1:])       # rows off a 16-byte boundary
    check_top(x[..., ::2].contiguous(), 33, device, xd=xd[..., ::2])     # copied
    check_top(x[0, 0], 33, device)
    for shape in [(0, 50), (2, 0, 50)]:
        assert ta.top_logits(torch.zeros(shape, device=device), 3).values.shape == shape[:-1] + (3,)


# ---- distillation ------------------------------------------------------------------------------

def teacher(rows, V, k, g, dtype, T, spread=2.0):
    t = torch.randn(rows, V, generator=g) * spread
    order = torch.argsort(t, dim=-1, descending=True)[:, :k]
    vals = t.gather(-1, order).to(dtype)
    # of the rounded logits, so that the kept entries' probabilities stay below one in all
    lse = torch.logsumexp(t.to(dtype).double() / T, -1).float()
    return vals, order.to(torch.int32), lse


def run_case(device, x, vals, idx, T, weight, mask, lse):
    x64 = x.double().requires_grad_()
    want = ref64.top_distil(x64, vals, idx, T, weight, mask, lse)
    want.backward()
    xd = x.to(device).requires_grad_()
    loss = ta.top_logits_distil_loss(xd, vals.to(device), idx.to(device), T, weight,
                                     None if mask is None else mask.to(device), None if lse is None else lse.to(device))
    loss.backward()
    # (a row's term moves by what its log probabilities do, and by one rounding of the 64-bit sum)
    assert abs(loss.item() - want.item()) <= weight * T * T * 2 * LOGP_ABS + 2.0 ** -23 * abs(want.item())
    n = x.reshape(-1, x.shape[-1]).shape[0] if mask is None else int(mask.sum())
    check_grad(xd.grad, x64.grad, x.dtype, coef=weight * T / max(n, 1))
    return loss, xd.grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,V,k,T", [(1, 1, 1, 1.0), (2, 2, 1, 1.0), (7, 5, 3, 2.0), (6, 100, 10, 4.0), (3, 256, 256, 2.0),
                                        (5, 1000, 17, 1.0), (3, 2049, 200, 3.5), (4, 30522, 64, 2.0), (3, 50257, 128, 1.0),
                                        (2, 131072, 256, 0.7), (2, 140003, 5, 1.0)])
def test_distil(device, rows, V, k, T, tail, dtype):
    g = seeded(3000 + V + k)
    vals, idx, lse = teacher(rows, V, k, g, dtype, T)
    x = (torch.randn(rows, V, generator=g) * 2).to(dtype)
    x.scatter_add_(1, idx.long(), (vals.float() * 0.6).to(dtype))
    mask = None
    if rows > 2:
        mask = torch.rand(rows, generator=g) < 0.7
        mask[0], mask[1] = True, False
    run_case(device, x, vals, idx, T, 64.0 * rows, mask, lse if tail else None)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V", [90, 5001, 40000])
def test_distil_odd_entries(device, V, tail):
    # absent entries, the same token twice, -inf values, rows of nothing but absent entries, int64 indices,
    # a teacher of another type
    g = seeded(3500 + V)
    rows, k, T = 6, 12, 2.0
    vals, idx, lse = teacher(rows, V, k, g, torch.bfloat16, T)
    idx = idx.long()
    lse = lse + 0.7  # room for the entries named twice
    idx[0, 3] = -1
    idx[0, 5] = V
    idx[1, 7] = idx[1, 2]
    idx[1, 8] = idx[1, 2]
    vals[2, 4:] = float("-inf")
    idx[3] = -1
    idx[4, 0] = 2 ** 40
    x = torch.randn(rows, V, generator=g) * 2
    loss, grad = run_case(device, x, vals, idx, T, 100.0, None, lse if tail else None)
    assert (grad[3] == 0).all() if not tail else grad[3].abs().max() < 1e-4


def test_distil_values_all_absent_or_minus_inf(device):
    x = torch.randn(3, 700, generator=seeded(5)).to(device).requires_grad_()
    vals = torch.full((3, 4), float("-inf"), device=device)
    idx = torch.arange(4, device=device).expand(3, 4).to(torch.int32)
    loss = ta.top_logits_distil_loss(x, vals, idx, 1.0)
    loss.backward()
    assert loss.item() == 0 and (x.grad == 0).all()


def test_distil_student_masked_vocabulary(device):
    # the student cannot reach part of the vocabulary: finite where the teacher does not ask for it,
    # infinite loss with a finite gradient where it does
    g = seeded(6)
    vals, idx, lse = teacher(2, 3000, 20, g, torch.float32, 1.0)
    x = torch.randn(2, 3000, generator=g)
    free = torch.ones(2, 3000, dtype=torch.bool)
    free.scatter_(1, idx.long(), False)
    far = free & (torch.rand(2, 3000, generator=g) < 0.5)
    x = x.masked_fill(far, float("-inf"))
    for l in (None, lse):
        run_case(device, x, vals, idx, 1.0, 10.0, None, l)
    y = x.clone()
    y[0, idx[0, 1]] = float("-inf")
    yd = y.to(device).requires_grad_()
    loss = ta.top_logits_distil_loss(yd, vals.to(device), idx.to(device), 1.0)
    loss.backward()
    assert loss.item() == float("inf") and torch.isfinite(yd.grad).all()
    z = x.masked_fill(free, float("-inf")).to(device).requires_grad_()  # nothing left for the rest
    loss = ta.top_logits_distil_loss(z, vals.to(device), idx.to(device), 1.0, t_logsumexp=lse.to(device))
    loss.backward()
    assert loss.item() == float("inf") and torch.isfinite(z.grad).all()


def test_distil_nan_outside_the_selection(device):
    g = seeded(9)
    vals, idx, lse = teacher(4, 2000, 8, g, torch.float32, 1.0)
    x = torch.randn(4, 2000, generator=g)
    x[1] = float("nan")
    mask = torch.tensor([True, False, True, True])
    xd = x.to(device).requires_grad_()
    loss = ta.top_logits_distil_loss(xd, vals.to(device), idx.to(device), 1.0, row_mask=mask.to(device))
    loss.backward()
    assert torch.isfinite(loss) and (xd.grad[1] == 0).all()
    loss = ta.top_logits_distil_loss(xd, vals.to(device), idx.to(device), 1.0)
    assert torch.isnan(loss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_all_entries_kept_is_the_dense_loss(device, dtype):
    g = seeded(21)
    rows, V, T = 40, 200, 3.0
    t, s = ((torch.randn(rows, V, generator=g) * 3).to(dtype).to(device) for _ in range(2))
    a, b = s.clone().requires_grad_(), s.clone().requires_grad_()
    dense = ta.kd_soft_target_loss(a, t, T)
    dense.backward()
    for tail in (False, True):
        b.grad = None
        top = ta.top_logits(t, V, T)
        sparse = ta.top_logits_distil_loss(b, top.values, top.indices, T, t_logsumexp=top.logsumexp if tail else None)
        sparse.backward()
        # each within 2 * 4e-6 * T^2 of the value (fp32 sums of the dense kernel included)
        assert abs(dense.item() - sparse.item()) < 4 * LOGP_ABS * T * T
        check_grad(b.grad, a.grad.double().cpu(), dtype, coef=4 * T / rows * (1 + torch.finfo(dtype).eps * 2 ** 20))


@pytest.mark.parametrize("V", [1501, 1504])
def test_distil_views_and_empty(device, V):
    # a slice of every sequence, read where it lies; the bits of a dense copy's where the rows start at the
    # same distance from a 16-byte boundary as its rows do (V a multiple of 8: the sums run in one order)
    g = seeded(23)
    B, L, k = 3, 4, 9
    vals, idx, lse = teacher(B * (L - 1), V, k, g, torch.float32, 1.0)
    vals, idx, lse = (t.view(B, L - 1, *t.shape[1:]).to(device) for t in (vals, idx, lse))
    whole = torch.randn(B, L, V, generator=g).to(device)
    dense = whole[:, :-1].contiguous().requires_grad_()
    a = ta.top_logits_distil_loss(dense, vals, idx, 2.0, t_logsumexp=lse)
    a.backward()
    leaf = whole.clone().requires_grad_()
    b = ta.top_logits_distil_loss(leaf[:, :-1], vals, idx, 2.0, t_logsumexp=lse)
    b.backward()
    x64 = whole[:, :-1].cpu().double().requires_grad_()
    want = ref64.top_distil(x64, vals.cpu(), idx.cpu(), 2.0, lse=lse.cpu())
    want.backward()
    for loss, grad in ((a, dense.grad), (b, leaf.grad[:, :-1])):
        assert abs(loss.item() - want.item()) <= 4 * 2 * LOGP_ABS + 2.0 ** -23 * abs(want.item())
        check_grad(grad, x64.grad, torch.float32, coef=2.0 / (B * (L - 1)))
    assert (leaf.grad[:, -1] == 0).all()
    if V % 8 == 0:
        assert bits_equal(a, b) and bits_equal(leaf.grad[:, :-1], dense.grad)
    x = torch.zeros(0, 50, device=device, requires_grad=True)
    loss = ta.top_logits_distil_loss(x, torch.zeros(0, 3, device=device), torch.zeros(0, 3, dtype=torch.int32, device=device), 1.0)
    assert torch.isnan(loss)
    loss.backward()
    x = torch.randn(4, 50, device=device, requires_grad=True)
    none = torch.zeros(4, dtype=torch.bool, device=device)
    loss = ta.top_logits_distil_loss(x, torch.zeros(4, 3, device=device), torch.zeros(4, 3, dtype=torch.int32, device=device), 1.0,
                                     row_mask=none)
    assert torch.isnan(loss)
    loss.backward()
    assert (x.grad == 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distil_against_differences(device, tail):
    g = seeded(25)
    vals, idx, lse = (t.to(device) for t in teacher(5, 600, 12, g, torch.float32, 2.0))
    x = torch.randn(5, 600, generator=g).to(device).requires_grad_()
    f = lambda t: ta.top_logits_distil_loss(t, vals, idx, 2.0, t_logsumexp=lse if tail else None)  # noqa: E731
    f(x).backward()
    d = torch.randn(5, 600, generator=g).to(device)
    h = 1e-2
    with torch.no_grad():
        numeric = (f(x + h * d).double() - f(x - h * d).double()).item() / (2 * h)
    # T^2 * 8e-6 over h, and h^2 / 6 times third derivatives of order T^-1
    assert abs(numeric - (x.grad.double() * d).sum().item()) < 4 * 2 * LOGP_ABS / h + h * h


def test_sparse_teacher_pipeline(device):
    # teacher stage -> entries -> student stage, through the plug-in, with the bits of the calls made by hand,
    # and close to the dense loss when the kept entries carry nearly all of the mass
    g = seeded(27)
    B, L, V = 3, 16, 4000

    class P:
        temperature, alpha_ce, top_k, restrict_ce_to_mask = 2.0, 0.5, 64, False

    t = (torch.randn(B, L, V, generator=g) * 6).to(torch.bfloat16).to(device)
    s = (torch.randn(B, L, V, generator=g) * 2).to(torch.bfloat16).to(device)
    att = (torch.rand(B, L, generator=g) < 0.8).to(device)
    labels = (torch.full((B, L), -1, device=device), att)
    a = s.clone().requires_grad_()
    loss = ta.top_distil_loss_fn({"logits": a}, {"logits": t}, labels, None, P(), 0)
    loss.backward()
    top = ta.top_logits(t, 64, 2.0)
    b = s.clone().requires_grad_()
    shipped = {"top_values": top.values, "top_indices": top.indices, "top_logsumexp": top.logsumexp}
    again = ta.top_distil_loss_fn({"logits": b}, shipped, labels, None, P(), 0)
    again.backward()
    assert bits_equal(loss, again) and bits_equal(a.grad, b.grad)
    dense = ta.distil_ce_loss(s, t, att, 2.0, 0.5)
    assert loss.item() <= dense.item() + 1e-3 and rel_err(loss.item(), dense.item()) < 0.2
    assert dense.item() > 0


def test_graph_capture_replays(device):
    g = seeded(29)
    t, s = ((torch.randn(64, 3001, generator=g) * 3).to(torch.bfloat16).to(device) for _ in range(2))
    static = s.clone().requires_grad_()

    def step(x):
        top = ta.top_logits(t, 32, 2.0)
        loss = ta.top_logits_distil_loss(x, top.values, top.indices, 2.0, t_logsumexp=top.logsumexp)
        return [*top, loss.detach(), torch.autograd.grad(loss, x)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for trial in range(4):
        fresh = (s.float() * (1 + 0.2 * trial)).to(torch.bfloat16)
        with torch.no_grad():
            static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(fresh.requires_grad_())):
            assert bits_equal(a, b), trial


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [700, 9000, 40000, 150001])
def test_masked_stretches(device, V, dtype):
    g = seeded(33 + V)
    rows = []
    for fill in (-1e4, float("-inf"), torch.finfo(dtype).min):
        for lo, hi in ((0, V // 2), (V // 2, V - 3)):
            r = torch.randn(V, generator=g) * 3
            r[lo:hi] = fill
            rows.append(r)
    rows.append(torch.randn(V, generator=g).abs() * -3 - 1)     # no logit above zero
    rows.append(torch.randn(V, generator=g).abs() * -3 - 1e4)
    x = torch.stack(rows).to(dtype)
    k = 50
    top = check_top(x, k, device)
    # the student is masked the same way, the teacher's kept entries are not among the masked
    s = x.float().clone()
    live = s > -9e3
    live[-1] = True
    s = torch.where(live, s + torch.randn(s.shape, generator=g) * 0.5, s).to(dtype)
    for lse in (None, top.logsumexp.cpu()):
        run_case(device, s, top.values.cpu(), top.indices.cpu(), 1.0, 64.0 * len(rows), None, lse)


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("V,k", [(150, 150), (900, 256), (2062, 256), (2063, 256), (4100, 200), (8200, 256), (16390, 256),
                                 (32790, 256), (70000, 256), (300000, 256)])
def test_top_logits_many_entries(device, V, k, rows):
    if rows * V > 10 ** 7:
        rows = 3
    g = seeded(V - k)
    for dtype in DTYPES:
        check_top((torch.randn(rows, V, generator=g) * 2).to(dtype), min(k, V), device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,k", [(200, 64), (2500, 64), (12000, 200), (30522, 64), (140001, 64)])
def test_top_logits_fewer_left_than_asked_for(device, V, k, dtype):
    # the vocabulary masked but for fewer than k tokens (or for just k, or one more): the masked ones follow by place
    g = seeded(41 + V)
    fi = torch.finfo(dtype)
    rows = []
    for fill in (float("-inf"), fi.min, -1e4, 0.0):
        for live in (0, 1, 2, k - 1, k, k + 1):
            r = torch.full((V,), fill)
            r[torch.randperm(V, generator=g)[:live]] = torch.randn(live, generator=g) * 3
            rows.append(r)
    x = torch.stack(rows).to(dtype)
    check_top(x, k, device)
    x[:, V // 2] = float("nan")  # with a NaN in every row: the largest, and the others in their order
    top = ta.top_logits(x.to(device), k)
    assert (top.indices[:, 0] == V // 2).all() and top.logsumexp.isnan().all()
    x[:, V // 2] = float("inf")
    assert torch.equal(top.indices.cpu().long(), ref64.top(x.float(), k)[1])


def test_offsets_beyond_32_bits(device):
    # 2.36e9 logits, 4.7 GB: the last rows against the same rows in a tensor of their own
    rows, V, n = 36000, 65536, 6
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=device)
    g = seeded(51)
    own = (torch.randn(n, V, generator=g) * 3).to(torch.bfloat16).to(device)
    x[-n:] = own
    live = torch.arange(rows, device=device) >= rows - n
    labels = torch.full((rows,), -100, device=device)
    labels[-n:] = torch.randint(0, V, (n,), generator=g).to(device)
    for a, b in zip(ta.top_logits(x, 20), ta.top_logits(own, 20)):
        assert bits_equal(a[-n:].contiguous(), b) and (a[0] == a[7]).all()
    top = ta.top_logits(own, 20)
    values, indices = torch.zeros(rows, 20, dtype=torch.bfloat16, device=device), torch.zeros(rows, 20, dtype=torch.int32, device=device)
    lse = torch.zeros(rows, device=device)
    values[-n:], indices[-n:], lse[-n:] = top.values, top.indices, top.logsumexp + 0.1
    ref, adv = torch.full((rows,), -9.0, device=device), torch.ones(rows, device=device)

    def losses(t, m):  # m: the rows' part of the inputs
        two = t.view(2, -1, V)
        pair = lambda v: v[m].view(2, -1)  # noqa: E731
        yield lambda: ta.token_log_probs(t, labels[m]).sum()
        yield lambda: ta.clipped_policy_loss(two, pair(labels), pair(ref), pair(adv), pair(ref), 0.1)
        yield lambda: ta.top_logits_distil_loss(t, values[m], indices[m], 2.0, row_mask=live[m], t_logsumexp=lse[m])

    every, last = slice(0, rows), slice(rows - n, rows)
    big, small = x.requires_grad_(), own.clone().requires_grad_()
    for f, h in zip(losses(big, every), losses(small, last)):
        a, b = f(), h()
        assert bits_equal(a.detach(), b.detach())
        ga, = torch.autograd.grad(a, big)
        gb, = torch.autograd.grad(b, small)
        assert bits_equal(ga[-n:].contiguous(), gb)
        assert not ga[:rows - n].any()
        del ga, a
    # the second answer of a pair lies behind the 32 bits
    big3, small3 = big.detach().view(2, -1, V).requires_grad_(), torch.zeros(2, n, V, dtype=torch.bfloat16, device=device)
    small3[1] = own
    small3.requires_grad_()
    lab3 = torch.full((2, n), -100, device=device)
    lab3[1] = labels[-n:]
    a = ta.preference_loss(big3, labels.view(2, -1), torch.zeros(2, device=device))
    b = ta.preference_loss(small3, lab3, torch.zeros(2, device=device))
    assert bits_equal(a.detach(), b.detach())
    ga, = torch.autograd.grad(a, big3)
    gb, = torch.autograd.grad(b, small3)
    assert bits_equal(ga[1, -n:].contiguous(), gb[1]) and gb[1].any() and not ga[0].any() and not ga[1, :-n].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,k", [(150001, 40), (150001, 256), (262144, 8)])
def test_distil_rows_too_long_for_registers(device, V, k, tail, dtype):
    # masked rows, absent and repeated entries, rows of the type's lowest value (uniform) and of -inf but for a few
    # tokens, rows that start at odd addresses and lie apart, no gradient wanted
    g = seeded(61 + V + k)
    n, L, T = 2, 4, 1.5
    vals, idx, lse = teacher(n * L, V, k, g, dtype, T)
    lse = lse + 0.7
    x = (torch.randn(n * L, V, generator=g) * 2).to(dtype)
    x.scatter_add_(1, idx.long(), (vals.float() * 0.6).to(dtype))
    idx[0, 1], idx[0, 2], idx[1, 3] = -1, V, idx[1, 0]
    x[3] = torch.finfo(dtype).min
    x[4] = float("-inf")
    x[4, -2:] = 1.0
    idx[4] = -1
    idx[4, 0], idx[4, 1] = V - 1, V - 2
    mask = torch.tensor([1, 1, 0, 1, 1, 0, 1, 1]).bool()
    lse = lse if tail else None
    if tail:  # (what the teacher leaves to others, the student of row 4 cannot reach)
        lse[4] = torch.logsumexp(vals[4, :2].double() / T, -1).float() - 1e-3
    loss, grad = run_case(device, x, vals, idx, T, 64.0 * n * L, mask, lse)
    assert (grad[~mask.to(device)] == 0).all()
    wide = torch.full((n, L + 1, V + 3), float("nan"), dtype=dtype, device=device)
    view = wide[:, 1:, 1:V + 1]
    view.copy_(x.view(n, L, V))
    leaf = view.detach().requires_grad_()
    three = lambda t: None if t is None else t.to(device).view(n, L, *t.shape[1:])  # noqa: E731
    again = ta.top_logits_distil_loss(leaf, three(vals), three(idx), T, 64.0 * n * L, three(mask), three(lse))
    again.backward()
    assert abs(again.item() - loss.item()) <= 64.0 * n * L * T * T * 4 * LOGP_ABS + 2.0 ** -22 * abs(loss.item())
    want = grad.view(n, L, V).double()
    # (a row that starts elsewhere is summed in another order: each of the two within its own bound)
    check_grad(leaf.grad, want.cpu(), dtype, coef=64.0 * T * n * L / 6 * 2 + 2 ** 22 * torch.finfo(dtype).eps / 2 * want.abs().cpu())
    with torch.no_grad():
        assert bits_equal(ta.top_logits_distil_loss(leaf, three(vals), three(idx), T, 64.0 * n * L, three(mask), three(lse)), again.detach())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("k", [64, 65, 130, 256])
def test_distil_tokens_named_again_and_again(device, k, tail):
    # one token twice, far apart and next to each other; every token twice; one token throughout; none twice;
    # tokens 512 apart and neighbours
    g = seeded(71 + k)
    rows, V, T = 7, 140001, 2.0
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)]).to(torch.int32)
    idx[0, k - 1] = idx[0, 0]
    idx[1, 1] = idx[1, 0]
    idx[2, 1::2] = idx[2, :k - 1:2] if k % 2 else idx[2, ::2]
    idx[3] = 77
    idx[5] = torch.arange(k) * 512 % V
    idx[6] = torch.arange(V - k, V)
    idx[6, 2] = -1
    vals = torch.randn(rows, k, generator=g).sort(-1, descending=True).values
    lse = torch.logsumexp(vals.double() / T, -1).float() + 0.5
    x = torch.randn(rows, V, generator=g) * 2
    run_case(device, x, vals, idx, T, 64.0 * rows, None, lse if tail else None)


def test_as_many_rows_as_are_taken(device):
    n, V, k = 4_194_302, 5, 2
    g = seeded(81)
    x = torch.randn(n, V, generator=g) * 2
    xd = x.to(device)
    top = ta.top_logits(xd, k)
    want_v, want_i = torch.sort(x, dim=-1, descending=True, stable=True)
    assert torch.equal(top.indices.cpu().long(), want_i[:, :k]) and torch.equal(top.values.cpu(), want_v[:, :k])
    labels = torch.randint(0, V, (n,), generator=g)
    go = torch.randn(n, generator=g)
    lp = x.double().log_softmax(-1)
    at = lp.gather(-1, labels[:, None])[:, 0]
    leaf, lab = xd.clone().requires_grad_(), labels.to(device)
    got = ta.token_log_probs(leaf, lab)
    assert ((got.detach().cpu().double() - at).abs() <= LOGP_ABS + 2.0 ** -24 * at.abs()).all()
    got.backward(go.to(device))
    onehot = torch.nn.functional.one_hot(labels, V).double()
    slope = onehot - lp.exp()
    check_grad(leaf.grad, go.double()[:, None] * slope, torch.float32, coef=go.abs()[:, None])
    # one token an answer, weights that make a row's factor of the order of one
    old, adv = (at + torch.randn(n, generator=g) * 0.05).float(), torch.randn(n, generator=g)
    ratio = (at - old.double()).exp()
    leaf = xd.clone().requires_grad_()
    loss = ta.clipped_policy_loss(leaf.view(n, 1, V), lab.view(n, 1), old.to(device).view(n, 1), adv.to(device), clip_low=0.9,
                                  clip_high=9.0, reduction="sequence", weight=float(n))
    loss.backward()
    terms = -ratio * adv.double()
    assert abs(loss.item() - terms.sum().item()) <= 1e-5 * terms.abs().sum().item()
    check_grad(leaf.grad, terms[:, None] * slope, torch.float32, coef=adv.abs()[:, None] * 1.5 * (1 + 1e-5 * 2 ** 22))
    ref = (at + torch.randn(n, generator=g) * 0.1).float()
    r = at - ref.double()
    h = r[0::2] - r[1::2]
    leaf = xd.clone().requires_grad_()
    loss, rewards = ta.preference_loss(leaf.view(n, 1, V), lab.view(n, 1), ref.to(device), 0.5, weight=n / 2.0,
                                       return_rewards=True)
    loss.backward()
    pair = torch.nn.functional.softplus(-0.5 * h)
    assert abs(loss.item() - pair.sum().item()) <= 1e-5 * pair.sum().item()
    assert ((rewards.cpu().double() - 0.5 * r).abs() <= LOGP_ABS + 2.0 ** -23 * r.abs()).all()
    c = torch.stack((-0.5 * torch.sigmoid(-0.5 * h), 0.5 * torch.sigmoid(-0.5 * h)), -1).view(-1)
    check_grad(leaf.grad, c[:, None] * slope, torch.float32, coef=c.abs()[:, None] * (1 + 1e-5 * 2 ** 22))
    leaf = xd.clone().requires_grad_()
    loss = ta.top_logits_distil_loss(leaf, top.values, top.indices, 1.0, weight=float(n))
    loss.backward()
    p = torch.zeros(n, V, dtype=torch.float64).scatter_(-1, want_i[:, :k], want_v[:, :k].double().softmax(-1))
    term = (torch.special.xlogy(p, p) - p * lp).sum()
    assert abs(loss.item() - term.item()) <= 1e-5 * term.item()
    check_grad(leaf.grad, lp.exp() - p, torch.float32, coef=torch.ones(n, 1))
    with pytest.raises(Exception):
        ta.top_logits(torch.zeros(1 << 22, 1, device=device), 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows", [257, 700])
def test_distil_wide_rows_by_the_hundred(device, rows, tail, dtype):
    # more rows than a GPU has compute units, of the widest arrangement: the same bits as a few rows at a time,
    # whatever rows are masked, need the true maximum or start at odd addresses
    V, k, T = (33003 if dtype == torch.float32 else 65607), 30, 2.0
    g = torch.Generator(device=device).manual_seed(91)
    x = torch.randn(rows, V, generator=g, device=device, dtype=torch.float32).mul_(2).to(dtype)
    x[5] = torch.finfo(dtype).min
    x[300:303] = float("-inf")
    x[300:303, 7] = 1.0
    mask = torch.rand(rows, generator=g, device=device) < 0.7
    mask[5] = mask[300:303] = True
    mask[256:259] = torch.tensor([True, False, True], device=device)[:max(0, rows - 256)]
    top = ta.top_logits(x.roll(1, 0), k, T)
    lse = top.logsumexp + 0.5 if tail else None

    def run(part):
        n = int(mask[part].sum())
        leaf = x[part].clone().requires_grad_()
        loss = ta.top_logits_distil_loss(leaf, top.values[part], top.indices[part], T, float(max(n, 1)), row_mask=mask[part],
                                         t_logsumexp=None if lse is None else lse[part])
        loss.backward()
        return loss.detach(), leaf.grad

    _, whole = run(slice(0, rows))
    for lo in range(0, rows, 8):
        part = slice(lo, min(lo + 8, rows))
        _, grad = run(part)
        for i in range(grad.shape[0]):  # (odd V: every row starts at another address than in the whole only if lo is odd)
            if mask[lo + i]:
                assert bits_equal(whole[lo + i], grad[i]), lo + i
            else:
                assert not whole[lo + i].any()
