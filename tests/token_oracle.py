"""Plain 64-bit statements of the losses on rows of vocabulary logits, on the
CPU; gradients by autograd.  A row that does not count has label -100."""
import torch

IGNORE = -100


def log_probs(x, labels, T=1.0):
    live = (labels >= 0) & (labels < x.shape[-1])
    lp = (x / T).log_softmax(-1).gather(-1, labels.where(live, torch.zeros_like(labels))[..., None])[..., 0]
    return torch.where(live, lp, torch.zeros_like(lp)), live


def preference(x, labels, ref, beta, kind="sigmoid", smoothing=0.0, average=False, weight=1.0):
    lp, live = log_probs(x, labels)
    per_token = ref.dim() == 2
    d = torch.where(live, lp - (ref if per_token else 0.0), torch.zeros_like(lp)).sum(-1)
    if average:
        d = d / live.sum(-1).clamp_min(1)
    if not per_token:
        d = d - ref
    h = d[0::2] - d[1::2]
    ls = torch.nn.functional.logsigmoid
    if kind == "sigmoid":
        f = -(1 - smoothing) * ls(beta * h) - smoothing * ls(-beta * h)
    elif kind == "hinge":
        f = torch.relu(1 - beta * h)
    else:
        f = (h - 1 / (2 * beta)) ** 2
    return weight * f.mean(), (beta * d).detach()


def policy(x, labels, old, adv, ref=None, kl=0.0, lo=0.2, hi=0.2, T=1.0, reduction="token", weight=1.0):
    lp, live = log_probs(x, labels, T)
    A = adv[:, None].expand_as(lp) if adv.dim() == 1 else adv
    r = (lp - old).exp()
    f = -torch.minimum(r * A, r.clamp(1 - lo, 1 + hi) * A)
    if kl:
        d = ref - lp
        f = f + kl * (d.exp() - d - 1)
    f = torch.where(live, f, torch.zeros_like(f))
    n = live.sum(-1)
    if reduction == "token":
        loss = f.sum() / n.sum()
    else:
        loss = (f.sum(-1) / n.clamp_min(1))[n > 0].mean()
    return weight * loss, torch.where(live, lp, torch.zeros_like(lp)).detach()


def top(x, k, T=1.0):
    """Stable: equal logits in the order of their places."""
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[..., :k]
    return x.gather(-1, order), order, torch.logsumexp(x.double() / T, -1)


def top_distil(x, tv, ti, T, weight=1.0, mask=None, lse=None):
    """Row by row; entries outside the classes are absent, a repeated one counts with each naming."""
    V = x.shape[-1]
    rows = x.reshape(-1, V)
    k = tv.shape[-1]
    tv, ti = tv.reshape(-1, k).double(), ti.reshape(-1, k).long()
    keep = torch.ones(rows.shape[0], dtype=torch.bool) if mask is None else mask.reshape(-1)
    total = rows.sum() * 0.0 if torch.isfinite(rows).all() else torch.zeros((), dtype=torch.float64)
    for r in range(rows.shape[0]):
        if not keep[r]:
            continue
        ok = (ti[r] >= 0) & (ti[r] < V)
        idx, v = ti[r][ok], tv[r][ok] / T
        lq = (rows[r] / T).log_softmax(-1)
        if lse is None:
            lp = v.log_softmax(-1) if v.numel() and (v > float("-inf")).any() else v
        else:
            lp = v - lse.reshape(-1)[r].double()
        p = lp.exp()
        some = p > 0
        term = (p[some] * (lp[some] - lq[idx[some]])).sum()
        if lse is not None:
            inside = torch.zeros(V, dtype=torch.bool)
            inside[idx] = True
            rest = (1 - p.sum()).clamp_min(0)
            if not inside.all() and rest > 0:
                term = term + rest * (rest.log() - torch.logsumexp(lq[~inside], -1))
        total = total + term
    return weight * T * T * total / keep.sum()
