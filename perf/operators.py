"""Measured cases of the sparse-teacher and post-training losses.

Five operators over rows of vocabulary logits:

  top            the k largest logits of each teacher row, in order, and the row's log-sum-exp
  distil         distillation from such rows, loss and gradient of the student logits
  log_probs      log probability of one token per row, and its gradient
  preference     paired log ratios against a reference model, loss and gradient
  policy         clipped policy loss with a KL term, loss and gradient

``run`` computes them from elementary torch operations in 32 bits, or, with ``own`` set, through
the package's public functions.  ``exact`` computes them in 64 bits from the definitions.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_IGNORE = -100
_BLOCK = 1 << 27  # logits worked on at a time where inputs and 64-bit values are made


def listed():
    return [
        # a handful of positions whose teacher rows are fetched on demand
        {"name": "top_few", "op": "top", "rows": 8, "vocab": 30522, "k": 16, "temperature": 1.0, "dtype": "bf16"},
        # the teacher's side of a masked-language-model step: 32 sequences of 128 tokens
        {"name": "top_batch", "op": "top", "rows": 4096, "vocab": 30522, "k": 64, "temperature": 2.0, "dtype": "bf16"},
        # a large vocabulary, many entries kept for storing to disk
        {"name": "top_wide", "op": "top", "rows": 1024, "vocab": 131072, "k": 128, "temperature": 1.0, "dtype": "bf16"},
        # image classification, 100 classes, the ten best kept
        {"name": "distil_classes", "op": "distil", "rows": 256, "vocab": 100, "k": 10, "temperature": 4.0, "tail": False,
         "live": 1.0, "dtype": "f32"},
        # the student's side of the same language-model step, padding masked, the teacher's remaining mass as one bucket
        {"name": "distil_batch", "op": "distil", "rows": 4096, "vocab": 30522, "k": 64, "temperature": 2.0, "tail": True,
         "live": 0.85, "dtype": "bf16"},
        # offline distillation over a large vocabulary, every row carries a term; half precision and its loss scale
        {"name": "distil_wide", "op": "distil", "rows": 1024, "vocab": 131072, "k": 128, "temperature": 1.0, "tail": False,
         "live": 1.0, "weight": 65536.0, "dtype": "f16"},
        # scoring one short answer under a frozen model
        {"name": "score_few", "op": "log_probs", "seqs": 1, "length": 24, "vocab": 30522, "temperature": 1.0,
         "grad": False, "live": 0.8, "dtype": "f32"},
        # a user's own objective on token log probabilities: forward and backward
        {"name": "score_train", "op": "log_probs", "seqs": 4, "length": 511, "vocab": 50257, "temperature": 1.0,
         "grad": True, "live": 0.9, "dtype": "bf16"},
        # one pair of short answers on one GPU's micro-batch
        {"name": "pairs_few", "op": "preference", "seqs": 2, "length": 37, "vocab": 30522, "beta": 0.1,
         "loss_type": "sigmoid", "smoothing": 0.0, "live": 0.7, "dtype": "bf16"},
        # eight pairs of ordinary length
        {"name": "pairs_batch", "op": "preference", "seqs": 16, "length": 512, "vocab": 32000, "beta": 0.1,
         "loss_type": "sigmoid", "smoothing": 0.1, "live": 0.7, "dtype": "bf16"},
        # a few short answers, full precision, every answer weighing the same
        {"name": "policy_few", "op": "policy", "seqs": 4, "length": 61, "vocab": 30522, "temperature": 1.0,
         "kl_weight": 0.05, "reduction": "sequence", "live": 0.7, "dtype": "f32"},
        # a training step on sampled answers, every token weighing the same
        {"name": "policy_batch", "op": "policy", "seqs": 8, "length": 1024, "vocab": 65536, "temperature": 0.9,
         "kl_weight": 0.02, "reduction": "token", "live": 0.7, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _loss_scale(case):
    """A gradient that is stored in half precision needs its loss scaled: without it most of it underflows."""
    if case["dtype"] != "f16" or case["op"] in ("top", "log_probs"):
        return case
    if case["op"] == "distil":
        terms = 64 * case["rows"]
    elif case["op"] == "policy":
        terms = 64 * case["seqs"] * case["length"]
    else:
        terms = (64 if case["loss_type"] == "ipo" else 1024) * case["seqs"] // 2
    case["weight"] = 2.0 ** round(math.log2(terms))
    return case


def draw(rng):
    op = rng.choice(["top", "distil", "log_probs", "preference", "policy"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    vocab = _log_int(rng, 100 if op in ("top", "distil") else 1000, 140000)
    most = max(1, min(8192, (1 << 28) // vocab))  # rows that keep a case below the largest listed one
    case = {"op": op, "vocab": vocab, "dtype": dtype, "temperature": rng.choice([0.7, 1.0, 1.0, 2.0, 3.5])}
    if op in ("top", "distil"):
        case["rows"] = _log_int(rng, 1, most)
        case["k"] = _log_int(rng, 1, min(256, vocab))
        if op == "distil":
            case["tail"] = rng.random() < 0.5
            case["live"] = rng.choice([1.0, 0.85, 0.3])
        return _loss_scale(case)
    case["live"] = rng.choice([1.0, 0.9, 0.6])
    case["length"] = _log_int(rng, 1, min(2048, max(1, most // 2)))
    case["seqs"] = _log_int(rng, 1, max(1, most // case["length"]))
    if op == "log_probs":
        case["grad"] = rng.random() < 0.6
    elif op == "preference":
        case["seqs"] = 2 * max(1, case["seqs"] // 2)
        del case["temperature"]
        case["beta"] = rng.choice([0.05, 0.1, 0.5])
        case["loss_type"] = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        case["smoothing"] = rng.choice([0.0, 0.1]) if case["loss_type"] == "sigmoid" else 0.0
    else:
        case["kl_weight"] = rng.choice([0.0, 0.02, 0.1])
        case["reduction"] = rng.choice(["token", "sequence"])
    return _loss_scale(case)


# -- inputs ---------------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) & 0x7FFFFFFF)
    return gen


def _normal(gen, shape, scale, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(0.0, scale, generator=gen)


def _row_log_probs(logits, labels, inv_t):
    """fp32 log probabilities of the labels, a block of rows at a time (inputs only)."""
    flat, lab = logits.reshape(-1, logits.shape[-1]), labels.reshape(-1).clamp_min(0)
    out = torch.empty(lab.shape, dtype=torch.float32, device=flat.device)
    step = max(1, _BLOCK // flat.shape[-1])
    for i in range(0, flat.shape[0], step):
        x = flat[i:i + step].float() * inv_t
        top = x.max(-1, keepdim=True).values
        lse = top[:, 0] + (x - top).exp().sum(-1).log()
        out[i:i + step] = x.gather(1, lab[i:i + step, None])[:, 0] - lse
    return out.view(labels.shape)


def _tokens(case, gen):
    """logits whose sampled token stands out, its labels, and the prompt and padding left out."""
    n, length, vocab = case["seqs"], case["length"], case["vocab"]
    logits = _normal(gen, (n, length, vocab), 2.0, _DTYPES[case["dtype"]])
    tokens = torch.randint(0, vocab, (n, length), device="cuda", generator=gen)
    lift = torch.rand((n, length, 1), device="cuda", generator=gen) * 12.0
    logits.scatter_(2, tokens[..., None], lift.to(logits.dtype))
    # the share of a sequence that is neither prompt nor padding: one run of tokens
    live = max(1, min(length, int(round(length * case["live"]))))
    start = (torch.rand((n, 1), device="cuda", generator=gen) * (length - live + 1)).long().clamp_max(length - live)
    place = torch.arange(length, device="cuda")[None]
    return logits, tokens.masked_fill((place < start) | (place >= start + live), _IGNORE)


def prepare(case, seed):
    gen = _generator(seed)
    dtype, vocab = _DTYPES[case["dtype"]], case["vocab"]
    state = {"case": case}
    if case["op"] == "top":
        state["logits"] = _normal(gen, (case["rows"], vocab), 3.0, dtype)
        return state
    if case["op"] == "distil":
        rows, k, t = case["rows"], case["k"], case["temperature"]
        # a teacher row's best entries: distinct tokens, falling logits, a log-sum-exp above them
        pick = torch.empty((rows, k), dtype=torch.int64, device="cuda")
        step = max(1, _BLOCK // vocab)
        for i in range(0, rows, step):
            r = torch.rand((min(step, rows - i), vocab), device="cuda", generator=gen)
            pick[i:i + step] = r.topk(k, dim=-1).indices
        values = (_normal(gen, (rows, k), 2.0, torch.float32) + 8.0).sort(-1, descending=True).values.to(dtype)
        mass = 0.5 + 0.45 * torch.rand((rows,), device="cuda", generator=gen)
        x = values.float() / t
        state["t_values"], state["t_indices"] = values, pick.to(torch.int32)
        state["t_logsumexp"] = x[:, 0] + (x - x[:, :1]).exp().sum(-1).log() - mass.log() if case["tail"] else None
        student = _normal(gen, (rows, vocab), 2.0, dtype)
        student.scatter_add_(1, pick, (values.float() * 0.7).to(dtype))
        state["logits"] = student.requires_grad_()
        state["row_mask"] = None if case["live"] >= 1.0 else torch.rand((rows,), device="cuda", generator=gen) < case["live"]
        if state["row_mask"] is not None:
            state["row_mask"][0] = True
        return state
    logits, labels = _tokens(case, gen)
    state["labels"] = labels
    if case["op"] == "log_probs":
        state["logits"] = logits.requires_grad_() if case["grad"] else logits
        if case["grad"]:
            state["grad_out"] = _normal(gen, labels.shape, 1.0, torch.float32)
        return state
    near = _row_log_probs(logits, labels, 1.0 / case.get("temperature", 1.0))
    state["ref_log_probs"] = near + _normal(gen, labels.shape, 0.1, torch.float32)
    if case["op"] == "preference":
        # the policy has moved a little towards the preferred answers, which come first in each pair
        state["ref_log_probs"][0::2] -= 0.01
        state["ref_log_probs"][1::2] += 0.01
    if case["op"] == "policy":
        # ratios on both sides of the clipping range, none so close to its ends that the last bits decide
        drift = _normal(gen, labels.shape, 0.2, torch.float32)
        at_end = torch.minimum(((-drift).exp() - 0.8).abs(), ((-drift).exp() - 1.2).abs()) < 1e-3
        state["old_log_probs"] = near + drift.masked_fill(at_end, 0.0)
        state["advantages"] = _normal(gen, (case["seqs"],), 1.0, torch.float32)  # one per sampled answer
    state["logits"] = logits.requires_grad_()
    return state


# -- one pass -------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import tspipe_amd as ta
    case, logits = state["case"], state["logits"]
    op = case["op"]
    if op == "top":
        top = ta.top_logits(logits, case["k"], temperature=case["temperature"])
        return top.values, top.indices, top.logsumexp
    if op == "log_probs":
        out = ta.token_log_probs(logits, state["labels"], temperature=case["temperature"])
        if not case["grad"]:
            return out
        return out.detach(), torch.autograd.grad(out, logits, state["grad_out"])[0]
    if op == "distil":
        loss = ta.top_logits_distil_loss(logits, state["t_values"], state["t_indices"], case["temperature"],
                                         weight=case.get("weight", 1.0), row_mask=state["row_mask"], t_logsumexp=state["t_logsumexp"])
        return loss.detach(), torch.autograd.grad(loss, logits)[0]
    if op == "preference":
        loss, rewards = ta.preference_loss(logits, state["labels"], state["ref_log_probs"], beta=case["beta"],
                                           loss_type=case["loss_type"], label_smoothing=case["smoothing"],
                                           weight=case.get("weight", 1.0), return_rewards=True)
        return loss.detach(), rewards, torch.autograd.grad(loss, logits)[0]
    loss, log_probs = ta.clipped_policy_loss(logits, state["labels"], state["old_log_probs"], state["advantages"],
                                             ref_log_probs=state["ref_log_probs"], kl_weight=case["kl_weight"],
                                             temperature=case["temperature"], reduction=case["reduction"],
                                             weight=case.get("weight", 1.0), return_log_probs=True)
    return loss.detach(), log_probs, torch.autograd.grad(loss, logits)[0]


def _softmax_parts(x):
    """x [rows, vocab] -> (exp(x - max), its sum, max), all [rows, ...] fp32."""
    top = x.max(-1, keepdim=True).values
    e = (x - top).exp()
    return e, e.sum(-1, keepdim=True), top


def _token_rows(logits, labels, inv_t):
    """(probabilities [rows, vocab], log probability of the label in 64 bits, live rows, labels with 0 where none).
    The rows' sums and the log probabilities are 64-bit: whole sequences of them are added up."""
    x = logits.detach().reshape(-1, logits.shape[-1]).float() * inv_t
    lab = labels.reshape(-1)
    live = lab != _IGNORE
    lab = lab.masked_fill(~live, 0)
    top = x.max(-1, keepdim=True).values
    e = (x - top).exp()
    z = e.sum(-1, keepdim=True, dtype=torch.float64)
    logp = ((x.gather(1, lab[:, None]).double() - top.double()) - z.log())[:, 0]
    return e.div_(z.float()), torch.where(live, logp, torch.zeros_like(logp)), live, lab


def _token_grad(p, lab, live, coef, logits):
    """coef * (onehot(label) - p) per row, zero where no label counts, in the logits' type and shape."""
    c = torch.where(live, coef, torch.zeros_like(coef))[:, None]
    g = p.mul_(-c)
    g.scatter_add_(1, lab[:, None], c)
    return g.to(logits.dtype).view(logits.shape)


def _run_plain(state):
    case, logits = state["case"], state["logits"]
    op = case["op"]
    if op == "top":
        # a stable descending sort keeps equal logits in the order of their index
        values, indices = torch.sort(logits, dim=-1, descending=True, stable=True)
        _, z, top = _softmax_parts(logits.float() / case["temperature"])
        k = case["k"]
        return values[:, :k].contiguous(), indices[:, :k].to(torch.int32), (top + z.log())[:, 0]
    if op == "distil":
        return _plain_distil(state)
    inv_t = 1.0 / case.get("temperature", 1.0)
    shape = state["labels"].shape
    p, logp, live, lab = _token_rows(logits, state["labels"], inv_t)
    if op == "log_probs":
        if not case["grad"]:
            return logp.float().view(shape)
        return logp.float().view(shape), _token_grad(p, lab, live, state["grad_out"].reshape(-1) * inv_t, logits)
    seq_live = live.view(shape)
    ref = state["ref_log_probs"]
    if op == "preference":
        ratio = torch.where(seq_live, logp.view(shape) - ref.double(), 0.0).sum(-1)
        h = ratio[0::2] - ratio[1::2]
        beta, eps = case["beta"], case["smoothing"]
        if case["loss_type"] == "sigmoid":
            bh = beta * h
            soft = lambda x: x.clamp_min(0) + (-x.abs()).exp().log1p()  # noqa: E731  log(1 + e^x)
            per = (1 - eps) * soft(-bh) + eps * soft(bh)
            slope = beta * (eps - 1 / (1 + bh.exp()) if eps else -1 / (1 + bh.exp()))
        elif case["loss_type"] == "hinge":
            per = (1 - beta * h).clamp_min(0)
            slope = torch.where(beta * h < 1, -beta, 0.0).to(h)
        else:
            per = (h - 1 / (2 * beta)) ** 2
            slope = 2 * (h - 1 / (2 * beta))
        pairs = h.numel()
        coef = torch.stack([slope, -slope], 1).reshape(-1, 1).expand(shape).reshape(-1) / pairs
        weight = case.get("weight", 1.0)
        return ((weight * per.mean()).float(), (beta * ratio).float(),
                _token_grad(p, lab, live, (weight * coef).float(), logits))
    # (terms of both signs nearly cancel in the loss: 64 bits until it is whole)
    old = state["old_log_probs"].reshape(-1).double()
    adv = state["advantages"].double()[:, None].expand(shape).reshape(-1)
    r = (logp - old).exp()
    free, held = r * adv, r.clamp(0.8, 1.2) * adv
    per = -torch.minimum(free, held)
    slope = torch.where(free <= held, -free, torch.zeros_like(free))
    d = ref.reshape(-1).double() - logp
    per = per + case["kl_weight"] * (d.exp() - d - 1)
    slope = slope + case["kl_weight"] * (1 - d.exp())
    counts = seq_live.sum(-1, keepdim=True)
    if case["reduction"] == "token":
        w = seq_live / counts.sum()
    else:
        w = seq_live / counts.clamp_min(1) / (counts > 0).sum()
    w = w.reshape(-1).double() * case.get("weight", 1.0)
    loss = torch.where(live, w * per, torch.zeros_like(per)).sum()
    return loss.float(), logp.float().view(shape), _token_grad(p, lab, live, (w * slope * inv_t).float(), logits)


def _plain_distil(state):
    case, logits = state["case"], state["logits"]
    t, mask = case["temperature"], state["row_mask"]
    idx = state["t_indices"].long()
    tv = state["t_values"].double() / t
    x = logits.detach().float() / t
    e, z, top = _softmax_parts(x)
    log_q = (x.gather(1, idx) - top - z.log()).double()
    n = x.shape[0] if mask is None else mask.sum()
    if state["t_logsumexp"] is None:
        log_p = tv - (tv.max(-1, keepdim=True).values + (tv - tv.max(-1, keepdim=True).values).exp().sum(-1, keepdim=True).log())
        per = (log_p.exp() * (log_p - log_q)).sum(-1)
        outside = torch.ones_like(z)
    else:
        log_p = tv - state["t_logsumexp"].double()[:, None]
        rest = (1 - log_p.exp().sum(-1)).clamp_min(0)
        e_out = e.scatter(1, idx, 0.0).sum(-1, keepdim=True)
        if case["k"] == case["vocab"]:
            rest = torch.zeros_like(rest)
        q_rest = (e_out / z)[:, 0].double()
        tail = torch.where(rest > 0, rest * (rest.log() - q_rest.log()), torch.zeros_like(rest))
        per = (log_p.exp() * (log_p - log_q)).sum(-1) + tail
        total = log_p.exp().sum(-1) + rest
        outside = (total - torch.where(rest > 0, rest / q_rest, torch.zeros_like(rest))).float()[:, None]
    p = log_p.exp().float()
    q = e.div_(z)
    g = q * outside
    inside = q.gather(1, idx) - p
    if state["t_logsumexp"] is not None:
        inside = q.gather(1, idx) * total.float()[:, None] - p
    g.scatter_(1, idx, inside)
    scale = case.get("weight", 1.0) * t / n
    if mask is not None:
        g = torch.where(mask[:, None], g, torch.zeros_like(g))
        per = torch.where(mask, per, torch.zeros_like(per))
    return (case.get("weight", 1.0) * t * t * per.sum() / n).float(), (g * scale).to(logits.dtype)


# -- what a pass cannot do without --------------------------------------------------------------

def work(case):
    size, vocab = (4 if case["dtype"] == "f32" else 2), case["vocab"]
    op = case["op"]
    if op == "top":
        rows, k = case["rows"], case["k"]
        # one comparison, one exponential and one addition an element
        return {"bytes": rows * (vocab * size + k * (size + 4) + 4), "flops": 3 * rows * vocab}
    if op == "distil":
        rows, k = case["rows"], case["k"]
        live = max(1, int(round(rows * case["live"])))
        move = live * vocab * size + rows * vocab * size + live * k * (size + 4) + (4 * live if case["tail"] else 0)
        return {"bytes": move + (rows if case["live"] < 1.0 else 0), "flops": 6 * live * vocab}
    rows = case["seqs"] * case["length"]
    live = case["seqs"] * max(1, min(case["length"], int(round(case["length"] * case["live"]))))
    move = live * vocab * size + 8 * rows
    if op == "log_probs":
        move += 4 * rows
        if case["grad"]:
            # the gradient of the log probabilities is known only after they were returned: a second reading
            return {"bytes": move + live * vocab * size + rows * vocab * size + 4 * live, "flops": 6 * live * vocab}
        return {"bytes": move, "flops": 3 * live * vocab}
    move += rows * vocab * size + (4 if op == "preference" else 12) * rows
    return {"bytes": move, "flops": 6 * live * vocab}


# -- 64-bit values --------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "top":
        return _exact_top(case, state["logits"])
    if case["op"] == "distil":
        return _exact_distil(case, state)
    return _exact_tokens(case, state)


def _blocks(rows, vocab):
    step = max(1, _BLOCK // vocab)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_top(case, logits):
    rows, vocab = logits.shape
    k = case["k"]
    values, indices, lse = [], [], []
    for lo, hi in _blocks(rows, vocab):
        x = logits[lo:hi].double()
        # equal logits keep the order of their places
        order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :k]
        values.append(logits[lo:hi].gather(1, order))
        indices.append(order.to(torch.int32))
        lse.append(torch.logsumexp(x / case["temperature"], dim=-1))
    return torch.cat(values).double(), torch.cat(indices), torch.cat(lse)


def _exact_distil(case, state):
    """Gradients by differentiating the definition in 64 bits."""
    logits, t, mask = state["logits"].detach(), case["temperature"], state["row_mask"]
    rows, vocab = logits.shape
    n = rows if mask is None else int(mask.sum())
    total = torch.zeros((), dtype=torch.float64, device=logits.device)
    grads = []
    for lo, hi in _blocks(rows, vocab):
        x = logits[lo:hi].double().requires_grad_()
        idx = state["t_indices"][lo:hi].long()
        tv = state["t_values"][lo:hi].double() / t
        log_all = (x / t).log_softmax(-1)
        if state["t_logsumexp"] is None:
            log_p = tv.log_softmax(-1)
            per = (log_p.exp() * (log_p - log_all.gather(1, idx))).sum(-1)
        else:
            log_p = tv - state["t_logsumexp"][lo:hi].double()[:, None]
            per = (log_p.exp() * (log_p - log_all.gather(1, idx))).sum(-1)
            if case["k"] < vocab:
                rest = (1.0 - log_p.exp().sum(-1)).clamp_min(0.0)
                log_rest = torch.logsumexp(log_all.scatter(1, idx, float("-inf")), -1)
                per = per + torch.special.xlogy(rest, rest) - rest * log_rest
        if mask is not None:
            per = torch.where(mask[lo:hi], per, torch.zeros_like(per))
        part = case.get("weight", 1.0) * t * t * per.sum() / n
        grads.append(torch.autograd.grad(part, x)[0])
        total = total + part.detach()
    return total, torch.cat(grads)


def _exact_tokens(case, state):
    logits, labels = state["logits"].detach(), state["labels"]
    n, length, vocab = logits.shape
    t = case.get("temperature", 1.0)
    flat, lab = logits.view(-1, vocab), labels.reshape(-1)
    live = lab != _IGNORE
    safe = lab.clamp_min(0)
    logp = torch.empty(lab.shape, dtype=torch.float64, device=logits.device)
    for lo, hi in _blocks(n * length, vocab):
        rows = (flat[lo:hi].double() / t).log_softmax(-1)
        logp[lo:hi] = rows.gather(1, safe[lo:hi, None])[:, 0]
    logp = torch.where(live, logp, torch.zeros_like(logp)).view(n, length)
    if case["op"] == "log_probs" and not case["grad"]:
        return logp
    lp = logp.clone().requires_grad_()
    on = live.view(n, length)
    if case["op"] == "log_probs":
        out, objective = (logp,), (lp * state["grad_out"].double()).sum()  # (no loss of its own to scale)
    elif case["op"] == "preference":
        beta, eps = case["beta"], case["smoothing"]
        ratio = ((lp - state["ref_log_probs"].double()) * on).sum(-1)
        margin = ratio.view(-1, 2)[:, 0] - ratio.view(-1, 2)[:, 1]
        if case["loss_type"] == "sigmoid":
            win = torch.nn.functional.logsigmoid
            objective = -((1 - eps) * win(beta * margin) + eps * win(-beta * margin)).mean()
        elif case["loss_type"] == "hinge":
            objective = torch.relu(1 - beta * margin).mean()
        else:
            objective = ((margin - 0.5 / beta) ** 2).mean()
        objective = case.get("weight", 1.0) * objective
        out = (objective.detach(), (beta * ratio).detach())
    else:
        adv = state["advantages"].double()[:, None]
        step = lp - state["old_log_probs"].double()
        gain = torch.minimum(step.exp() * adv, step.exp().clamp(0.8, 1.2) * adv)
        away = state["ref_log_probs"].double() - lp
        per = case["kl_weight"] * (away.exp() - away - 1.0) - gain
        per = torch.where(on, per, torch.zeros_like(per))
        if case["reduction"] == "token":
            objective = per.sum() / on.sum()
        else:
            sizes = on.sum(-1)
            objective = (per.sum(-1) / sizes.clamp_min(1))[sizes > 0].mean()
        objective = case.get("weight", 1.0) * objective
        out = (objective.detach(), logp)
    coef = torch.autograd.grad(objective, lp)[0].reshape(-1) * live / t
    grad = torch.empty(flat.shape, dtype=torch.float64, device=flat.device)
    for lo, hi in _blocks(n * length, vocab):
        probs = (flat[lo:hi].double() / t).softmax(-1)
        g = -probs * coef[lo:hi, None]
        g.scatter_add_(1, safe[lo:hi, None], coef[lo:hi, None])
        grad[lo:hi] = g
    return out + (grad.view(logits.shape),)
