"""Refusals of the token losses and the sparse-teacher operators: before any
GPU work, so they run without a GPU."""
import pytest
import torch

import tspipe_amd as ta
from tspipe_amd import _lib, _vocab

P = 0x1000  # an aligned address that is never touched: every call below is refused first


def test_entry_points_validate_before_launching():
    lib = _lib.lib()
    ARG, ALIGN, RANGE = -1, -4, -5
    fwd = lambda s=P, n=2, L=3, V=10, ls=30, lt=10, lab=P, T=1.0, out=P, st=None, dt=0: lib.ts_token_logp_fwd(  # noqa: E731
        s, n, L, V, ls, lt, lab, None, -100, T, out, st, dt, None)
    assert fwd(dt=7) == ARG and fwd(s=None) == ARG and fwd(V=0) == ARG and fwd(n=-1) == ARG and fwd(lt=-1) == ARG
    assert fwd(T=0.0) == ARG and fwd(T=float("nan")) == ARG and fwd(T=1e-40) == ARG and fwd(lab=None) == ARG
    assert fwd(out=None) == ARG and fwd(s=P + 2) == ALIGN and fwd(lab=P + 4) == ALIGN and fwd(st=P + 4) == ALIGN
    assert fwd(n=1 << 13, L=1 << 12) == RANGE and fwd(V=2 ** 31 - 64) == RANGE
    assert fwd(n=0, s=None, lab=None, out=None) == 0
    assert lib.ts_token_logp_bwd(P, 2, 3, 10, 30, 10, P, None, -100, 1.0, None, P, P, 0, None) == ARG
    assert lib.ts_token_logp_bwd(P, 2, 3, 10, 30, 10, P, None, -100, 1.0, P, P, P + 2, 0, None) == ALIGN
    pref = lambda n=2, beta=0.1, kind=0, sm=0.0, ref=P, ws=P, loss=P: lib.ts_preference_fwd_bwd(  # noqa: E731
        P, n, 3, 10, 30, 10, P, None, -100, ref, 1, beta, kind, sm, 0, 1.0, ws, loss, None, None, 0, None)
    assert pref(n=3) == ARG and pref(beta=0.0) == ARG and pref(kind=3) == ARG and pref(sm=1.5) == ARG
    assert pref(kind=1, sm=0.1) == ARG and pref(ref=None) == ARG and pref(ws=None) == ARG and pref(ws=P + 8) == ALIGN
    pol = lambda old=P, ref=P, kl=0.1, lo=0.8, hi=1.2, ws=P: lib.ts_policy_fwd_bwd(  # noqa: E731
        P, 2, 3, 10, 30, 10, P, None, -100, 1.0, old, ref, P, 0, kl, lo, hi, 0, 1.0, ws, P, None, None, 0, None)
    assert pol(old=None) == ARG and pol(ref=None) == ARG and pol(lo=1.3) == ARG and pol(ws=P + 4) == ALIGN
    top = lambda k=3, V=10, v=P, dt=1: lib.ts_top_logits(P, 1, 2, V, 0, V, k, 1.0, v, P, P, dt, None)  # noqa: E731
    assert top(k=0) == ARG and top(k=11) == ARG and top(k=257, V=1000) == RANGE and top(v=P + 1) == ALIGN and top(v=None) == ARG
    dis = lambda k=3, V=10, tdt=0, lse=None, ws=P, T=1.0: lib.ts_top_distil_fwd_bwd(  # noqa: E731
        P, 1, 2, V, 0, V, P, tdt, P, lse, k, None, T, 1.0, ws, P, None, 0, None)
    assert dis(k=0) == ARG and dis(k=257) == RANGE and dis(tdt=5) == ARG and dis(T=-1.0) == ARG and dis(ws=P + 8) == ALIGN
    assert dis(V=(1 << 20) + 1, lse=P) == RANGE
    assert lib.ts_token_loss_workspace_bytes(-1, 4) == 0 and lib.ts_token_loss_workspace_bytes(4, 7) > 4 * 7 * 16
    assert lib.ts_top_distil_workspace_bytes(5, 7) >= 5 * (8 + 7 * 4)


def test_host_tensors_are_refused():
    x = torch.zeros(2, 3, 10)
    lab = torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ta.token_log_probs(x, lab), lambda: ta.preference_loss(x, lab, x[..., 0]),
                 lambda: ta.clipped_policy_loss(x, lab, x[..., 0], x[..., 0]), lambda: ta.top_logits(x, 3),
                 lambda: ta.top_logits_distil_loss(x, x[..., :3], lab[..., None].expand(2, 3, 3), 1.0)):
        with pytest.raises(TypeError):
            call()


def test_bad_arguments():
    x = torch.zeros(2, 3, 10)
    lab = torch.zeros(2, 3, dtype=torch.int64)
    z = torch.zeros(2, 3)
    with pytest.raises(ValueError):
        ta.token_log_probs(x, lab, temperature=0.0)
    for kw in (dict(loss_type="other"), dict(beta=0.0), dict(label_smoothing=0.1, loss_type="ipo"), dict(label_smoothing=-0.1)):
        with pytest.raises(ValueError):
            ta.preference_loss(x, lab, z, **kw)
    with pytest.raises(ValueError):
        ta.preference_loss(torch.zeros(3, 3, 10), torch.zeros(3, 3, dtype=torch.int64), torch.zeros(3, 3))
    with pytest.raises(ValueError):
        ta.preference_loss(x[0], lab[0], z[0])
    for kw in (dict(reduction="sum"), dict(kl_weight=0.1), dict(clip_low=-0.1), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            ta.clipped_policy_loss(x, lab, z, z, **kw)
    with pytest.raises(ValueError):
        ta.top_logits_distil_loss(x, z, lab, T=0.0)


def test_helpers_refuse_what_does_not_fit():
    z = torch.zeros(2, 3)
    for bad in (torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)):
        with pytest.raises(TypeError):
            _vocab.labels_of(bad, (2, 3), "x")
    with pytest.raises(ValueError):
        _vocab.labels_of(torch.zeros(3, 2, dtype=torch.int64), (2, 3), "x")
    with pytest.raises(ValueError):
        _vocab.mask_of(torch.zeros(5), (2, 3), "x")
    assert _vocab.mask_of(torch.tensor([0.0, 0.5, -1.0]), (3,), "x").tolist() == [0, 1, 1]
    with pytest.raises(TypeError):
        _vocab.floats_of(torch.zeros(2, 3, dtype=torch.int64), (2, 3), "x")
    with pytest.raises(ValueError):
        _vocab.floats_of(z, (3, 2), "x")
    assert _vocab.floats_of(z.double(), (2, 3), "x").dtype == torch.float32
    with pytest.raises(ValueError):
        _vocab.same_device(torch.device("cuda", 0), labels=z)


def test_plug_ins_are_picklable():
    import pickle
    for f in (ta.preference_loss_fn, ta.policy_loss_fn, ta.top_distil_loss_fn):
        assert pickle.loads(pickle.dumps(f)) is f
