"""Refusals of the loss and block-table entry points that need no device, and the 64-bit definitions against automatic
differentiation."""
import ctypes as C

import numpy as np
import pytest
import torch

import loss_ref as ref

P = 0x1000  # an address that no refused call touches


def status(fn, *args):
    from whirl_llm_b200 import api
    s = getattr(api.lib, fn)(*args)
    return s, api.lib.whirl_last_error().decode()


def test_logprobs_refusals():
    ok = [P, 0, 4, 100, 100, P, 1.0, None, P, P, None, None]
    for i, v, what in [(0, None, "null"), (1, 7, "dtype"), (2, -1, "rows"), (3, 0, "n"), (4, 99, "ld"), (5, None, "null"), (6, 0.0, "inv_t"),
                       (6, -1.0, "inv_t"), (6, float("nan"), "inv_t"), (6, float("inf"), "inv_t"), (0, P + 2, "aligned")]:
        a = list(ok)
        a[i] = v
        s, msg = status("whirl_token_logprobs", *a)
        assert s == 1 and what in msg, (i, v, s, msg)
    a = list(ok)
    a[2] = 0
    assert status("whirl_token_logprobs", *a)[0] == 0          # no rows: nothing to do
    a = list(ok)
    a[8] = a[9] = None
    assert status("whirl_token_logprobs", *a)[0] == 0          # no outputs


def test_grad_refusals():
    big = P + 100 * 4 * 4
    ok = [P, 0, 4, 100, 100, P, 1.0, None, P, None, P, None, big, 100, None]
    for i, v in [(8, None), (10, None), (12, None), (11, P), (13, 99), (12, P + 4), (12, big - 4), (12, big + 1)]:
        a = list(ok)
        a[i] = v
        assert status("whirl_token_logprobs_grad", *a)[0] == 1, (i, v)


def test_policy_refusals():
    from whirl_llm_b200 import api
    need = api.lib.whirl_loss_workspace_bytes(4, 2)

    def call(ws=P, ws_bytes=need, x=P, ld_dx=100, loss=P, dx=None, **kw):
        p = dict(token=P, adv=P, seqs=0, mean=1, inv_t=1.0, clip_low=0.2, clip_high=0.2)
        p.update(kw)
        o = api.PolicyOut(loss=loss, dx=dx, ld_dx=ld_dx)
        return status("whirl_policy_loss", x, 0, 4, 100, 100, C.byref(api.PolicyParams(**p)), C.byref(o), ws, ws_bytes, None)
    for kw in (dict(loss=None), dict(token=None), dict(adv=None), dict(mean=3), dict(mean=2), dict(mean=2, seq_start=P, seqs=-1), dict(clip_low=-0.1),
               dict(clip_high=float("nan")), dict(dual_clip=-1.0), dict(kl_coef=float("nan")), dict(ent_coef=float("nan")), dict(inv_t=0.0),
               dict(dx=P + 8), dict(dx=P + 100000, ld_dx=99)):
        assert call(**kw)[0] == 1, kw
    assert call(ws=None)[0] == 3 and call(ws_bytes=need - 400)[0] == 3
    assert status("whirl_policy_loss", P, 0, 4, 100, 100, None, None, P, need, None)[0] == 1


def test_preference_refusals():
    from whirl_llm_b200 import api
    need = api.lib.whirl_loss_workspace_bytes(4, 2)

    def call(ws=P, ws_bytes=need, loss=P, dx=None, **kw):
        p = dict(token=P, seq_start=P, pairs=2, kind=0, inv_t=1.0, beta=0.1)
        p.update(kw)
        o = api.PreferenceOut(loss=loss, dx=dx, ld_dx=100)
        return status("whirl_preference_loss", P, 0, 4, 100, 100, C.byref(api.PreferenceParams(**p)), C.byref(o), ws, ws_bytes, None)
    for kw in (dict(loss=None), dict(token=None), dict(seq_start=None), dict(pairs=-1), dict(kind=3), dict(beta=0.0), dict(beta=float("nan")),
               dict(smoothing=-0.1), dict(smoothing=1.1), dict(margin=float("nan")), dict(dx=P + 8)):
        assert call(**kw)[0] == 1, kw
    assert call(ws=None)[0] == 3 and call(ws_bytes=300)[0] == 3


def test_block_tables_refusals():
    from whirl_llm_b200 import api
    need = api.lib.whirl_block_workspace_bytes(4)

    def call(length=P, n_new=P, ws=P, ws_bytes=need, rows=None, **kw):
        t = dict(table=P, owned=P, free_ids=P, free_count=P, seqs=4, max_blocks=8, num_blocks=16, block_size=16)
        t.update(kw)
        o = dict(slot=P, row0=P, status=P, max_rows=32)
        o.update(rows or {})
        return status("whirl_block_tables_step", length, n_new, C.byref(api.BlockTables(**t)), C.byref(api.StepRowsOut(**o)), ws, ws_bytes, None)
    for kw in (dict(table=None), dict(owned=None), dict(free_ids=None), dict(free_count=None), dict(seqs=-1), dict(max_blocks=-1), dict(num_blocks=-1),
               dict(block_size=0), dict(length=None), dict(n_new=None), dict(rows=dict(slot=None)), dict(rows=dict(row0=None)),
               dict(rows=dict(status=None)), dict(rows=dict(max_rows=-1))):
        assert call(**kw)[0] == 1, kw
    assert call(seqs=api.MAX_SEQS + 1)[0] == 4
    assert call(ws=None)[0] == 3 and call(ws_bytes=100)[0] == 3


def test_binding_refuses_cpu_tensors_and_bad_shapes():
    from whirl_llm_b200 import api
    x = torch.zeros((2, 8))
    with pytest.raises(ValueError):
        api.token_logprobs(x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        api.block_tables_step(*[torch.zeros(1, dtype=torch.int32)] * 2, torch.zeros((1, 1), dtype=torch.int32), *[torch.zeros(1, dtype=torch.int32)] * 3,
                              block_size=16, max_rows=4)


def test_definitions_against_automatic_differentiation():
    g = torch.Generator().manual_seed(3)
    rows, n = 7, 23
    x = torch.randn((rows, n), generator=g, dtype=torch.float64).requires_grad_()
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    it = torch.full((rows,), 0.8, dtype=torch.float64)
    lp = torch.log_softmax(x * 0.8, 1)
    logp, h = lp.gather(1, token.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1)
    adv, old, rf = torch.randn(rows, generator=g).double(), logp.detach() + 0.1, logp.detach() - 0.2
    scale = ref.row_scale(torch.rand(rows, generator=g).double(), 2, [0, 3, 3, 7])
    row, _, gl = ref.policy(logp, h, scale, adv, old, rf, kl_coef=0.3, ent_coef=0.05)
    (dx,) = torch.autograd.grad((scale * row).sum(), x)
    m, s, _, e = ref.row_stats(x.detach(), it)
    want, _, _ = ref.dlogits(x.detach(), token, it, (m, s), (scale * gl).detach(), -0.05 * scale, e)
    np.testing.assert_allclose(want.numpy(), dx.numpy(), atol=1e-12)
    for kind in range(3):
        hh = torch.linspace(-3, 3, 11, dtype=torch.float64).requires_grad_()
        loss, dh = ref.pair_loss(hh, kind, 0.4, 0.2)
        (want,) = torch.autograd.grad(loss.sum(), hh)
        np.testing.assert_allclose(dh.detach().numpy(), want.numpy(), atol=1e-12)
