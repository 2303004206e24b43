"""The losses' rows that are unlike the others: outside every sequence, far from any reference, without a distribution, masked beside
such rows; against the 64-bit definitions (loss_ref.py)."""
import math

import pytest
import torch

import loss_ref as ref
from test_gpu_losses import DT, close, make, ones, policy_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("rows,n,pad,off,dtype", [(1, 50, 0, 0, "f32"), (17, 1003, 1, 0, "f32"), (40, 4096, 0, 0, "bf16"), (24, 33001, 0, 1, "f32"),
                                                  (9, 151936, 0, 0, "bf16"), (5, 262144, 64, 0, "f32"), (3, 1000003, 0, 0, "f32")])
def test_policy_rows_outside_the_sequences(rows, n, pad, off, dtype, grad):
    """The mean over sequences: rows of positive weight before the first sequence and behind the last have all their outputs, no share
    in the loss and a gradient of zero, whatever their logits are."""
    from whirl_llm_b200 import api
    x, x64, token, it, (m, s, logp, h), adv, old, rf, weight = policy_inputs(rows, n, dtype, seed=5, pad=pad, off=off, inv_t=1.25)
    first, mid, end = min(1, rows - 1), rows // 2, max(min(1, rows - 1), rows - 2)
    starts = [first, max(first, mid), max(first, mid), end]
    weight[0], weight[-1] = 1.0, 0.5
    kw = dict(clip_low=0.2, clip_high=0.28, dual_clip=1.5, kl_coef=0.1, ent_coef=0.02)
    st = torch.tensor(starts, dtype=torch.int32).cuda()
    call = lambda y: api.policy_loss(y, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), st, inv_t=1.25, mean=api.MEAN_SEQS,  # noqa: E731
                                     want_grad=grad, **kw)
    r = call(x)
    w = weight.double()
    live, inside = w > 0, torch.zeros(rows, dtype=torch.bool)
    inside[starts[0]: starts[-1]] = True
    scale = ref.row_scale(torch.where(inside, w, 0.0), 2, starts)
    row, kl, g = ref.policy(logp, h, scale, adv.double(), old.double(), rf.double(), **kw)
    on = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    le = ref.logp_tol(n, logp)
    # a row's loss moves with its log-probability (ratio up to 1.5, exp(k) - 1 up to 3) and its entropy
    rt = (g.abs() + 1.5 * adv.double().abs() + 0.3) * le * 1.1 + 0.02 * ref.entropy_tol(n) + 4 * ref.EPS32 * row.abs() + 1e-9
    close(r.logp, on(logp), le, "logp")
    close(r.entropy, on(h), ref.entropy_tol(n), "entropy")
    close(r.kl, on(kl), torch.expm1((rf.double() - logp).clamp(-20, 20)).abs() * le * 1.1 + 4 * ref.EPS32 * kl + 1e-9, "kl")
    close(r.row_loss, on(row), rt, "row_loss")
    close(r.row_scale, scale, 3 * ref.EPS32 * scale, "scale")
    close(r.loss, (scale * on(row)).sum(), (scale * (rt + 3 * ref.EPS32 * row.abs())).sum() + 1e-9, "loss")
    assert (r.g_logp.cpu()[~inside] == 0).all()
    assert not grad or (r.dx[~inside.cuda()] == 0).all()
    # outside the sequences a row without a distribution shows in its outputs and nowhere else
    y = x.clone()
    r = call(y)  # (the clone's rows lie closer together: sums in another order)
    y[0, 0] = math.nan
    q = call(y)
    if not inside[0]:
        assert math.isnan(q.logp[0].item()) and math.isnan(q.row_loss[0].item())
        assert torch.equal(q.loss, r.loss) and torch.equal(q.logp[1:], r.logp[1:])
        assert not grad or torch.equal(q.dx, r.dx)
