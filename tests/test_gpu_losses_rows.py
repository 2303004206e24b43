"""The losses' rows that are unlike the others: outside every sequence, far from any reference, without a distribution, masked beside
such rows; against the 64-bit definitions (loss_ref.py)."""
import math

import numpy as np
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


def far_rows(n, dtype):
    """Rows whose largest logit times inv_t is far from what a float's reference resolves, and their temperatures."""
    g = torch.Generator().manual_seed(n)
    fill = [-1e9, -3e9, -1e10, -1e30, 1e10, 30.0, 1e36]
    it = torch.tensor([1.0, 1.25, 1.0, 0.8, 1.0, 1e8, 10.0, 1.0, 1.25, 1.0, 1e9, 1.0, 1e-3], dtype=torch.float32)
    rows = len(it)
    x = torch.randn((rows, n), generator=g) * 3
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    for r, v in enumerate(fill):
        x[r] = v
    x[7, token[7]] = 1e10                     # one huge logit, on the token
    x[8, (token[8] + 1) % n] = 1e10           # ... and beside it
    x[9, ::2], x[9, 1::2] = -1e30, -2e30      # a masked row of two levels
    x[11, : n // 2] = -1e30                   # an ordinary row, half of it masked
    x[12] = 1e12 + 4e11 * x[12]               # a wide row at a temperature that leaves it ordinary differences
    x = x.to(DT[dtype])
    return x, x.double(), token, it


def check_dx(dx, x64, token, it, stats, g, dtype, n, what):
    d, p, lp = ref.dlogits(x64, token, it.double(), stats, g)
    close(dx, d, ref.dx_tol(p, lp.clamp_min(-1e30), g, it.double(), DT[dtype], d, n=n), what)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [64, 1003, 20001, 60000, 1000003])
def test_far_rows_in_every_gradient(n, dtype):
    """Rows filled with masks of -1e9 to -1e30, huge logits, temperatures near zero: the same statistics and the same gradient in every
    path (given statistics, the policy loss, the preference loss; n = 1000003 f32: the policy loss in two launches)."""
    from whirl_llm_b200 import api
    x, x64, token, it = far_rows(n, dtype)
    rows = len(it)
    xd, tok, itd = x.cuda(), token.cuda(), it.cuda()
    m, s, lp, h = ref.row_stats(x64, it.double())
    want = lp.gather(1, token.long()[:, None])[:, 0]
    tol = ref.logp_tol(n, want)
    r = api.token_logprobs(xd, tok, inv_t_rows=itd, want_entropy=True)
    close(r.logp, want, tol, "logp")
    close(r.entropy, h, ref.entropy_tol(n), "entropy")
    assert torch.equal(r.stats[:, 0].double().cpu(), m)
    close(r.stats[:, 1], s, s * ref.sum_error(n), "sum")
    g = torch.linspace(-1, 1.1, rows)
    dx = api.token_logprobs_grad(xd, tok, r.stats, g.cuda(), inv_t_rows=itd)
    stats = (r.stats[:, 0].double().cpu(), r.stats[:, 1].double().cpu())
    check_dx(dx, x64, token, it, stats, g.double(), dtype, n, "dx of given statistics")
    adv = g.cuda()
    for kw in (dict(), dict(ent_coef=0.01)):
        q = api.policy_loss(xd, tok, adv, inv_t_rows=itd, mean=api.MEAN_SUM, **kw)
        close(q.logp, want, tol, "logp of the policy loss")
        close(q.g_logp, -g.double(), ref.EPS32 * g.double().abs(), "g_logp")
        if not kw:
            check_dx(q.dx, x64, token, it, (m, s), -g.double(), dtype, n, "dx of the policy loss")
        else:
            hh = torch.full((rows,), -0.01).double()
            d, p, lpd = ref.dlogits(x64, token, it.double(), (m, s), -g.double(), hh, h)
            close(q.dx, d, ref.dx_tol(p, lpd.clamp_min(-1e30), g.double(), it.double(), DT[dtype], d, hh, h, n), "dx with entropy")
    starts = torch.tensor([0, 4, 7, 9, rows], dtype=torch.int32, device="cuda")
    # (the rows' own log-probabilities as reference: the pairs' losses stay ordinary)
    f = api.preference_loss(xd, tok, starts, r.logp, inv_t_rows=itd, beta=0.5)
    close(f.logp, want, tol, "logp of the preference loss")
    assert (f.g_logp[:7].abs() > 1e-3).all()  # (a float of -1e10 is off by hundreds: the other pair is decided)
    check_dx(f.dx, x64, token, it, (m, s), f.g_logp.double().cpu(), dtype, n, "dx of the preference loss")


@pytest.mark.parametrize("dtype,n", [("f32", 2500), ("bf16", 4200), ("f32", 20011)])
@pytest.mark.parametrize("place", ["apart", "in place", "misaligned"])
def test_policy_many_rows_of_every_kind(dtype, n, place):
    """Clusters that take many rows: every third far (lowest value, the type's maximum, masks), rows without a distribution, masked ones
    and ordinary ones in turn, each against the definition."""
    from whirl_llm_b200 import api
    rows = 2000 if n < 10000 else 700
    g = torch.Generator().manual_seed(n)
    x = (torch.randn((rows, n), generator=g) * 3).to(DT[dtype])
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    weight = torch.ones(rows)
    k = torch.arange(rows)
    lim = torch.finfo(DT[dtype])
    x[k % 9 == 0] = lim.min
    x[(k % 9 == 3).nonzero()[:, 0], token[k % 9 == 3].long()] = lim.max
    x[k % 9 == 6] = -1e30
    x[(k % 5 == 1) & (k % 3 != 0), 7] = math.nan
    weight[k % 4 == 2] = 0.0
    x64, it = x.double(), ones(1.25, rows)
    m, s, lp, h = ref.row_stats(x64, it)
    logp = lp.gather(1, token.long()[:, None])[:, 0].float().double()  # (as float32: -4e38 is -inf there)
    adv = torch.randn(rows, generator=g)
    xd = x.cuda()
    out = {"apart": None, "in place": xd, "misaligned": torch.zeros((rows, n + 1), dtype=DT[dtype], device="cuda")[:, 1:]}[place]
    r = api.policy_loss(xd, token.cuda(), adv.cuda(), weight=weight.cuda(), inv_t=1.25, mean=api.MEAN_SUM, dx=out)
    live = weight > 0
    want = torch.where(live, logp, 0.0)
    close(r.logp, want, ref.logp_tol(n, want.clamp_min(-1e30)), "logp")
    gl = torch.where(live, torch.where(torch.isnan(logp), torch.nan, -adv.double()), 0.0)
    close(r.g_logp, gl, 1e-30, "g_logp")
    good = ~(torch.isnan(logp) & live)
    d, p, lpd = ref.dlogits(x64[good], torch.where(live, token, -1)[good], it[good], (m[good], s[good]), gl[good])
    close(r.dx[good.cuda()], d, ref.dx_tol(p, lpd.clamp_min(-1e30), gl[good], it[good], DT[dtype], d, n=n), "dx")
    assert torch.isnan(r.dx[~good.cuda()]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1003, 20001, 60000])
def test_masked_rows_of_a_pair_without_a_finite_factor(n, dtype):
    """A pair whose loss is NaN (a row without a distribution) or infinite (squared loss, a forbidden token): its rows that do not count
    get zeros, and so do the rows outside the pairs."""
    from whirl_llm_b200 import api
    x, _, token = make(10, n, dtype, seed=6)
    x = x.clone()
    starts = torch.tensor([0, 3, 5, 7, 9], dtype=torch.int32, device="cuda")
    weight = torch.tensor([1.0, 0, 1, 0, 1, 1, 0, 1, 0, 1], device="cuda")
    dead = weight == 0
    dead[9] = True
    x[2, 5] = math.nan
    r = api.preference_loss(x, token.cuda(), starts, weight=weight)
    assert math.isnan(r.pair_loss[0].item()) and math.isfinite(r.pair_loss[1].item())
    assert (r.g_logp[dead] == 0).all() and (r.dx[dead] == 0).all() and (r.logp[dead] == 0).all()
    assert torch.isnan(r.g_logp[[0, 2, 4]]).all() and torch.isnan(r.dx[[0, 2, 4]]).all()
    assert torch.isfinite(r.dx[[5, 7]]).all() and (r.dx[[5, 7]] != 0).any()
    x[2, 5] = 0.0
    x[2, token[2]] = -math.inf
    r = api.preference_loss(x, token.cuda(), starts, weight=weight, kind=api.PREF_SQUARED)
    assert r.pair_loss[0].item() == math.inf and math.isfinite(r.pair_loss[1].item())
    assert (r.g_logp[dead] == 0).all() and (r.dx[dead] == 0).all() and (r.logp[dead] == 0).all()


@pytest.mark.parametrize("n", [1003, 20001, 60000])
@pytest.mark.parametrize("shift", [1e4, 1e5, -1e5, 1e6, -1e6])
def test_gradient_of_logits_with_an_offset(n, shift):
    """bf16 logits that all lie far from zero (by less than far rows): probabilities from differences of a few steps."""
    from whirl_llm_b200 import api
    rows = 6
    g = torch.Generator().manual_seed(n + int(shift))
    x = (shift + abs(shift) * torch.randint(-3, 3, (rows, n), generator=g) / 256).to(torch.bfloat16)
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    it = torch.full((rows,), 300.0 / abs(shift))   # a step (shift / 256 or / 128) is worth one or two units
    it[3:] = 1.25
    x64 = x.double()
    m, s, lp, h = ref.row_stats(x64, it.double())
    xd, tok, itd = x.cuda(), token.cuda(), it.cuda()
    r = api.token_logprobs(xd, tok, inv_t_rows=itd, want_entropy=True)
    want = lp.gather(1, token.long()[:, None])[:, 0]
    close(r.logp, want, ref.logp_tol(n, want), "logp")
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    stats, e64 = (r.stats[:, 0].double().cpu(), r.stats[:, 1].double().cpu()), r.entropy.double().cpu()
    for use_h in (False, True):
        dx = api.token_logprobs_grad(xd, tok, r.stats, gl.cuda(), inv_t_rows=itd, entropy=r.entropy if use_h else None, g_entropy=gh.cuda() if use_h else None)
        d, p, lpd = ref.dlogits(x64, token, it.double(), stats, gl.double(), gh.double() if use_h else None, e64)
        close(dx, d, ref.dx_tol(p, lpd, gl.double(), it.double(), torch.bfloat16, d, gh.double() if use_h else None, e64, n), "dx")
    q = api.policy_loss(xd, tok, gl.cuda(), inv_t_rows=itd, mean=api.MEAN_SUM, ent_coef=0.5)
    hh = torch.full((rows,), -0.5).double()
    d, p, lpd = ref.dlogits(x64, token, it.double(), (m, s), -gl.double(), hh, h)
    close(q.dx, d, ref.dx_tol(p, lpd, gl.double(), it.double(), torch.bfloat16, d, hh, h, n), "dx of the policy loss")


@pytest.mark.parametrize("n", [1003, 20001])
@pytest.mark.parametrize("inv_t", [1e-36, 3e-34, 1e-30])
def test_smallest_inv_t(n, inv_t):
    """Logits of up to 1e38 at an inverse temperature near the smallest normal number."""
    from whirl_llm_b200 import api
    g = torch.Generator().manual_seed(n)
    rows = 5
    it = torch.full((rows,), inv_t)
    x = torch.randn((rows, n), generator=g) * float(3 / it[0])
    x[1, ::3] = -math.inf
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    m, s, lp, h = ref.row_stats(x.double(), it.double())
    want = lp.gather(1, token.long()[:, None])[:, 0]
    r = api.token_logprobs(x.cuda(), token.cuda(), inv_t=it[0].item(), want_entropy=True)
    close(r.logp, want, ref.logp_tol(n, want), "logp")
    close(r.stats[:, 1], s, s * ref.sum_error(n), "sum")
    close(r.entropy, h, ref.entropy_tol(n), "entropy")
    gl = torch.full((rows,), 1e36)
    dx = api.token_logprobs_grad(x.cuda(), token.cuda(), r.stats, gl.cuda(), inv_t=it[0].item())
    d, p, lpd = ref.dlogits(x.double(), token, it.double(), (r.stats[:, 0].double().cpu(), r.stats[:, 1].double().cpu()), gl.double())
    close(dx, d, ref.dx_tol(p, lpd, gl.double(), it.double(), torch.float32, d, n=n), "dx")


@pytest.mark.parametrize("rows,n,dtype,inv_t", [(4000, 1003, "f32", 1.0), (4000, 1003, "bf16", 1.25), (3000, 9000, "f32", 1.0), (4000, 20001, "bf16", 1.0), (2000, 60000, "f32", 0.8)])
def test_errors_of_many_rows_do_not_add_up(rows, n, dtype, inv_t):
    """The log-probability of a long sequence: a row's errors are roundings that fall either way (its sum's float, some ten partial sums
    and the largest terms: less than one half step of a float in the mean square) and what is left of the mean error of the
    hardware's exponential (less than 1e-8, see the kernels)."""
    from whirl_llm_b200 import api
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.randn((rows, n), generator=g, device="cuda") * 3).to(DT[dtype])
    token = torch.randint(0, n, (rows,), generator=g, device="cuda")
    x.scatter_(1, token[:, None], (math.log(n) + 2 + 3 * torch.randn(rows, generator=g, device="cuda")).to(x.dtype)[:, None])
    z = torch.cat([torch.log_softmax(v.double() * float(np.float32(inv_t)), 1).gather(1, t[:, None])[:, 0] for v, t in zip(x.split(500), token.split(500))])
    starts = torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda")
    r = api.preference_loss(x, token.int(), starts, ref_logp=z.float(), inv_t=inv_t, beta=1.0)   # what is left is small: no rounding of its own
    want = (z - z.float().double()).sum()
    assert abs(r.reward[0, 0].double() - want) < 1e-8 * rows + 6 * ref.EPS32 * math.sqrt(rows), ((r.reward[0, 0].double() - want) / rows).item()


@pytest.mark.parametrize("n", [1003, 20001, 1000003])
def test_policy_inputs_that_are_nan(n):
    """An advantage, an old or a reference log-probability that is NaN: the row's loss and gradient are NaN, nobody else's."""
    from whirl_llm_b200 import api
    x, _, token, _, (_, _, logp, _), adv, old, rf, _ = policy_inputs(6, n, "f32", seed=8, masked=0.0)
    want = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), mean=api.MEAN_SUM, kl_coef=0.1, dual_clip=2.0)
    adv, old, rf = adv.clone(), old.clone(), rf.clone()
    adv[1], old[2], rf[4] = math.nan, math.nan, math.nan
    r = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), mean=api.MEAN_SUM, kl_coef=0.1, dual_clip=2.0)
    bad = torch.tensor([1, 2, 4])
    good = torch.tensor([0, 3, 5])
    assert torch.isnan(r.row_loss[bad]).all() and torch.isnan(r.g_logp[bad]).all() and torch.isnan(r.dx[bad]).all() and torch.isnan(r.loss)
    assert torch.equal(r.row_loss[good], want.row_loss[good]) and torch.equal(r.dx[good], want.dx[good]) and torch.equal(r.logp, want.logp)


@pytest.mark.parametrize("n", [1003, 20001, 60000])
def test_largest_inv_t(n):
    """Temperatures of next to nothing: the maxima share the row, wherever they lie."""
    from whirl_llm_b200 import api
    x = -1.0 - torch.rand((4, n))
    x[:, 5], x[:, n - 2], x[:, 700] = 0.0, 0.0, 0.0
    x[1] += 5.0
    x[2] -= 3.0
    x[3, ::2] = -math.inf
    x[3, 5] = x[3, n - 2] = x[3, 700] = 0.0
    token = torch.tensor([5, 700, 5, n - 2], dtype=torch.int32)
    for inv_t in (3.3e38, 2e38, 1e30):
        it = ones(inv_t, 4)
        m, s, lp, h = ref.row_stats(x.double(), it)
        r = api.token_logprobs(x.cuda(), token.cuda(), inv_t=inv_t, want_entropy=True)
        assert torch.allclose(r.logp.cpu(), torch.full((4,), -math.log(3.0)), atol=1e-6) and (r.stats[:, 1] == 3).all()
        close(r.entropy, h, ref.entropy_tol(n), "entropy")
        g = torch.ones(4) / np.float32(inv_t)
        p = api.policy_loss(x.cuda(), token.cuda(), -g.cuda(), inv_t=inv_t, mean=api.MEAN_SUM)
        for dx in (api.token_logprobs_grad(x.cuda(), token.cuda(), r.stats, g.cuda(), inv_t=inv_t), p.dx):
            want = torch.zeros((4, n))
            want[:, [5, 700, n - 2]] = -1 / 3
            want[torch.arange(4), token.long()] = 2 / 3
            assert torch.allclose(dx.cpu(), want, atol=1e-6)
