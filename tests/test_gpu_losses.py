"""Token log-probabilities, the policy and preference losses and their gradients against the 64-bit definitions (loss_ref.py),
through the public binding."""
import math
import threading

import numpy as np
import pytest
import torch

import loss_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(rows, n, dtype, pad=0, off=0, seed=0, sd=3.0):
    """Logits [rows, n] on the GPU inside rows of n + pad + off elements, their first `off` elements skipped; token ids."""
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + n)
    x = (torch.randn((rows, n), generator=g) * sd).to(DT[dtype])
    buf = torch.full((rows, n + pad + off), 7.0, dtype=DT[dtype], device="cuda")
    buf[:, off: off + n] = x.cuda()
    token = torch.randint(0, n, (rows,), generator=g, dtype=torch.int32)
    return buf[:, off: off + n], x.double(), token


def ones(v, rows):
    return torch.full((rows,), float(np.float32(v)), dtype=torch.float64)


def close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN")
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), (what, "infinities")
    tol = tol if torch.is_tensor(tol) else torch.full_like(want, tol)
    bad = ((got - want).abs() > tol) & fine
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


SHAPES = [(1, 1, 0, 0), (3, 2, 0, 0), (2, 7, 0, 0), (4, 8, 0, 0), (3, 9, 1, 0), (5, 127, 0, 0), (3, 1000, 0, 1), (2, 4097, 0, 0), (3, 4096, 8, 3),
          (2, 33001, 3, 0), (1, 131072, 0, 0), (9, 20000, 0, 0), (2, 151936, 0, 0), (1, 300001, 0, 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,pad,off", SHAPES)
@pytest.mark.parametrize("inv_t", [1.0, 1.25])
def test_logprobs_and_gradient(rows, n, pad, off, dtype, inv_t):
    from whirl_llm_b200 import api
    x, x64, token = make(rows, n, dtype, pad, off)
    it = ones(inv_t, rows)
    m, s, lp, h = ref.row_stats(x64, it)
    r = api.token_logprobs(x, token.cuda(), inv_t=inv_t, want_entropy=True)
    want = lp.gather(1, token.long()[:, None])[:, 0]
    close(r.logp, want, ref.logp_tol(n, want), "logp")
    assert torch.equal(r.stats[:, 0].double().cpu(), m)
    close(r.stats[:, 1], s, s * ref.sum_error(n), "sum")
    close(r.entropy, h, ref.entropy_tol(n), "entropy")
    plain = api.token_logprobs(x, token.cuda(), inv_t=inv_t)
    assert plain.entropy is None
    close(plain.logp, want, ref.logp_tol(n, want), "logp without entropy")

    g = torch.randn(rows, generator=torch.Generator().manual_seed(1)).float()
    ge = torch.randn(rows, generator=torch.Generator().manual_seed(2)).float()
    stats64 = (r.stats[:, 0].double().cpu(), r.stats[:, 1].double().cpu())
    for use_h in (False, True):
        dx = api.token_logprobs_grad(x, token.cuda(), r.stats, g.cuda(), inv_t=inv_t, entropy=r.entropy if use_h else None,
                                     g_entropy=ge.cuda() if use_h else None)
        e64 = r.entropy.double().cpu()
        d, p, lpd = ref.dlogits(x64, token, it, stats64, g.double(), ge.double() if use_h else None, e64)
        close(dx, d, ref.dx_tol(p, lpd, g.double(), it, x.dtype, d, ge.double() if use_h else None, e64, n), "dx")
        assert dx.shape == x.shape and dx.dtype == x.dtype
    # a dense dx beside padded rows (another alignment), and dx = x
    out = torch.full((rows, n), 9.0, dtype=x.dtype, device="cuda")
    api.token_logprobs_grad(x, token.cuda(), r.stats, g.cuda(), inv_t=inv_t, dx=out)
    again = api.token_logprobs_grad(x, token.cuda(), r.stats, g.cuda(), inv_t=inv_t)
    assert torch.equal(out, again)
    x2 = x.clone()
    assert api.token_logprobs_grad(x2, token.cuda(), r.stats, g.cuda(), inv_t=inv_t, dx=x2) is x2
    assert torch.equal(x2, again)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_every_kind(dtype):
    """Forbidden tokens at -inf and at the type's lowest value, rows without a distribution, rows that do not count."""
    from whirl_llm_b200 import api
    rows, n = 12, 1500
    x, x64, token = make(rows, n, dtype, seed=3)
    low = torch.finfo(DT[dtype]).min
    g = torch.Generator().manual_seed(5)
    x = x.clone()
    hide = torch.rand((rows, n), generator=g) < 0.5
    hide[torch.arange(rows), token.long()] = False
    x[0][hide[0].cuda()] = -math.inf
    x[1][hide[1].cuda()] = low
    x[2] = low                      # a row of the lowest value alone: uniform
    x[3] = -math.inf                # nothing left
    x[4, 700] = math.nan
    x[5, 1499] = math.inf
    x[6] = -math.inf
    x[6, token[6].item()] = 2.5     # one token left
    x[7, token[7].item()] = -math.inf  # the token itself is forbidden
    x[8] = 0.0                      # all alike
    x[9, 3] = torch.finfo(DT[dtype]).max
    token[10] = -1
    token[11] = n
    x[10:] = math.nan               # rows that do not count are not looked at
    x64 = x.double().cpu()
    it = ones(0.8, rows)
    m, s, lp, h = ref.row_stats(x64, it)
    r = api.token_logprobs(x, token.cuda(), inv_t=0.8, want_entropy=True)
    want = lp.gather(1, token.clamp(0, n - 1).long()[:, None])[:, 0]
    for v in (want, h, m, s):
        v[10:] = 0.0
    m = torch.where(torch.isnan(x64).any(1) & (torch.arange(rows) < 10), torch.nan, m)  # (which number stands there is not promised)
    close(r.logp, want, ref.logp_tol(n, want), "logp")
    close(r.entropy, h, ref.entropy_tol(n), "entropy")
    keep = ~torch.isnan(m)
    assert torch.equal(r.stats[:, 0].double().cpu()[keep], m[keep])
    close(r.stats[:, 1], s, s.nan_to_num() * ref.sum_error(n), "sum")
    gl, ge = torch.randn(rows, generator=g).float(), torch.randn(rows, generator=g).float()
    e64 = r.entropy.double().cpu()
    dx = api.token_logprobs_grad(x, token.cuda(), r.stats, gl.cuda(), inv_t=0.8, entropy=r.entropy, g_entropy=ge.cuda())
    d, p, lpd = ref.dlogits(x64, token, it, (r.stats[:, 0].double().cpu(), r.stats[:, 1].double().cpu()), gl.double(), ge.double(), e64)
    d[[3, 4, 5]] = math.nan
    d[10:] = 0.0
    good = torch.ones(rows, dtype=torch.bool)
    good[[3, 4, 5]] = False
    close(dx[good.cuda()], d[good], ref.dx_tol(p[good], lpd[good], gl.double()[good], it[good], x.dtype, d[good], ge.double()[good], e64[good], n), "dx")
    assert torch.isnan(dx[3:6]).all()
    gl[4] = 0.0
    dx = api.token_logprobs_grad(x, token.cuda(), r.stats, gl.cuda(), inv_t=0.8)
    assert (dx[4] == 0).all() and (dx[10:] == 0).all()


def test_inv_t_per_row_and_sampler_stats():
    """Per-row temperatures, and the statistics of the sampler as the backward pass's."""
    from whirl_llm_b200 import api
    rows, n = 6, 32768
    x, x64, token = make(rows, n, "f32", seed=4)
    it = torch.tensor([0.5, 1.0, 1.25, 2.0, 0.9, 1.0], dtype=torch.float32)
    r = api.token_logprobs(x, token.cuda(), inv_t_rows=it.cuda())
    m, s, lp, _ = ref.row_stats(x64, it.double())
    want = lp.gather(1, token.long()[:, None])[:, 0]
    close(r.logp, want, ref.logp_tol(n, want))
    sampled = api.sample_rows(x.contiguous(), api.RowParams(inv_t=it.cuda(), u=torch.rand(rows, dtype=torch.float64, device="cuda")))
    g = torch.randn(rows, device="cuda")
    a = api.token_logprobs_grad(x, sampled.token, sampled.stats, g, inv_t_rows=it.cuda())
    d, p, lpd = ref.dlogits(x64, sampled.token.cpu(), it.double(), (m, s), g.double().cpu())
    # (the sampler's own sum may be off by 1e-5, which is what its tests allow)
    close(a, d, ref.dx_tol(p, lpd, g.double().cpu(), it.double(), x.dtype, d, n=n) + 1e-5 * p * g.double().cpu().abs()[:, None] * it.double()[:, None])


def policy_inputs(rows, n, dtype, seed, pad=0, off=0, masked=0.3, inv_t=1.0):
    x, x64, token = make(rows, n, dtype, pad, off, seed)
    g = torch.Generator().manual_seed(seed + 100)
    it = ones(inv_t, rows)
    m, s, lp, h = ref.row_stats(x64, it)
    logp = lp.gather(1, token.long()[:, None])[:, 0]
    adv = torch.randn(rows, generator=g)
    d = 0.3 * torch.randn(rows, generator=g, dtype=torch.float64)
    for edge in (math.log(0.8), math.log(1.2), math.log(1.28), math.log(1.5)):  # (a last bit would decide which side is clipped)
        d = torch.where((d - edge).abs() < 1e-3, d + 2e-3, d)
    old = (logp - d).float()
    rf = (logp + 0.4 * torch.randn(rows, generator=g)).float()
    weight = torch.where(torch.rand(rows, generator=g) < masked, 0.0, 0.25 + torch.rand(rows, generator=g))
    return x, x64, token, it, (m, s, logp, h), adv, old, rf, weight


def check_policy(r, x64, token, it, stats, adv, old, rf, weight, mean, starts, dtype, n, **kw):
    m, s, logp, h = stats
    rows = len(adv)
    w = weight.double() if weight is not None else torch.ones(rows, dtype=torch.float64)
    w = torch.where((token >= 0) & (token < n), w, 0.0)
    if mean == 2:
        inside = torch.zeros(rows, dtype=torch.bool)
        inside[starts[0]: starts[-1]] = True
        w = torch.where(inside, w, 0.0)
    scale = ref.row_scale(w, mean, starts)
    live = w > 0
    row, kl, g = ref.policy(logp, h, scale, adv.double(), None if old is None else old.double(), None if rf is None else rf.double(), **kw)
    zero = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    kl_coef, ent_coef = kw.get("kl_coef", 0.0), kw.get("ent_coef", 0.0)
    le = ref.logp_tol(n, logp)
    # ratios move with logp: d row / d logp times its error, the kl's second derivative included
    slope = g.abs() + adv.double().abs() * 1.5 + kl_coef * 3
    kt = (torch.expm1((rf.double() - logp).clamp(-20, 20)).abs() * le * 1.1 if rf is not None else 0.0) + 4 * ref.EPS32 * kl + 1e-9
    rt = slope * le * 1.1 + abs(ent_coef) * ref.entropy_tol(n) + 4 * ref.EPS32 * row.abs() + 1e-9
    close(r.logp, zero(logp), le, "logp")
    close(r.row_loss, zero(row), rt, "row_loss")
    if rf is not None:
        close(r.kl, zero(kl), kt, "kl")
    close(r.row_scale, torch.where(live, scale, 0.0), 3 * ref.EPS32 * scale, "scale")
    close(r.loss, (scale * zero(row)).sum(), (scale * (rt + 3 * ref.EPS32 * zero(row).abs())).sum() + 1e-9, "loss")
    gt = scale * (adv.double().abs() * 2 + kl_coef * 4) * le * 1.2 + 5 * ref.EPS32 * (scale * g).abs() + 1e-12
    close(r.g_logp, zero(scale * g), gt, "g_logp")
    if r.dx is not None:
        hh = torch.where(live, -ent_coef * scale, 0.0) if ent_coef else None
        tok = torch.where(live, token, -1)
        d, p, lpd = ref.dlogits(x64, tok, it, (m, s), zero(scale * g), hh, h)
        tol = ref.dx_tol(p, lpd, zero(scale * g), it, DT[dtype], d, hh, h, n) + (gt * it)[:, None] * (p + 0.0) * 1.1
        tol[torch.arange(rows), token.clamp(0, n - 1).long()] += gt * it
        close(r.dx, d, tol, "dx")
        assert (r.dx[~live.cuda()] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("mean", [0, 1, 2])
@pytest.mark.parametrize("rows,n,pad,off", [(1, 50, 0, 0), (17, 1003, 1, 0), (40, 4096, 0, 0), (24, 33001, 0, 1), (9, 151936, 0, 0), (5, 262144, 64, 0)])
def test_policy(rows, n, pad, off, mean, dtype):
    from whirl_llm_b200 import api
    x, x64, token, it, stats, adv, old, rf, weight = policy_inputs(rows, n, dtype, seed=mean + 1, pad=pad, off=off, inv_t=1.25)
    starts = sorted(np.random.default_rng(rows).integers(0, rows + 1, 5).tolist())
    starts[2] = starts[1]  # an empty sequence
    kw = dict(clip_low=0.2, clip_high=0.28, dual_clip=1.5, kl_coef=0.1, ent_coef=0.02)
    st = torch.tensor(starts, dtype=torch.int32).cuda()
    call = lambda **k: api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), st, inv_t=1.25, mean=mean, **{**kw, **k})  # noqa: E731
    r = call()
    check_policy(r, x64, token, it, stats, adv, old, rf, weight, mean, starts, dtype, n, **kw)
    again = call()
    for k in ("loss", "logp", "stats", "entropy", "kl", "row_loss", "g_logp", "row_scale", "dx"):
        assert torch.equal(getattr(r, k), getattr(again, k))  # the same bits
    f = call(want_grad=False)
    assert f.dx is None  # (another kernel: its sums run in another order)
    check_policy(f, x64, token, it, stats, adv, old, rf, weight, mean, starts, dtype, n, **kw)
    # no entropy, no KL, no weights, on-policy
    kw2 = dict(clip_low=0.2, clip_high=0.2)
    r = api.policy_loss(x, token.cuda(), adv.cuda(), seq_start=st, inv_t=1.25, mean=mean, **kw2)
    assert r.entropy is None and r.kl is None
    check_policy(r, x64, token, it, stats, adv, None, None, None, mean, starts, dtype, n, **kw2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_policy_rows_that_do_not_count(dtype):
    """Weights of zero, below zero and NaN, tokens outside the vocabulary: nothing of the row is read; a batch without a live row."""
    from whirl_llm_b200 import api
    rows, n = 10, 2000
    x, x64, token, it, stats, adv, old, rf, weight = policy_inputs(rows, n, dtype, seed=9, masked=0.0)
    x = x.clone()
    weight[2], weight[3], weight[4] = 0.0, -1.0, math.nan
    token[5] = -100
    for k in (2, 3, 4, 5):
        x[k], adv[k], old[k], rf[k] = math.nan, math.nan, math.nan, math.nan
    r = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), kl_coef=0.1)
    w = weight.nan_to_num(0).clamp_min(0)
    check_policy(r, x64, token, it, stats, adv.nan_to_num(0), old.nan_to_num(0), rf.nan_to_num(0), w, 1, None, dtype, n, kl_coef=0.1)
    for v in (r.logp, r.kl, r.row_loss, r.g_logp, r.row_scale, r.dx.float().abs().amax(1), r.stats.abs().amax(1)):
        assert (v[2:6] == 0).all()
    r = api.policy_loss(x, token.cuda(), adv.cuda(), weight=torch.zeros(rows, device="cuda"))
    assert r.loss.item() == 0 and (r.dx == 0).all()
    r = api.policy_loss(x[:0], token[:0].cuda(), adv[:0].cuda())
    assert r.loss.item() == 0 and r.dx.shape == (0, n)


def test_policy_far_off_policy():
    """Ratios past the clamp: finite values, no gradient through it."""
    from whirl_llm_b200 import api
    rows, n = 6, 64
    x, x64, token, it, stats, adv, old, rf, _ = policy_inputs(rows, n, "f32", seed=11)
    old = (stats[2] + torch.tensor([60.0, -60.0, 0.01, 30.0, -30.0, -1e30])).float()
    rf = (stats[2] + torch.tensor([100.0, -100.0, 0.5, -0.5, 25.0, 1e30])).float()
    adv = torch.tensor([1.0, -1.0, 2.0, -2.0, 1.0, 0.0])
    r = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), mean=0, kl_coef=1e-9)
    row, kl, g = ref.policy(stats[2], stats[3], None, adv.double(), old.double(), rf.double(), kl_coef=1e-9)
    close(r.row_loss, row, 1e-4 * row.abs() + 1e-5)
    close(r.kl, kl, 1e-4 * kl + 1e-5)
    close(r.g_logp, g, 1e-4 * g.abs() + 1e-6)
    assert torch.isfinite(r.dx).all()


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("dtype,n,pad", [("f32", 1003, 0), ("bf16", 4096, 0), ("f32", 50, 3), ("bf16", 151936, 0)])
def test_preference(dtype, n, pad, kind, average):
    from whirl_llm_b200 import api
    rows, pairs = 61, 5
    x, x64, token, it, stats, _, _, rf, weight = policy_inputs(rows, n, dtype, seed=20 + kind, pad=pad)
    cuts = np.sort(np.random.default_rng(n + kind).integers(1, rows - 3, 2 * pairs + 1))
    cuts[4] = cuts[3]                          # an empty sequence
    starts = torch.tensor(cuts, dtype=torch.int32)
    weight[cuts[6]: cuts[7]] = 0.0             # one whose rows are all masked
    kw = dict(beta=0.3, kind=kind, smoothing=0.1 if kind == 0 else 0.0, margin=0.2, average=average)
    r = api.preference_loss(x, token.cuda(), starts.cuda(), rf.cuda(), weight.cuda(), **kw)
    w = weight.double().clone()
    w[: cuts[0]] = 0
    w[cuts[-1]:] = 0
    live = w > 0
    logp = torch.where(live, stats[2], 0.0)
    le = ref.logp_tol(n, logp)
    ratio = torch.where(live, logp - rf.double(), 0.0)
    P, W, pt = [], [], []
    for a, b in zip(cuts, cuts[1:]):
        t = w[a:b].sum()
        k = (1.0 / t if t > 0 else 0.0) if average else 1.0
        P.append((w[a:b] * ratio[a:b]).sum() * k), W.append(torch.as_tensor(k, dtype=torch.float64)), pt.append((w[a:b] * le[a:b]).sum() * k)
    P, W, pt = torch.stack(P), torch.stack(W), torch.stack(pt)
    h = kw["beta"] * (P[0::2] - P[1::2]) - kw["margin"]
    ht = kw["beta"] * (pt[0::2] + pt[1::2]) + 1e-9
    loss, dh = ref.pair_loss(h, kind, kw["beta"], kw["smoothing"])
    close(r.logp, logp, le, "logp")
    close(r.reward, (kw["beta"] * P).view(-1, 2), (kw["beta"] * pt).view(-1, 2) + 3 * ref.EPS32 * (kw["beta"] * P).view(-1, 2).abs() + 1e-9, "reward")
    lt = (dh.abs() + 1) * ht * (1 if kind < 2 else 2 / kw["beta"] ** 2 * (1 + ht)) + 3 * ref.EPS32 * loss + 1e-9
    close(r.pair_loss, loss, lt, "pair_loss")
    close(r.loss, loss.mean(), lt.mean() + 2 * ref.EPS32 * loss.mean(), "loss")
    coef = torch.stack([dh, -dh], 1).view(-1) * kw["beta"] * W / pairs
    curve = 0.25 if kind == 0 else (0.0 if kind == 1 else 2 / kw["beta"] ** 2)
    ct = torch.stack([ht, ht], 1).view(-1) * curve * kw["beta"] * W / pairs
    g, gt = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    for s, (a, b) in enumerate(zip(cuts, cuts[1:])):
        g[a:b], gt[a:b] = w[a:b] * coef[s], w[a:b] * ct[s]
    gt = gt * 1.1 + 5 * ref.EPS32 * g.abs() + 1e-12
    close(r.g_logp, g, gt, "g_logp")
    d, p, lpd = ref.dlogits(x64, torch.where(live, token, -1), it, (stats[0], stats[1]), g)
    tol = ref.dx_tol(p, lpd, g, it, DT[dtype], d, n=n) + gt[:, None] * p * 1.1
    tol[torch.arange(rows), token.long()] += gt
    close(r.dx, d, tol, "dx")
    again = api.preference_loss(x, token.cuda(), starts.cuda(), rf.cuda(), weight.cuda(), **kw)
    for k in ("loss", "pair_loss", "reward", "logp", "stats", "g_logp", "dx"):
        assert torch.equal(getattr(r, k), getattr(again, k))
    f = api.preference_loss(x, token.cuda(), starts.cuda(), rf.cuda(), weight.cuda(), want_grad=False, **kw)
    assert f.dx is None
    close(f.loss, loss.mean(), lt.mean() + 2 * ref.EPS32 * loss.mean(), "loss without gradient")
    close(f.g_logp, g, gt, "g_logp without gradient")


def test_preference_edges():
    from whirl_llm_b200 import api
    x, x64, token = make(4, 100, "f32")
    st = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    r = api.preference_loss(x, token.cuda(), st(0))                      # no pairs
    assert r.loss.item() == 0 and (r.dx == 0).all() and (r.logp == 0).all()
    r = api.preference_loss(x, token.cuda(), st(2, 2, 2))                # a pair without a row: h = 0
    assert abs(r.loss.item() - math.log(2)) < 1e-6 and (r.dx == 0).all()
    r = api.preference_loss(x[:0], token[:0].cuda(), st(0, 0, 0))
    assert abs(r.loss.item() - math.log(2)) < 1e-6 and r.dx.shape == (0, 100)
    far = torch.tensor([-3000.0, 0, 0, 0], device="cuda")                # log ratios of thousands: no overflow
    for sign in (1, -1):
        r = api.preference_loss(x, token.cuda(), st(0, 1, 2), ref_logp=sign * far, beta=1.0, smoothing=0.0)
        assert torch.isfinite(r.loss) and torch.isfinite(r.dx).all() and (r.loss.item() < 1e-6 if sign == 1 else r.loss.item() > 2900)
        r = api.preference_loss(x, token.cuda(), st(0, 1, 2), ref_logp=sign * far, beta=1.0, smoothing=1.0)
        assert torch.isfinite(r.loss) and torch.isfinite(r.dx).all()


def test_gradients_against_differences():
    """Central differences of the kernels' own losses (float32: steps of 1e-2 leave errors of about 1e-4)."""
    from whirl_llm_b200 import api
    rows, n = 6, 11
    x, x64, token, it, stats, adv, old, rf, weight = policy_inputs(rows, n, "f32", seed=31, masked=0.2, inv_t=0.9)
    x = x.contiguous()
    starts = torch.tensor([0, 2, 3, 5, 6], dtype=torch.int32).cuda()
    pol = lambda v, grad: api.policy_loss(v, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), inv_t=0.9, clip_low=5.0, clip_high=5.0,  # noqa: E731
                                          kl_coef=0.2, ent_coef=0.1, want_grad=grad)
    pref = lambda v, grad: api.preference_loss(v, token.cuda(), starts, rf.cuda(), weight.cuda(), inv_t=0.9, beta=0.7, smoothing=0.1,  # noqa: E731
                                               average=True, want_grad=grad)
    for f in (pol, pref):
        dx = f(x, True).dx.double().cpu()
        num = torch.zeros_like(dx)
        for i in range(rows):
            for j in range(n):
                v = []
                for e in (1e-2, -1e-2):
                    y = x.clone()
                    y[i, j] += e
                    v.append(f(y, False).loss.double().item())
                num[i, j] = (v[0] - v[1]) / 2e-2
        assert (num - dx).abs().max() < 3e-4, (num - dx).abs().max()
        assert dx.abs().max() > 1e-2


def test_rows_past_2_to_31_elements():
    """9000 rows of 262144 bf16 logits: offsets pass 32 bits; all rows but a few do not count and are not read."""
    from whirl_llm_b200 import api
    rows, n = 9000, 262144
    x = torch.empty((rows, n), dtype=torch.bfloat16, device="cuda")
    pick = [0, 8191, 8192, 8999]
    g = torch.Generator(device="cuda").manual_seed(1)
    token = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    for i, r in enumerate(pick):
        x[r].normal_(0, 3, generator=g)
        token[r] = 1000 * i + 5
    res = api.token_logprobs(x, token)
    small = api.token_logprobs(x[pick].contiguous(), token[pick].contiguous())
    # (a batch of four rows is split over more thread blocks: sums in another order)
    close(res.logp[pick], small.logp.cpu(), 2 * ref.logp_tol(n, small.logp.cpu().double()))
    close(res.stats[pick], small.stats.cpu(), 2 * ref.sum_error(n) * small.stats.cpu().double())
    gl = torch.ones(rows, device="cuda")
    d = api.token_logprobs_grad(x[pick].contiguous(), token[pick].contiguous(), small.stats, gl[:4])
    res.stats[pick] = small.stats
    dx = api.token_logprobs_grad(x, token, res.stats, gl)
    assert torch.equal(dx[pick], d) and (dx[100] == 0).all() and (dx[8998] == 0).all()
    adv = torch.ones(rows, device="cuda")
    p = api.policy_loss(x, token, adv, mean=0, dx=dx)
    q = api.policy_loss(x[pick].contiguous(), token[pick].contiguous(), adv[:4], mean=0)
    close(p.loss, q.loss.cpu(), 1e-6 * q.loss.abs().item())
    # both are off by at most a bf16 half step and some 1e-6 from the same value
    close(dx[pick], q.dx.cpu(), 2 * (2.0 ** -8 + 1e-5) * q.dx.cpu().double().abs() + 1e-6)
    assert (dx[8998] == 0).all()


def test_streams_threads_and_graphs():
    """The same results on a side stream, from two threads at once, and from a captured graph replayed on new inputs."""
    from whirl_llm_b200 import api
    rows, n = 33, 20011
    sets = [policy_inputs(rows, n, "f32", seed=50 + k) for k in range(2)]
    args = [[v.cuda() for v in (s[0], s[2], s[5], s[6], s[7], s[8])] for s in sets]
    starts = torch.tensor([0, 9, 20, 20, 33], dtype=torch.int32, device="cuda")

    def both(a):
        x, token, adv, old, rf, w = a
        p = api.policy_loss(x, token, adv, old, rf, w, kl_coef=0.1, ent_coef=0.01)
        q = api.preference_loss(x, token, starts, rf, w)
        return [p.loss, p.dx, p.row_loss, q.loss, q.dx]
    want = [[v.clone() for v in both(a)] for a in args]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(args[0])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    out = [[], []]

    def work(k):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                out[k] = both(args[k])
        st.synchronize()
    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(out[k], want[k]))
    # two graphs, replayed at the same time on two streams
    live = [[v.clone() for v in args[k]] for k in range(2)]
    graphs, outs = [], []
    for k in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(live[k]))
        graphs.append(gr)
    for k in range(2):  # other inputs than those of the capture
        for a, b in zip(live[k], args[1 - k]):
            a.copy_(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[k], want[1 - k]))


@pytest.mark.parametrize("rows,n,pad,dtype", [(2500, 4103, 1, "bf16"), (2500, 2049, 0, "f32"), (2400, 8200, 0, "f32"), (2400, 16385, 7, "bf16")])
def test_many_rows_of_middle_length(rows, n, pad, dtype):
    """Rows that a warp streams through its registers; some do not count."""
    from whirl_llm_b200 import api
    x, x64, token, it, stats, adv, old, rf, weight = policy_inputs(rows, n, dtype, seed=77, pad=pad, inv_t=0.8)
    token[5], token[100] = -1, n
    r = api.token_logprobs(x, token.cuda(), inv_t=0.8, want_entropy=True)
    ok = (token >= 0) & (token < n)
    want = torch.where(ok, stats[2], 0.0)
    close(r.logp, want, ref.logp_tol(n, want))
    close(r.entropy, torch.where(ok, stats[3], 0.0), ref.entropy_tol(n))
    g = torch.randn(rows, generator=torch.Generator().manual_seed(3))
    g[7] = 0.0
    dx = api.token_logprobs_grad(x, token.cuda(), r.stats, g.cuda(), inv_t=0.8)
    d, p, lp = ref.dlogits(x64, token, it, (stats[0], stats[1]), g.double())
    close(dx, d, ref.dx_tol(p, lp, g.double(), it, DT[dtype], d, n=n), "dx")
    assert (dx[[5, 7, 100]] == 0).all()
    out = torch.empty((rows, n), dtype=DT[dtype], device="cuda")
    assert torch.equal(api.token_logprobs_grad(x, token.cuda(), r.stats, g.cuda(), inv_t=0.8, dx=out), dx)
    f = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), inv_t=0.8, kl_coef=0.1, want_grad=False)
    check_policy(f, x64, token, it, stats, adv, old, rf, weight, 1, None, dtype, n, kl_coef=0.1)
    f = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), inv_t=0.8, kl_coef=0.1)
    check_policy(f, x64, token, it, stats, adv, old, rf, weight, 1, None, dtype, n, kl_coef=0.1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(40, 1003), (24, 33001), (70, 50000), (9, 151936)])
def test_losses_in_place_and_temperatures_per_row(rows, n, dtype):
    """dx = x, and inv_t per row, give the same bits as a dx of its own and the one inv_t."""
    from whirl_llm_b200 import api
    x, _, token, it, _, adv, old, rf, weight = policy_inputs(rows, n, dtype, seed=61, inv_t=0.8)
    x = x.contiguous()
    cuda = [v.cuda() for v in (token, adv, old, rf, weight)]
    starts = torch.tensor([0, rows // 3, rows // 2, rows // 2, rows - 1], dtype=torch.int32, device="cuda")
    per_row = torch.full((rows,), 0.8, device="cuda")

    def both(y, dx, **t):
        tok, a, o, r, w = cuda
        return (lambda d: api.policy_loss(y, tok, a, o, r, w, kl_coef=0.1, ent_coef=0.02, dx=d, **t),
                lambda d: api.preference_loss(y, tok, starts, r, w, dx=d, **t))
    for k in range(2):
        want = both(x, None, inv_t=0.8)[k](None)
        y = x.clone()
        got = both(y, y, inv_t=0.8)[k](y)
        assert got.dx is y and torch.equal(got.dx, want.dx) and torch.equal(got.loss, want.loss) and torch.equal(got.logp, want.logp)
        got = both(x, None, inv_t_rows=per_row)[k](None)
        assert torch.equal(got.dx, want.dx) and torch.equal(got.loss, want.loss) and torch.equal(got.stats, want.stats)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1003, 20001, 60000])
def test_policy_rows_of_every_kind(n, dtype):
    """Rows of the type's lowest value, rows without a distribution, huge logits and a single token left, through the policy loss."""
    from whirl_llm_b200 import api
    rows = 8
    x, _, token = make(rows, n, dtype, seed=71)
    x = x.clone().contiguous()
    low, high = torch.finfo(DT[dtype]).min, torch.finfo(DT[dtype]).max
    x[0] = low
    x[1] = -math.inf
    x[2, 5] = math.nan
    x[3] = -math.inf
    x[3, token[3].item()] = 1.0
    x[4, 17] = high
    x[5, : n // 2] = low
    x[6] = high
    x64, it = x.double().cpu(), ones(1.25, rows)
    m, s, lp, h = ref.row_stats(x64, it)
    want = lp.gather(1, token.long()[:, None])[:, 0].float().double()  # (as float32: -4e38 is -inf there)
    for place in (False, True):
        y = x.clone()
        r = api.policy_loss(y, token.cuda(), torch.ones(rows, device="cuda"), inv_t=1.25, mean=0, want_entropy=True, dx=y if place else None)
        close(r.logp, want, ref.logp_tol(n, want.clamp_min(-1e30)), "logp")
        close(r.entropy, h, ref.entropy_tol(n), "entropy")
        assert torch.isnan(r.loss)
        g = torch.full((rows,), -1.0, dtype=torch.float64)
        d, p, lpd = ref.dlogits(x64, token, it, (m, s), g)
        good = torch.tensor([0, 3, 4, 5, 6, 7])
        close(r.dx[good.cuda()], d[good], ref.dx_tol(p[good], lpd[good].clamp_min(-1e30), g[good], it[good], DT[dtype], d[good], n=n), "dx")
        assert torch.isnan(r.dx[1:3]).all()
        q = api.token_logprobs(x, token.cuda(), inv_t=1.25)
        close(q.logp, want, ref.logp_tol(n, want.clamp_min(-1e30)), "logp alone")
        dx = api.token_logprobs_grad(x, token.cuda(), q.stats, g.float().cuda(), inv_t=1.25)
        close(dx[good.cuda()], d[good], ref.dx_tol(p[good], lpd[good].clamp_min(-1e30), g[good], it[good], DT[dtype], d[good], n=n), "dx alone")


def test_rows_longer_than_a_cluster_holds():
    from whirl_llm_b200 import api
    rows, n = 3, 1000003
    x, x64, token, it, stats, adv, old, rf, weight = policy_inputs(rows, n, "f32", seed=81, masked=0.0)
    weight[1] = 0.0
    r = api.policy_loss(x, token.cuda(), adv.cuda(), old.cuda(), rf.cuda(), weight.cuda(), kl_coef=0.1, ent_coef=0.01)
    check_policy(r, x64, token, it, stats, adv, old, rf, weight, 1, None, "f32", n, kl_coef=0.1, ent_coef=0.01)
