"""The losses, log-probabilities and gradients of include/whirl_b200.h in 64 bits on the CPU, and the cache bookkeeping of one
step, one sequence after the other; and how far a 32-bit kernel may be from them."""
import math

import numpy as np
import torch

EPS32 = 2.0 ** -24  # half a step of float32


def row_stats(x, inv_t):
    """x [rows, n] float64, inv_t [rows] -> max, sum, log p [rows, n], entropy."""
    m = x.amax(1)
    z = (x - m[:, None]) * inv_t[:, None]
    w = z.exp()
    s = w.sum(1)
    lp = z - s.log()[:, None]
    p = lp.exp()
    bad = ~torch.isfinite(m) | torch.isnan(x).any(1)
    s = torch.where(bad, torch.nan, s)
    lp = torch.where(bad[:, None], torch.nan, lp)
    h = -(torch.where(p > 0, p * lp, 0.0)).sum(1)
    h = torch.where(bad, torch.nan, h)
    return m, s, lp, h


def dlogits(x, token, inv_t, stats, g, h=None, entropy=None):
    """The gradient by the logits from given (float64) max / sum, g = dL/dlogp, h = dL/dentropy; rows with g = h = 0 are zero."""
    m, s = stats
    lp = (x - m[:, None]) * inv_t[:, None] - s.log()[:, None]
    p = lp.exp()
    n = x.shape[1]
    ok = (token >= 0) & (token < n)
    zero = ~ok | ((g == 0) & (True if h is None else (h == 0)))
    d = -g[:, None] * p
    d[torch.arange(len(g)), token.clamp(0, n - 1).long()] += g
    if h is not None:
        d = d - h[:, None] * torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)
    d = d * inv_t[:, None]
    d[zero] = 0.0
    return d, p, lp


def sum_error(n):
    """Relative error of a float32 sum of n exponentials 2^t: a thread adds up to n / 256 of them one by one (half a step each), some 20
    partial sums are joined (three roundings each), a term is off by the exponential (2^-22) and by two roundings of its exponent and one
    of log2 e (1.5 steps of t, and sum w |t| / sum w <= log2 n)."""
    return (n / 256 + 60 + 4) * EPS32 + 3 * math.log2(max(n, 2)) * EPS32


def logp_tol(n, logp):
    return sum_error(n) + 2 * EPS32 * logp.abs().nan_to_num(0, 0, 0) + 1e-12


def entropy_tol(n):
    return 4 * sum_error(n) * (1 + math.log(max(n, 2)))


def dx_tol(p, lp, g, inv_t, dtype, value, h=None, entropy=None, n=2):
    """Per element: p is off by the exponential, the exponent's roundings (3 half steps of log2 p, each worth ln 2 of it), 1 / sum and
    the coefficient; the result is rounded to its type."""
    rel = 12 * EPS32 + 3 * EPS32 * lp.abs().nan_to_num(0, 0, 0) + sum_error(n)
    size = p * g.abs()[:, None] * rel + EPS32 * 2 * g.abs()[:, None]
    if h is not None:
        size = size + h.abs()[:, None] * p * (lp.abs().nan_to_num(0, 0, 0) + entropy.abs()[:, None] + 1) * (2 * rel + 4 * EPS32) + h.abs()[:, None] * p * entropy_tol(n)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else EPS32
    return size * inv_t[:, None] * 1.01 + half * value.abs() + 1e-37


def policy(logp, entropy, scale, adv, old=None, ref=None, clip_low=0.2, clip_high=0.2, dual_clip=0.0, kl_coef=0.0, ent_coef=0.0):
    """Row losses, kl and d row / d logp (float64 in, float64 out)."""
    d = torch.zeros_like(logp) if old is None else (logp - old)
    free_d = torch.ones_like(d, dtype=torch.bool) if old is None else (d > -20) & (d < 20)
    r = d.clamp(-20, 20).exp()
    a, b = r * adv, r.clamp(1 - clip_low, 1 + clip_high) * adv
    pg, g = torch.where(a <= b, -a, -b), torch.where((a <= b) & free_d, -a, 0.0)
    if dual_clip > 0:
        over = (adv < 0) & (pg > -dual_clip * adv)
        pg, g = torch.where(over, -dual_clip * adv, pg), torch.where(over, 0.0, g)
    kl = torch.zeros_like(pg)
    if ref is not None:
        k = ref - logp
        free_k = (k > -20) & (k < 20)
        k = k.clamp(-20, 20)
        kl = torch.expm1(k) - k
        g = g - torch.where(free_k, kl_coef * torch.expm1(k), 0.0)
    row = pg + kl_coef * kl - (ent_coef * entropy if ent_coef else 0.0)
    return row, kl, g


def row_scale(weight, mean, seq_start=None):
    """weight: float64, 0 for the rows that do not count."""
    if mean == 0:
        return weight.clone()
    if mean == 1:
        t = weight.sum()
        return weight / t if t > 0 else torch.zeros_like(weight)
    s = torch.zeros_like(weight)
    parts = [(a, b) for a, b in zip(seq_start[:-1], seq_start[1:]) if weight[a:b].sum() > 0]
    for a, b in parts:
        s[a:b] = weight[a:b] / weight[a:b].sum() / len(parts)
    return s


def pair_loss(h, kind, beta, smoothing):
    """Loss and d loss / dh."""
    if kind == 0:
        up = torch.sigmoid(h)
        return ((1 - smoothing) * torch.nn.functional.softplus(-h, threshold=1e9) + smoothing * torch.nn.functional.softplus(h, threshold=1e9),
                smoothing * up - (1 - smoothing) * (1 - up))
    if kind == 1:
        return (1 - h).clamp_min(0), torch.where(h < 1, -1.0, 0.0).double()
    t = (h - 0.5) / beta
    return t * t, 2 * t / beta


def step(length, n_new, table, owned, free_ids, free_count, block_size, max_rows):
    """One step of the cache bookkeeping; numpy arrays, updated copies returned."""
    table, owned, stack, top = table.copy(), owned.copy(), free_ids.copy(), int(free_count[0])
    seqs, width = table.shape
    status, plan, asked = np.zeros(seqs, np.int32), {}, 0
    for s in range(seqs):
        ln, nn = int(length[s]), int(n_new[s])
        target = -(-(ln + nn) // block_size)
        if ln < 0 or nn < 0 or ln + nn > 2 ** 31 - 1 or target > width:
            status[s] = 2
            continue
        asked += nn
        if nn and asked > max_rows:
            status[s] = 1
            continue
        plan[s] = target
        for j in range(target, int(owned[s])):
            stack[top] = table[s, j]
            top += 1
    have, wanted = top, 0
    slot, position, seq = np.full(max_rows, -1, np.int64), np.zeros(max_rows, np.int32), np.full(max_rows, -1, np.int32)
    row0, at = [0], 0
    for s in range(seqs):
        if s in plan:
            need = max(0, plan[s] - int(owned[s]))
            wanted += need
            if need and wanted > have:
                status[s] = 1
            else:
                for j in range(need):
                    top -= 1
                    table[s, int(owned[s]) + j] = stack[top]
                owned[s] = plan[s]
                for i in range(int(n_new[s])):
                    p = int(length[s]) + i
                    slot[at], position[at], seq[at] = int(table[s, p // block_size]) * block_size + p % block_size, p, s
                    at += 1
        row0.append(at)
    return dict(slot=slot, position=position, seq=seq, row0=np.array(row0, np.int32), status=status, table=table, owned=owned, free_ids=stack,
                free_count=np.array([top], np.int32))
