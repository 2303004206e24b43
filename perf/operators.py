"""What the operators around a sampled token cost: log-probabilities of given tokens and their gradient, the clipped policy
loss and the preference loss with their gradients down to the logits, and the cache block tables of the next step.

`run` computes an operator in its plain form (elementary torch operations) or, where `own` is true, through
whirl_llm_b200.api.  A case is a dict of plain values; `op` names the operator.
"""
import math

import numpy as np
import torch

own = False

MEANS = {"sum": 0, "tokens": 1, "seqs": 2}      # api.MEAN_*
KINDS = {"sigmoid": 0, "hinge": 1, "squared": 2}  # api.PREF_*


# ---- cases ------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one decoded token's log-probability: the smallest call, latency only
        dict(name="logprobs 1 x 151936 bf16", op="logprobs", rows=1, n=151936, dtype="bf16", pad=0, temp=1.0, entropy=False, masked=False),
        # scoring a rollout batch at the sampler's headline size, entropy for the log book, 1 % of the vocabulary forbidden
        dict(name="logprobs 1024 x 262144 f32", op="logprobs", rows=1024, n=262144, dtype="f32", pad=0, temp=0.8, entropy=True, masked=True),
        # the gradient of a user's own loss on a small batch
        dict(name="grad 64 x 151936 f32", op="logprobs_grad", rows=64, n=151936, dtype="f32", pad=0, temp=1.0, entropy=False),
        # the same for a large batch, with a gradient through the entropy
        dict(name="grad 1024 x 262144 bf16", op="logprobs_grad", rows=1024, n=262144, dtype="bf16", pad=0, temp=0.8, entropy=True),
        # policy step on a handful of short answers (16 sequences x 9 tokens)
        dict(name="policy 144 x 151936 f32", op="policy", rows=144, n=151936, dtype="f32", pad=0, temp=1.0, mask=0.0, seqs=16, kl=0.05, ent=0.0,
             high=0.2, dual=0.0, mean="tokens"),
        # a micro-batch of a policy step, a third of it prompt
        dict(name="policy 4096 x 151936 bf16", op="policy", rows=4096, n=151936, dtype="bf16", pad=0, temp=1.0, mask=0.33, seqs=24, kl=0.02,
             ent=0.0, high=0.28, dual=3.0, mean="tokens"),
        # odd vocabulary inside padded rows, entropy bonus, every sequence weighing the same
        dict(name="policy 1000 x 131071 f32", op="policy", rows=1000, n=131071, dtype="f32", pad=1, temp=0.8, mask=0.1, seqs=13, kl=0.05,
             ent=0.01, high=0.2, dual=0.0, mean="seqs"),
        # pairs of short answers, a small vocabulary
        dict(name="preference 600 x 32768 bf16", op="preference", rows=600, n=32768, dtype="bf16", pad=0, temp=1.0, mask=0.25, pairs=8,
             kind="sigmoid", beta=0.1, smoothing=0.0, margin=0.0, average=False),
        # a micro-batch of preference training, label smoothing, half of it prompt
        dict(name="preference 4096 x 151936 bf16", op="preference", rows=4096, n=151936, dtype="bf16", pad=0, temp=1.0, mask=0.5, pairs=8,
             kind="sigmoid", beta=0.1, smoothing=0.1, margin=0.0, average=False),
        # speculative decoding of 16 sequences with up to 8 drafts each
        dict(name="blocks 16 x 9", op="blocks", seqs=16, rows=144, block=16, max_blocks=256, pool=0.7),
        # a busy server: 1024 sequences of up to 16384 tokens
        dict(name="blocks 1024 x 9", op="blocks", seqs=1024, rows=9216, block=16, max_blocks=1024, pool=0.5),
        # prompts coming in: half a million new rows over 256 sequences
        dict(name="blocks prefill 256 x 2048", op="blocks", seqs=256, rows=524288, block=64, max_blocks=256, pool=0.6),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs_grad", "policy", "preference", "blocks"])
    if op == "blocks":
        seqs = _log_int(rng, 1, 1024)
        rows = min(524288, seqs * _log_int(rng, 1, 2048))
        block = rng.choice([1, 8, 16, 24, 32, 64, 128])
        most = max(4, min(1048576 // seqs, 2 * (rows // seqs) // block + _log_int(rng, 8, 1024)))
        return dict(op=op, seqs=seqs, rows=rows, block=block, max_blocks=most, pool=rng.choice([0.3, 0.5, 0.7, 1.0]))
    n = _log_int(rng, 1000, 262144)
    dtype = rng.choice(["f32", "bf16"])
    most = {"logprobs": 1024 * 262144, "logprobs_grad": 1024 * 262144, "policy": 2048 * 151936, "preference": 2048 * 151936}[op]
    rows = _log_int(rng, 1 if op.startswith("logprobs") else 16, min(8192, most // n))
    case = dict(op=op, rows=rows, n=n, dtype=dtype, pad=rng.choice([0, 0, 0, 1, 8, 64]), temp=rng.choice([0.7, 0.8, 1.0, 1.0, 1.2]))
    if op == "logprobs":
        return dict(case, entropy=rng.random() < 0.5, masked=rng.random() < 0.3)
    if op == "logprobs_grad":
        return dict(case, entropy=rng.random() < 0.5)
    case["mask"] = rng.choice([0.0, 0.1, 0.33, 0.5])
    if op == "policy":
        return dict(case, seqs=max(1, rows // _log_int(rng, 8, 512)), kl=rng.choice([0.0, 0.02, 0.1]), ent=rng.choice([0.0, 0.0, 0.01]),
                    high=rng.choice([0.2, 0.28]), dual=rng.choice([0.0, 3.0]), mean=rng.choice(sorted(MEANS)))
    return dict(case, pairs=max(1, rows // (2 * _log_int(rng, 8, 512))), kind=rng.choice(sorted(KINDS)), beta=rng.choice([0.1, 0.5]),
                smoothing=rng.choice([0.0, 0.1]), margin=rng.choice([0.0, 0.5]), average=rng.random() < 0.4)


def _size(case):
    return 4 if case["dtype"] == "f32" else 2


def _live(case):
    """Rows that weigh something (prompt tokens and the rows behind the last sequence do not)."""
    return case["rows"] - int(case["rows"] * case.get("mask", 0.0))


def work(case):
    if case["op"] == "blocks":
        # lengths, counts and outputs of every sequence; slot (8 B), position and sequence of every row; one block id in for each block
        # that the rows touch and one out for each new one (about a block id per `block` rows, one per sequence at least)
        ids = max(case["seqs"], case["rows"] // case["block"])
        return {"bytes": 20.0 * case["seqs"] + 16.0 * case["rows"] + 8.0 * ids, "flops": 0.0}
    full, live = case["rows"] * case["n"] * _size(case), _live(case) * case["n"] * _size(case)
    per_logit = {"logprobs": 4, "logprobs_grad": 4, "policy": 8, "preference": 8}[case["op"]] + 2 * bool(case.get("entropy") or case.get("ent"))
    moved = {"logprobs": full, "logprobs_grad": 2 * full, "policy": live + full, "preference": live + full}[case["op"]]
    return {"bytes": float(moved + 32 * case["rows"]), "flops": float(per_logit) * _live(case) * case["n"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _logits(case, g):
    """Logits N(0, 3^2) with a sampled token that stands out as sampled tokens do, and (masked) 1 % of the vocabulary at -inf."""
    rows, n = case["rows"], case["n"]
    x = torch.empty((rows, n + case["pad"]), dtype=torch.float32 if case["dtype"] == "f32" else torch.bfloat16, device="cuda")
    x.normal_(0.0, 3.0, generator=g)
    x = x[:, :n]
    if case.get("masked"):
        x.masked_fill_(torch.rand((rows, n), device="cuda", generator=g) < 0.01, -math.inf)
    token = torch.randint(0, n, (rows,), device="cuda", generator=g)
    top = math.log(n) + 2.0 + 3.0 * torch.randn(rows, device="cuda", generator=g)
    x.scatter_(1, token[:, None], top.to(x.dtype)[:, None])
    return x, token.to(torch.int32)


def _stats64(x, token, inv_t):
    """max, sum, log-probability of the token and entropy of every row in 64 bits."""
    rows, n = x.shape
    step = max(1, (1 << 26) // n)
    parts = []
    for r in range(0, rows, step):
        z = x[r: r + step].double()
        m = z.amax(1)
        z = (z - m[:, None]) * inv_t
        w = z.exp()
        s = w.sum(1)
        t = z.gather(1, token[r: r + step].long()[:, None])[:, 0]
        parts.append(torch.stack([m, s, t - s.log(), s.log() - torch.where(w > 0, w * z, 0.0).sum(1) / s]))
    return torch.cat(parts, 1)


def _starts(case, seqs, g):
    """Ragged sequences over most of the rows, one of them empty where there are several: seq_start [seqs + 1]."""
    share = -torch.rand(seqs, device="cuda", generator=g).clamp_min(1e-6).log() + 0.2
    if seqs > 3:
        share[seqs // 2] = 0.0
    ends = (share.cumsum(0) / share.sum() * (case["rows"] * 0.98)).floor()
    return torch.cat([torch.zeros(1, device="cuda"), ends]).to(torch.int32)


def _weights(case, g):
    """1 for the answers' tokens, 0 for the rest."""
    w = torch.ones(case["rows"], device="cuda")
    w[torch.randperm(case["rows"], device="cuda", generator=g)[: int(case["rows"] * case["mask"])]] = 0.0
    return w


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "blocks":
        return _prepare_blocks(case, g)
    x, token = _logits(case, g)
    st = dict(case=case, x=x, token=token, inv_t=float(np.float32(1.0 / case["temp"])))
    rows = case["rows"]
    if case["op"] == "logprobs":
        return st
    m, s, logp, entropy = _stats64(x, token, st["inv_t"])
    if case["op"] == "logprobs_grad":  # what the forward pass left, and the gradients that come back to it
        st["stats"] = torch.stack([m, s], 1).float()
        st["entropy"] = entropy.float() if case["entropy"] else None
        st["g_logp"] = torch.randn(rows, device="cuda", generator=g) / rows
        st["g_entropy"] = torch.randn(rows, device="cuda", generator=g) / rows if case["entropy"] else None
        return st
    st["weight"] = _weights(case, g)
    if case["op"] == "policy":
        st["seq_start"] = _starts(case, case["seqs"], g)
        # advantages: their mean over the tokens is not zero, since good answers and bad ones differ in length
        st["adv"] = 0.4 + torch.randn(rows, device="cuda", generator=g)
        # the sampling policy was close to the present one; no ratio within 1e-3 of a clip edge, where a last bit decides
        d = 0.15 * torch.randn(rows, device="cuda", generator=g, dtype=torch.float64)
        for edge in (math.log(0.8), math.log(1.0 + case["high"])) + ((math.log(case["dual"]),) if case["dual"] else ()):
            d = torch.where((d - edge).abs() < 1e-3, d + 2e-3, d)
        st["old_logp"] = (logp - d).float()
        st["ref_logp"] = (logp + 0.3 * torch.randn(rows, device="cuda", generator=g)).float() if case["kl"] else None
        return st
    st["seq_start"] = _starts(case, 2 * case["pairs"], g)
    st["ref_logp"] = None if case["average"] else (logp + 0.3 * torch.randn(rows, device="cuda", generator=g)).float()
    return st


def _prepare_blocks(case, g):
    seqs, bs, width = case["seqs"], case["block"], case["max_blocks"]
    rand = lambda: torch.rand(seqs, device="cuda", generator=g)  # noqa: E731
    plans = []
    for k in range(2):  # two steps of the same server, taken in turn: most sequences grow, one in eight is over and another takes its place
        if case["rows"] <= 16 * seqs:
            new = 1 + (rand() * (2 * case["rows"] // seqs - 1)).floor()
        else:
            share = -rand().clamp_min(1e-6).log() + 0.05
            new = (share / share.sum() * case["rows"]).floor()
        new = new.clamp_max(bs * width).to(torch.int64)
        new = torch.where(new.cumsum(0) <= case["rows"], new, 0)
        room = (bs * width - new).clamp_min(0).double()
        length = (0.8 * room * rand().double()).floor() if k == 0 else plans[0][0].double() + 1
        length = torch.where(rand() < 0.125, torch.zeros_like(length), torch.minimum(length, room)).to(torch.int64)
        plans.append((length, new))
    blocks = max(1, int(case["pool"] * seqs * width))
    return dict(case=case, plans=[(a.to(torch.int32), b.to(torch.int32)) for a, b in plans], turn=0,
                table=torch.full((seqs, width), -1, dtype=torch.int32, device="cuda"), owned=torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                free_ids=torch.randperm(blocks, device="cuda", generator=g).to(torch.int32),
                free_count=torch.full((1,), blocks, dtype=torch.int32, device="cuda"))


# ---- one pass -----------------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logprobs": _own_logprobs, "logprobs_grad": _own_grad, "policy": _own_policy, "preference": _own_preference, "blocks": _own_blocks}[op](state)
    return {"logprobs": _plain_logprobs, "logprobs_grad": _plain_grad, "policy": _plain_policy, "preference": _plain_preference,
            "blocks": _plain_blocks}[op](state)


def _turn(st):
    plan = st["plans"][st["turn"]]
    st["turn"] ^= 1
    return plan


def _own_logprobs(st):
    from whirl_llm_b200 import api
    r = api.token_logprobs(st["x"], st["token"], inv_t=st["inv_t"], want_entropy=st["case"]["entropy"])
    return dict(logp=r.logp, stats=r.stats, entropy=r.entropy)


def _own_grad(st):
    from whirl_llm_b200 import api
    return api.token_logprobs_grad(st["x"], st["token"], st["stats"], st["g_logp"], inv_t=st["inv_t"], entropy=st["entropy"],
                                   g_entropy=st["g_entropy"])


def _own_policy(st):
    from whirl_llm_b200 import api
    c = st["case"]
    r = api.policy_loss(st["x"], st["token"], st["adv"], old_logp=st["old_logp"], ref_logp=st["ref_logp"], weight=st["weight"],
                        seq_start=st["seq_start"] if c["mean"] == "seqs" else None, inv_t=st["inv_t"], clip_low=0.2, clip_high=c["high"],
                        dual_clip=c["dual"], kl_coef=c["kl"], ent_coef=c["ent"], mean=MEANS[c["mean"]], want_grad=True)
    return dict(loss=r.loss, logp=r.logp, kl=r.kl, entropy=r.entropy, row_loss=r.row_loss, dx=r.dx)


def _own_preference(st):
    from whirl_llm_b200 import api
    c = st["case"]
    r = api.preference_loss(st["x"], st["token"], st["seq_start"], ref_logp=st["ref_logp"], weight=st["weight"], inv_t=st["inv_t"],
                            beta=c["beta"], kind=KINDS[c["kind"]], smoothing=c["smoothing"], margin=c["margin"], average=c["average"],
                            want_grad=True)
    return dict(loss=r.loss, pair_loss=r.pair_loss, reward=r.reward, logp=r.logp, dx=r.dx)


def _own_blocks(st):
    from whirl_llm_b200 import api
    c = st["case"]
    length, new = _turn(st)
    r = api.block_tables_step(length, new, st["table"], st["owned"], st["free_ids"], st["free_count"], block_size=c["block"], max_rows=c["rows"])
    return dict(slot=r.slot, position=r.position, seq=r.seq, row0=r.row0, status=r.status, table=st["table"], owned=st["owned"],
                free_ids=st["free_ids"], free_count=st["free_count"])


# ---- the plain forms ------------------------------------------------------------------------------------------------------


def _softmax(x, inv_t):
    """Row maximum, exponents (x - max) inv_t, their exponentials and sums, in 32 bits."""
    xf = x.float()
    m = xf.amax(1)
    d = (xf - m[:, None]) * inv_t
    w = d.exp()
    return m, d, w, w.sum(1)


def _at(d, token):
    return d.gather(1, token.long()[:, None])[:, 0]


def _entropy(d, w, s):
    return s.log() - torch.where(w > 0, w * d, 0.0).sum(1) / s


def _dlogits(d, w, s, token, g, h, entropy, inv_t, dtype):
    """inv_t (g (delta - p) - h p (log p + H))."""
    p = w / s[:, None]
    dx = p * -g[:, None]
    dx.scatter_add_(1, token.long()[:, None], g[:, None])
    if h is not None:
        dx = dx - torch.where(p > 0, h[:, None] * p * (d - s.log()[:, None] + entropy[:, None]), 0.0)
    return (dx * inv_t).to(dtype)


def _plain_logprobs(st):
    m, d, w, s = _softmax(st["x"], st["inv_t"])
    return dict(logp=_at(d, st["token"]) - s.log(), stats=torch.stack([m, s], 1), entropy=_entropy(d, w, s) if st["case"]["entropy"] else None)


def _plain_grad(st):
    d = (st["x"].float() - st["stats"][:, :1]) * st["inv_t"]
    return _dlogits(d, d.exp(), st["stats"][:, 1], st["token"], st["g_logp"], st["g_entropy"], st["entropy"], st["inv_t"], st["x"].dtype)


def _seq_of(seq_start, rows):
    """Sequence of every row; `seqs` for the rows behind the last one."""
    return torch.searchsorted(seq_start[1:].long(), torch.arange(rows, device=seq_start.device), right=True)


def _seq_sums(v, seq, seqs):
    return torch.zeros(seqs + 1, dtype=torch.float64, device=v.device).index_add_(0, seq, v.double())[:seqs]


def _row_scale(weight, seq_start, mean, rows):
    if mean == "sum":
        return weight.double()
    if mean == "tokens":
        total = weight.double().sum()
        return torch.where(total > 0, weight.double() / total, 0.0)
    seqs = seq_start.numel() - 1
    seq = _seq_of(seq_start, rows)
    total = _seq_sums(weight, seq, seqs)
    share = torch.where(total > 0, 1.0 / (total * (total > 0).sum()), 0.0)
    return weight.double() * torch.cat([share, share.new_zeros(1)])[seq]


def _policy_rows(logp, old, ref, adv, entropy, c):
    """Row losses and their derivatives by logp; the rows' own arithmetic is in 64 bits (differences of log-probabilities)."""
    d = (logp - old.double()).clamp(-20, 20)
    r = d.exp()
    a = adv.double()
    plain, clipped = r * a, r.clamp(1 - 0.2, 1 + c["high"]) * a
    pg, dpg = -torch.minimum(plain, clipped), torch.where((plain <= clipped) & (d.abs() < 20), -a * r, 0.0)
    if c["dual"]:
        over = (a < 0) & (pg > -c["dual"] * a)
        pg, dpg = torch.where(over, -c["dual"] * a, pg), torch.where(over, 0.0, dpg)
    kl = torch.zeros_like(pg)
    if ref is not None:
        k = (ref.double() - logp).clamp(-20, 20)
        kl = torch.expm1(k) - k
        dpg = dpg - c["kl"] * torch.where(k.abs() < 20, torch.expm1(k), 0.0)
    row = pg + c["kl"] * kl
    return (row - c["ent"] * entropy if entropy is not None else row), kl, dpg


def _plain_policy(st):
    c, x = st["case"], st["x"]
    _, d, w, s = _softmax(x, st["inv_t"])
    live = st["weight"] > 0
    logp = _at(d, st["token"]).double() - s.double().log()
    entropy = _entropy(d, w, s) if c["ent"] else None
    scale = _row_scale(st["weight"], st["seq_start"], c["mean"], c["rows"])
    row, kl, dlogp = _policy_rows(logp, st["old_logp"], st["ref_logp"], st["adv"], None if entropy is None else entropy.double(), c)
    g = torch.where(live, scale * dlogp, 0.0).float()
    h = (-c["ent"] * scale).float() if c["ent"] else None
    dx = _dlogits(d, w, s, st["token"], g, h, entropy, st["inv_t"], x.dtype)
    on = lambda v: torch.where(live, v, 0.0).float()  # noqa: E731
    return dict(loss=(on(row).double() * scale).sum().float(), logp=on(logp), kl=on(kl) if st["ref_logp"] is not None else None,
                entropy=on(entropy) if c["ent"] else None, row_loss=on(row), dx=dx)


def _pair_losses(u, c):
    """Loss and derivative of every pair by u, the difference of the log ratios."""
    h = c["beta"] * u - c["margin"]
    if c["kind"] == "sigmoid":
        ls = c["smoothing"]
        loss = -(1 - ls) * torch.nn.functional.logsigmoid(h) - ls * torch.nn.functional.logsigmoid(-h)
        return loss, c["beta"] * (ls * torch.sigmoid(h) - (1 - ls) * torch.sigmoid(-h))
    if c["kind"] == "hinge":
        return (1 - h).clamp_min(0), torch.where(h < 1, -c["beta"], 0.0).to(h.dtype)
    t = (h - 0.5) / c["beta"]
    return t * t, 2 * t


def _plain_preference(st):
    c, x, pairs, rows = st["case"], st["x"], st["case"]["pairs"], st["case"]["rows"]
    _, d, w, s = _softmax(x, st["inv_t"])
    seq = _seq_of(st["seq_start"], rows)
    weight = torch.where(seq < 2 * pairs, st["weight"], 0.0).double()
    logp = torch.where(weight > 0, _at(d, st["token"]).double() - s.double().log(), 0.0)
    share = torch.ones(2 * pairs, dtype=torch.float64, device=x.device)
    if c["average"]:
        total = _seq_sums(weight, seq, 2 * pairs)
        share = torch.where(total > 0, 1.0 / total, 0.0)
    ratio = logp if st["ref_logp"] is None else logp - st["ref_logp"].double()
    p = _seq_sums(weight * ratio, seq, 2 * pairs) * share
    loss, du = _pair_losses(p[0::2] - p[1::2], c)
    coef = torch.stack([du, -du], 1).reshape(-1) * share / pairs
    g = weight * torch.cat([coef, coef.new_zeros(1)])[seq]
    dx = _dlogits(d, w, s, st["token"], g.float(), None, None, st["inv_t"], x.dtype)
    return dict(loss=loss.mean().float(), pair_loss=loss.float(), reward=(c["beta"] * p).float().view(pairs, 2), logp=logp.float(), dx=dx)


def _plain_blocks(st):
    c = st["case"]
    length, new = (v.long() for v in _turn(st))
    table, owned, free_ids, count = st["table"], st["owned"].long(), st["free_ids"], st["free_count"].long()
    seqs, width = table.shape
    bs, rows, dev = c["block"], c["rows"], table.device
    target = (length + new + bs - 1) // bs
    valid = (length >= 0) & (new >= 0) & (target <= width)
    asked = torch.where(valid, new, 0)
    fits = valid & ((new == 0) | (asked.cumsum(0) <= rows))
    release = torch.where(fits, (owned - target).clamp_min(0), 0)
    need = torch.where(fits, (target - owned).clamp_min(0), 0)
    back, taken = release.cumsum(0), need.cumsum(0)
    have = count + back[-1]
    granted = fits & ((need == 0) | (taken <= have))
    status = torch.where(valid, torch.where(granted, 0, 1), 2).int()
    # released ids go on the stack of free blocks in the sequences' order, new ones come from its top
    col = torch.arange(width, device=dev)[None, :]
    out = (col >= target[:, None]) & (col < owned[:, None]) & (release > 0)[:, None]
    spot = torch.where(out, count + (back - release)[:, None] + col - target[:, None], free_ids.numel())
    stack = torch.cat([free_ids, free_ids.new_zeros(1)])
    stack.scatter_(0, spot.view(-1), torch.where(out, table, 0).view(-1))
    free_ids.copy_(stack[:-1])
    got = (col >= owned[:, None]) & (col < target[:, None]) & (granted & (need > 0))[:, None]
    source = torch.where(got, have - 1 - (taken - need)[:, None] - (col - owned[:, None]), 0)
    table.copy_(torch.where(got, free_ids[source], table))
    st["owned"].copy_(torch.where(granted, target, owned))
    st["free_count"].copy_(have - torch.where(granted, need, 0).sum())
    n = torch.where(granted, new, 0)
    ends = n.cumsum(0)
    row0 = torch.cat([ends.new_zeros(1), ends]).int()
    r = torch.arange(rows, device=dev)
    seq = torch.searchsorted(ends, r, right=True)
    live, at = seq < seqs, seq.clamp_max(seqs - 1)
    position = torch.where(live, length[at] + r - row0[at], 0)
    slot = table[at, torch.where(live, position // bs, 0)].long() * bs + position % bs
    return dict(slot=torch.where(live, slot, -1), position=position.int(), seq=torch.where(live, seq, -1).int(), row0=row0, status=status,
                table=table, owned=st["owned"], free_ids=free_ids, free_count=st["free_count"])


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "blocks":
        return _exact_blocks(st)
    x, token, inv_t = st["x"], st["token"].long(), st["inv_t"]
    m, s, logp, entropy = _stats64(x, token, inv_t)
    if case["op"] == "logprobs":
        return dict(logp=logp, stats=torch.stack([m, s], 1), entropy=entropy if case["entropy"] else None)
    if case["op"] == "logprobs_grad":
        m, s = st["stats"].double().unbind(1)
        h = st["g_entropy"].double() if case["entropy"] else None
        return _exact_dx(x, token, m, s, st["g_logp"].double(), h, None if h is None else st["entropy"].double(), inv_t)
    rows, w = case["rows"], st["weight"].double()
    starts = st["seq_start"].tolist()
    if case["op"] == "policy":
        scale = torch.zeros_like(w)
        if case["mean"] == "sum":
            scale = w
        elif case["mean"] == "tokens":
            scale = w / max(float(w.sum()), 1e-300)
        else:
            sums = [float(w[a:b].sum()) for a, b in zip(starts, starts[1:])]
            for (a, b), total in zip(zip(starts, starts[1:]), sums):
                if total > 0:
                    scale[a:b] = w[a:b] / total / sum(v > 0 for v in sums)
        at = logp.clone().requires_grad_()
        ratio = (at - st["old_logp"].double()).clamp(-20, 20).exp()
        a = st["adv"].double()
        row = torch.maximum(-ratio * a, -ratio.clamp(0.8, 1 + case["high"]) * a)
        if case["dual"]:
            row = torch.where(a < 0, torch.minimum(row, -case["dual"] * a), row)
        kl = None
        if st["ref_logp"] is not None:
            k = (st["ref_logp"].double() - at).clamp(-20, 20)
            kl = torch.expm1(k) - k
            row = row + case["kl"] * kl
        if case["ent"]:
            row = row - case["ent"] * entropy
        live = (w > 0).double()
        (scale * live * row).sum().backward()
        row = row.detach() * live
        dx = _exact_dx(x, token, m, s, at.grad, -case["ent"] * scale if case["ent"] else None, entropy, inv_t)
        return dict(loss=(scale * row).sum(), logp=logp * live, kl=None if kl is None else kl.detach() * live,
                    entropy=entropy * live if case["ent"] else None, row_loss=row, dx=dx)
    w[starts[-1]:] = 0.0
    at = torch.where(w > 0, logp, 0.0).requires_grad_()
    ratio = at if st["ref_logp"] is None else at - st["ref_logp"].double()
    sums = [(w[a:b] * ratio[a:b]).sum() / (max(float(w[a:b].sum()), 1e-300) if case["average"] else 1.0) for a, b in zip(starts, starts[1:])]
    p = torch.stack(sums)
    h = case["beta"] * (p[0::2] - p[1::2]) - case["margin"]
    if case["kind"] == "sigmoid":
        loss = (1 - case["smoothing"]) * torch.nn.functional.softplus(-h, threshold=1e9) + case["smoothing"] * torch.nn.functional.softplus(h, threshold=1e9)
    elif case["kind"] == "hinge":
        loss = torch.relu(1 - h)
    else:
        loss = ((h - 0.5) / case["beta"]) ** 2
    loss.mean().backward()
    dx = _exact_dx(x, token, m, s, at.grad, None, None, inv_t)
    return dict(loss=loss.mean().detach(), pair_loss=loss.detach(), reward=(case["beta"] * p).detach().view(-1, 2), logp=at.detach(), dx=dx)


def _exact_dx(x, token, m, s, g, h, entropy, inv_t):
    """The gradient by the logits, a block of rows at a time; rows whose coefficients are zero are zero."""
    out = []
    step = max(1, (1 << 26) // x.shape[1])
    for r in range(0, x.shape[0], step):
        b = slice(r, r + step)
        lp = (x[b].double() - m[b, None]) * inv_t - s[b].log()[:, None]
        p = lp.exp()
        v = -g[b, None] * p
        v[torch.arange(v.shape[0], device=v.device), token[b]] += g[b]
        if h is not None:
            v -= h[b, None] * torch.where(p > 0, p * (lp + entropy[b, None]), 0.0)
        out.append(v.mul_(inv_t).to(torch.float32 if x.dtype == torch.bfloat16 else torch.float64))
    return torch.cat(out)


def _exact_blocks(st):
    """The server's bookkeeping, one sequence after the other."""
    c = st["case"]
    length, new = (v.tolist() for v in _turn(st))
    table, owned, stack = st["table"].cpu().numpy().copy(), st["owned"].tolist(), st["free_ids"].cpu().numpy().copy()
    top, bs, rows = int(st["free_count"]), c["block"], c["rows"]
    seqs, width = table.shape
    status, plan, asked = [0] * seqs, {}, 0
    for s in range(seqs):
        target = -(-(length[s] + new[s]) // bs)
        if length[s] < 0 or new[s] < 0 or target > width:
            status[s] = 2
            continue
        asked += new[s]
        if new[s] and asked > rows:
            status[s] = 1
            continue
        plan[s] = target
        for j in range(target, owned[s]):
            stack[top] = table[s, j]
            top += 1
    have, wanted = top, 0
    slot, position, seq, row0, at = np.full(rows, -1, np.int64), np.zeros(rows, np.int32), np.full(rows, -1, np.int32), [0], 0
    for s in range(seqs):
        if s in plan:
            need = max(0, plan[s] - owned[s])
            wanted += need
            if need and wanted > have:
                status[s] = 1
            else:
                table[s, owned[s]: owned[s] + need] = stack[top - need: top][::-1]
                top -= need
                owned[s] = plan[s]
                p = length[s] + np.arange(new[s])
                slot[at: at + new[s]] = table[s, p // bs].astype(np.int64) * bs + p % bs
                position[at: at + new[s]], seq[at: at + new[s]] = p, s
                at += new[s]
        row0.append(at)
    i32 = lambda v: np.array(v, dtype=np.int32)  # noqa: E731
    return dict(slot=slot, position=position, seq=seq, row0=i32(row0), status=i32(status), table=table, owned=i32(owned), free_ids=stack,
                free_count=i32([top]))
