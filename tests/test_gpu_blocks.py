"""Cache block tables and slot maps: the device step against the bookkeeping one sequence after the other (loss_ref.step),
and a run of the serving and training calls together, as an engine would make them."""
import numpy as np
import pytest
import torch

import loss_ref as ref
from gpu_util import dev

pytestmark = pytest.mark.gpu


def fresh(rng, seqs, width, blocks):
    return dict(table=np.full((seqs, width), -1, np.int32), owned=np.zeros(seqs, np.int32), free_ids=rng.permutation(blocks).astype(np.int32),
                free_count=np.array([blocks], np.int32))


def check_step(st, d, length, n_new, block_size, max_rows):
    """One step on both sides; st: numpy state (replaced by the new one), d: device state."""
    from whirl_llm_b200 import api
    want = ref.step(length, n_new, **st, block_size=block_size, max_rows=max_rows)
    r = api.block_tables_step(dev(length.astype(np.int32)), dev(n_new.astype(np.int32)), d["table"], d["owned"], d["free_ids"], d["free_count"],
                              block_size=block_size, max_rows=max_rows)
    got = dict(slot=r.slot, position=r.position, seq=r.seq, row0=r.row0, status=r.status, **d)
    for k, v in got.items():
        assert np.array_equal(v.cpu().numpy(), want[k]), (k, v.cpu().numpy()[:20], want[k][:20])
    for k in st:
        st[k] = want[k]
    return want


CASES = [(1, 4, 4, 1, 4), (3, 5, 9, 16, 40), (40, 33, 700, 16, 200), (31, 64, 1000, 24, 4000), (1024, 12, 9000, 8, 6000), (1025, 7, 4000, 1, 3000),
         (2500, 9, 15000, 16, 30000), (5000, 3, 9000, 64, 20000), (8, 1000, 6000, 128, 60000)]


@pytest.mark.parametrize("seqs,width,blocks,block_size,max_rows", CASES)
def test_steps(seqs, width, blocks, block_size, max_rows):
    rng = np.random.default_rng(seqs * 7 + width)
    st = fresh(rng, seqs, width, blocks)
    d = {k: dev(v) for k, v in st.items()}
    length = np.zeros(seqs, np.int64)
    seen = set()
    for k in range(6):
        n_new = rng.integers(0, max(2, 2 * max_rows // seqs), seqs)
        if k % 3 == 2:                                   # some sequences are over
            gone = rng.random(seqs) < 0.4
            length[gone], n_new[gone] = 0, 0
        if k == 4:                                       # and some calls are wrong
            length[rng.random(seqs) < 0.1] = -5
            n_new[rng.random(seqs) < 0.1] = -1
            n_new[rng.random(seqs) < 0.1] = 2 ** 31 - 1
        want = check_step(st, d, length, n_new, block_size, max_rows)
        seen |= set(want["status"].tolist())
        ok = want["status"] == 0
        length = np.where(ok, length + (n_new * rng.random(seqs)).astype(np.int64), length)
        length = np.clip(length, 0, width * block_size)
        # what is owned and what is free are the blocks, each once
        have = np.concatenate([want["table"][s, : want["owned"][s]] for s in range(seqs)] + [want["free_ids"][: want["free_count"][0]]])
        assert np.array_equal(np.sort(have), np.arange(blocks))
    assert 0 in seen and (seqs < 40 or 2 in seen)  # (refusals, status 1, come in most of the cases and in the tight pool below)


def test_tight_pool_takes_blocks_given_back_in_the_same_step():
    rng = np.random.default_rng(3)
    st = fresh(rng, 4, 8, 10)
    d = {k: dev(v) for k, v in st.items()}
    check_step(st, d, np.zeros(4, np.int64), np.array([64, 64, 32, 0]), 16, 200)      # all ten blocks are out
    w = check_step(st, d, np.array([0, 64, 32, 0]), np.array([0, 1, 0, 60]), 16, 200)  # 4 come back, 1 + 4 are wanted
    assert w["status"].tolist() == [0, 0, 0, 1] and w["free_count"][0] == 3
    w = check_step(st, d, np.array([0, 65, 32, 0]), np.array([0, 1, 0, 48]), 16, 200)
    assert w["status"].tolist() == [0, 0, 0, 0] and w["free_count"][0] == 0


def test_sizes_of_zero_and_long_caches():
    from whirl_llm_b200 import api
    e = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    r = api.block_tables_step(e(0), e(0), e(0, 4), e(0), e(5), e(1), block_size=16, max_rows=7)
    assert r.slot.tolist() == [-1] * 7 and r.seq.tolist() == [-1] * 7 and r.row0.tolist() == [0]
    r = api.block_tables_step(e(3), e(3), e(3, 0), e(3), e(0), e(1), block_size=16, max_rows=0)
    assert r.status.tolist() == [0, 0, 0] and r.row0.tolist() == [0, 0, 0, 0]
    # slots pass 32 bits: block ids near 2^28 with 4096 tokens a block; lengths near 2^31
    t, own, ids, cnt = e(2, 600000), e(2), e(4), e(1)
    ids.copy_(torch.tensor([1, 2, 3, 2 ** 28 + 5]))
    cnt.fill_(4)
    r = api.block_tables_step(torch.tensor([0, 0], dtype=torch.int32, device="cuda"), torch.tensor([3, 2], dtype=torch.int32, device="cuda"), t, own,
                              ids, cnt, block_size=4096, max_rows=5)
    assert r.slot.tolist() == [(2 ** 28 + 5) * 4096, (2 ** 28 + 5) * 4096 + 1, (2 ** 28 + 5) * 4096 + 2, 3 * 4096, 3 * 4096 + 1]
    own[1] = 2 ** 31 // 4096 - 1
    t[1, 2 ** 31 // 4096 - 2] = 77
    last = (2 ** 31 // 4096 - 1) * 4096
    r = api.block_tables_step(torch.tensor([3, last - 2], dtype=torch.int32, device="cuda"), torch.tensor([0, 2], dtype=torch.int32, device="cuda"), t,
                              own, ids, cnt, block_size=4096, max_rows=5)
    assert r.slot.tolist()[:2] == [77 * 4096 + 4094, 77 * 4096 + 4095] and r.position.tolist()[:2] == [last - 2, last - 1]


def test_step_in_a_graph_and_given_outputs():
    from whirl_llm_b200 import api
    rng = np.random.default_rng(8)
    seqs, width, blocks, bs, mr = 50, 40, 1500, 16, 300
    st = fresh(rng, seqs, width, blocks)
    d = {k: dev(v) for k, v in st.items()}
    length, n_new = dev(np.zeros(seqs, np.int32)), dev(np.zeros(seqs, np.int32))
    out = api.StepRows(torch.empty(mr, dtype=torch.int64, device="cuda"), *[torch.empty(k, dtype=torch.int32, device="cuda") for k in (mr, mr, seqs + 1, seqs)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        api.block_tables_step(length, n_new, **d, block_size=bs, max_rows=mr, rows=out)
    ln = np.zeros(seqs, np.int64)
    for k in range(4):
        nn = rng.integers(0, 9, seqs)
        want = ref.step(ln, nn, **st, block_size=bs, max_rows=mr)
        length.copy_(dev(ln.astype(np.int32)))
        n_new.copy_(dev(nn.astype(np.int32)))
        g.replay()
        torch.cuda.synchronize()
        for name, v in dict(slot=out.slot, position=out.position, seq=out.seq, row0=out.row0, status=out.status, **d).items():
            assert np.array_equal(v.cpu().numpy(), want[name]), (k, name)
        for name in st:
            st[name] = want[name]
        ln = np.where(want["status"] == 0, ln + nn, ln)
    with pytest.raises(TypeError):
        api.block_tables_step(length, n_new, **d, block_size=bs, max_rows=mr + 1, rows=out)


def test_decode_then_train():
    """Speculative decoding of a few sequences with every per-step decision on the device - rows and slots, sampling, acceptance - and
    then the losses on what was sampled."""
    from whirl_llm_b200 import api
    rng = np.random.default_rng(21)
    seqs, D, V, bs, width, blocks = 6, 4, 4096, 16, 8, 60
    g = torch.Generator(device="cuda").manual_seed(4)
    embed = torch.randn((V, 64), device="cuda", generator=g)
    head = torch.randn((64, V), device="cuda", generator=g) * 0.3
    st = fresh(rng, seqs, width, blocks)
    d = {k: dev(v) for k, v in st.items()}
    cache = torch.full((blocks * bs,), -1, dtype=torch.int64, device="cuda")   # the token that each slot holds
    length = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    nxt = torch.arange(seqs, dtype=torch.int32, device="cuda") + 3
    text = [[int(t)] for t in nxt.tolist()]
    rows_x, rows_tok, rows_seq = [], [], []
    max_rows = seqs * (D + 1) + 2
    nd = torch.full((seqs,), D, dtype=torch.int32, device="cuda")
    for k in range(7):
        r = api.block_tables_step(length, nd + 1, **d, block_size=bs, max_rows=max_rows)
        drafts = torch.randint(0, V, (seqs, D), device="cuda", generator=g).to(torch.int32)
        drafts[:, 0] = torch.where(torch.arange(seqs, device="cuda") % 2 == 0, (embed[nxt.long()] @ head).argmax(1).to(torch.int32), drafts[:, 0])
        live = r.slot >= 0
        off = torch.arange(max_rows, device="cuda") - r.row0[r.seq.clamp_min(0).long()]
        fed = torch.cat([nxt[:, None], drafts], 1)[r.seq.clamp_min(0).long(), off.clamp(0, D).long()]
        cache[r.slot[live]] = fed[live].long()
        logits = embed[fed.long()] @ head
        greedy = torch.ones(max_rows, dtype=torch.uint8, device="cuda")
        tok = api.sample_rows(logits, api.RowParams(greedy=greedy)).token
        acc, chosen = api.accept_tokens(tok, drafts, nd, r.row0[:-1].contiguous())
        keep = live & (off <= acc[r.seq.clamp_min(0).long()])
        rows_x.append(logits[keep])
        rows_tok.append(tok[keep])
        rows_seq.append(r.seq[keep])
        for s in range(seqs):
            text[s] += drafts[s, : int(acc[s])].tolist() + [int(chosen[s])]
        length = length + acc + 1
        nxt = chosen
        # the cache holds every sequence's text where its table says
        table, ln = d["table"].cpu().numpy(), length.cpu().numpy()
        for s in range(seqs):
            p = np.arange(ln[s])
            assert cache.cpu().numpy()[table[s, p // bs].astype(np.int64) * bs + p % bs].tolist() == text[s][:-1][: ln[s]]
    x, token, seq = torch.cat(rows_x), torch.cat(rows_tok), torch.cat(rows_seq)
    order = torch.argsort(seq.long(), stable=True)
    x, token, seq = x[order].contiguous(), token[order].contiguous(), seq[order]
    start = torch.searchsorted(seq.contiguous(), torch.arange(seqs + 1, dtype=torch.int32, device="cuda")).to(torch.int32)
    scored = api.token_logprobs(x, token, want_entropy=True)
    assert torch.isfinite(scored.logp).all() and x.shape[0] == sum(len(t) for t in text) - seqs
    adv = torch.randn(x.shape[0], device="cuda", generator=g)
    p = api.policy_loss(x, token, adv, old_logp=scored.logp, ref_logp=scored.logp, seq_start=start, mean=api.MEAN_SEQS, kl_coef=0.1)
    assert (p.logp - scored.logp).abs().max() < 1e-5 and p.kl.abs().max() < 1e-9
    counts = (start[1:] - start[:-1]).double()
    want = -(adv.double() / counts[seq.long()] / seqs).sum()      # every ratio is 1
    assert abs(p.loss.double() - want) < 1e-5
    q = api.token_logprobs_grad(x, token, scored.stats, p.g_logp)
    assert (q - p.dx).abs().max() < 1e-6
    pref = api.preference_loss(x, token, start, ref_logp=scored.logp, beta=0.5)
    assert abs(pref.loss.item() - np.log(2)) < 1e-5               # the reference is the model itself
    fb = api.token_logprobs_grad(x, token, pref.stats, pref.g_logp)
    assert (fb - pref.dx).abs().max() < 1e-6
