"""Refusals of the loss and block-table entry points at sizes and addresses that the kernels do not take.  No device is needed."""
import ctypes as C

import pytest

P = 0x1000  # an address that no refused call touches


def status(fn, *args):
    from whirl_llm_b200 import api
    s = getattr(api.lib, fn)(*args)
    return s, api.lib.whirl_last_error().decode()


def policy(rows=4, x=P, ws=P, ws_bytes=1 << 40, out=None, **kw):
    from whirl_llm_b200 import api
    p = dict(token=P, adv=P, seqs=0, mean=1, inv_t=1.0, clip_low=0.2, clip_high=0.2)
    p.update(kw)
    o = dict(loss=P)
    o.update(out or {})
    return status("whirl_policy_loss", x, 0, rows, 100, 100, C.byref(api.PolicyParams(**p)), C.byref(api.PolicyOut(**o)), ws, ws_bytes, None)


def preference(rows=4, out=None, **kw):
    from whirl_llm_b200 import api
    p = dict(token=P, seq_start=P, pairs=2, kind=0, inv_t=1.0, beta=0.1)
    p.update(kw)
    o = dict(loss=P)
    o.update(out or {})
    return status("whirl_preference_loss", P, 0, rows, 100, 100, C.byref(api.PreferenceParams(**p)), C.byref(api.PreferenceOut(**o)), P, 1 << 40, None)


def test_more_rows_or_sequences_than_a_loop_counter_holds():
    """The kernels' loops over rows step past the last one: from 2^31 - 8192 rows on an int would wrap."""
    for rows in (2 ** 30 + 1, 2 ** 31 - 1):
        assert status("whirl_token_logprobs", P, 0, rows, 1, 1, P, 1.0, None, P, P, None, None)[0] == 4
        assert status("whirl_token_logprobs_grad", P, 0, rows, 1, 1, P, 1.0, None, P, None, P, None, P, 1, None)[0] == 4
        assert policy(rows)[0] == 4 and preference(rows)[0] == 4
        assert policy(mean=2, seqs=rows, seq_start=P)[0] == 4


def test_binding_refuses_what_a_c_int_would_cut():
    from whirl_llm_b200 import api
    assert api._i32(2 ** 31 - 1, "n") == 2 ** 31 - 1
    for v in (2 ** 31, 2 ** 32 + 16, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            api._i32(v, "block_size")


def test_arrays_not_aligned_to_their_type():
    """A load or store at such an address is a fault of the device; every array is looked at."""
    from whirl_llm_b200 import api
    ok = [P, 0, 4, 100, 100, P, 1.0, P, P, P, P, None]
    for i in (0, 5, 7, 8, 9, 10):
        a = list(ok)
        a[i] = P + 2
        s, msg = status("whirl_token_logprobs", *a)
        assert s == 1 and "aligned" in msg, i
    ok = [P, 0, 4, 100, 100, P, 1.0, P, P, P, P, P, P + 100000, 100, None]
    for i in (0, 5, 7, 8, 9, 10, 11, 12):
        a = list(ok)
        a[i] += 2
        s, msg = status("whirl_token_logprobs_grad", *a)
        assert s == 1 and "aligned" in msg, i
    for k in ("token", "adv", "old_logp", "ref_logp", "weight", "inv_t_rows"):
        assert "aligned" in policy(**{k: P + 1})[1], k
    assert "aligned" in policy(mean=2, seqs=1, seq_start=P + 2)[1]
    for k in ("loss", "logp", "stats", "entropy", "kl", "row_loss", "g_logp", "row_scale"):
        assert "aligned" in policy(out={k: P + 2})[1], k
    assert "aligned" in policy(out=dict(dx=P + 100002, ld_dx=100))[1]
    for k in ("token", "seq_start", "ref_logp", "weight", "inv_t_rows"):
        assert "aligned" in preference(**{k: P + 2})[1], k
    for k in ("loss", "pair_loss", "reward", "logp", "stats", "g_logp"):
        assert "aligned" in preference(out={k: P + 2})[1], k

    def blocks(length=P, n_new=P, **kw):
        t = dict(table=P, owned=P, free_ids=P, free_count=P, seqs=4, max_blocks=8, num_blocks=16, block_size=16)
        o = dict(slot=P, position=P, seq=P, row0=P, status=P, max_rows=32)
        for k, v in kw.items():
            (t if k in t else o)[k] = v
        return status("whirl_block_tables_step", length, n_new, C.byref(api.BlockTables(**t)), C.byref(api.StepRowsOut(**o)), P, 1 << 40, None)
    for k in ("length", "n_new", "table", "owned", "free_ids", "free_count", "position", "seq", "row0", "status"):
        s, msg = blocks(**{k: P + 2})
        assert s == 1 and "aligned" in msg, k
    assert "aligned" in blocks(slot=P + 4)[1]


def test_dx_beside_x_in_one_buffer():
    """Columns of one buffer do not overlap; one element in common does."""
    def grad(x, dx, ld=200, ld_dx=200, n=100, rows=4):
        return status("whirl_token_logprobs_grad", x, 0, rows, n, ld, P, 1.0, None, P, None, P, None, dx, ld_dx, None)
    for x, dx in ((P, P + 400), (P + 400, P), (P, P + 400 + 800), (P + 400, P + 800)):
        s, msg = grad(x, dx)
        assert "overlaps" not in msg or s != 1, (x, dx)          # (no device here: the launch itself fails)
    for x, dx in ((P, P + 396), (P + 396, P), (P, P + 404), (P, P + 800), (P, P + 4), (P + 4, P)):
        s, msg = grad(x, dx)
        assert s == 1 and "overlaps" in msg, (x, dx)
    assert grad(P, P + 400, ld_dx=201)[0] == 1                   # (rows drift into one another)
