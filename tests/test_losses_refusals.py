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
