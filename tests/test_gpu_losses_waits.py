"""The policy loss's bounded waits: thread blocks that share a row exchange its statistics, and a wait for them that runs out is reported.
It is made to run out on the host's request (the library's testing aid shortens the budget and leaves one exchange out); nothing
faults, traps or spins without a limit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n,dtype", [(3000, 2500, torch.float32), (1500, 20011, torch.float32), (900, 70000, torch.bfloat16), (40, 151936, torch.float32)])
@pytest.mark.parametrize("ent", [0.0, 0.1])
def test_wait_that_runs_out_is_reported(rows, n, dtype, ent):
    from whirl_llm_b200 import api
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.randn((rows, n), device="cuda", generator=g) * 3).to(dtype)
    token = torch.randint(0, n, (rows,), device="cuda", generator=g, dtype=torch.int32)
    weight = torch.ones(rows, device="cuda")
    weight[0] = 0.0                                   # (the exchange left out is the first cluster's first)
    x[5] = torch.finfo(dtype).min                     # a row that takes two exchanges
    call = lambda: api.policy_loss(x, token, torch.ones(rows, device="cuda"), weight=weight, mean=api.MEAN_SUM, ent_coef=ent)  # noqa: E731
    want = call()
    assert api.loss_check(want) == 0 and torch.isfinite(want.loss)
    api.test_waits(20000, True)                       # 20 ms a wait
    try:
        r = call()
        where = api.loss_check(r)
    finally:
        api.test_waits(0, False)
    assert where == 1 and torch.isnan(r.loss)
    lost = torch.isnan(r.logp)
    k = lost.nonzero()[:, 0]
    assert 0 < len(k) < rows and (len(k) == 1 or (k[1:] - k[:-1] == k[1] - k[0]).all()), k   # the first cluster's rows, every so many
    assert torch.isnan(r.dx[lost]).all() and torch.isnan(r.g_logp[lost]).all() and torch.isnan(r.row_loss[lost]).all()
    keep = ~lost
    assert (r.dx[0] == 0).all()
    for a, b in ((r.logp, want.logp), (r.dx, want.dx), (r.row_loss, want.row_loss), (r.stats, want.stats)):
        assert torch.equal(a[keep], b[keep])          # nobody else's rows are touched
    again = call()                                    # the next call, with the defaults back, is as before
    assert api.loss_check(again) == 0
    for a in ("loss", "logp", "dx", "row_loss"):
        assert torch.equal(getattr(again, a), getattr(want, a))


def test_loss_check_refusals():
    from whirl_llm_b200 import api
    assert api.lib.whirl_loss_check(None, 1 << 20, None, None) == 1
    assert api.lib.whirl_loss_check(0x1000, 8, None, None) == 3
    empty = api.policy_loss(torch.zeros((0, 9), device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, device="cuda"))
    assert api.loss_check(empty) == 0
