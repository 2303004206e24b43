"""What the binding of the losses and block tables takes and refuses, and how it stands with autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_sizes_that_a_c_int_would_cut():
    from whirl_llm_b200 import api
    e = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="block_size"):
        api.block_tables_step(e(1), e(1), e(1, 4), e(1), e(5), e(1), block_size=2 ** 32 + 16, max_rows=7)
    with pytest.raises(ValueError, match="max_rows"):
        api.block_tables_step(e(1), e(1), e(1, 4), e(1), e(5), e(1), block_size=16, max_rows=2 ** 32 + 7)


@pytest.mark.parametrize("n,dtype", [(1003, torch.float32), (1000, torch.bfloat16), (40002, torch.float32), (40000, torch.bfloat16)])
def test_dx_beside_x_in_one_buffer(n, dtype):
    from whirl_llm_b200 import api
    rows = 50
    g = torch.Generator(device="cuda").manual_seed(n)
    buf = torch.randn((rows, 2 * n + 8), device="cuda", generator=g).to(dtype)
    x, dx, rest = buf[:, :n], buf[:, n + 8:], buf[:, n: n + 8].clone()
    token = torch.randint(0, n, (rows,), device="cuda", generator=g, dtype=torch.int32)
    adv = torch.randn(rows, device="cuda", generator=g)
    x0 = x.clone()
    want = api.policy_loss(x, token, adv).dx
    r = api.policy_loss(x, token, adv, dx=dx)
    assert torch.equal(r.dx, want) and torch.equal(x, x0) and torch.equal(buf[:, n: n + 8], rest)
    s = api.token_logprobs(x, token)
    want = api.token_logprobs_grad(x, token, s.stats, adv)
    assert torch.equal(api.token_logprobs_grad(x, token, s.stats, adv, dx=dx), want) and torch.equal(x, x0) and torch.equal(buf[:, n: n + 8], rest)
    with pytest.raises(api.WhirlError, match="overlaps"):
        api.policy_loss(x, token, adv, dx=buf[:, n - 1: 2 * n - 1])


def test_gradient_of_rows_far_apart_takes_no_more_than_its_rows():
    """The last position of every sequence of a batch: rows a whole sequence of logits apart."""
    from whirl_llm_b200 import api
    for n in (5000, 5003):
        x = torch.randn((6, 100, n), device="cuda")[:, -1]
        token = torch.arange(6, device="cuda", dtype=torch.int32)
        adv = torch.ones(6, device="cuda")
        s = api.token_logprobs(x, token)
        for dx in (api.policy_loss(x, token, adv).dx, api.token_logprobs_grad(x, token, s.stats, -adv / 6),
                   api.preference_loss(x, token, torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")).dx):
            assert dx.shape == x.shape and dx.untyped_storage().nbytes() <= 4 * 6 * (n + 4)
        assert torch.equal(api.policy_loss(x, token, adv).dx, api.policy_loss(x, token, adv, dx=torch.empty_like(x)).dx)


def test_gradient_in_place_is_seen_by_autograd():
    """A graph that kept the logits for its own backward pass must not use what dx = x put there."""
    from whirl_llm_b200 import api
    n = 2000
    token = torch.arange(8, device="cuda", dtype=torch.int32)
    adv = torch.ones(8, device="cuda")
    starts = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")

    def grads(y):
        d = y.detach()
        s = api.token_logprobs(d, token)
        return (lambda dx: api.policy_loss(d, token, adv, dx=dx).dx, lambda dx: api.preference_loss(d, token, starts, dx=dx).dx,
                lambda dx: api.token_logprobs_grad(d, token, s.stats, adv, dx=dx))
    for k in range(3):
        w = torch.randn((8, n), device="cuda", requires_grad=True)
        y = torch.tanh(w)                       # tanh keeps its result
        dx = grads(y)[k](y.detach())
        with pytest.raises(RuntimeError, match="inplace operation"):
            y.backward(dx)
        w = torch.randn((8, n), device="cuda", requires_grad=True)
        y = w * 2.0                             # a product by a number keeps nothing
        want = grads(y)[k](None).clone()
        y.backward(grads(y)[k](y.detach()))
        assert torch.equal(w.grad, 2.0 * want)
        out = torch.empty_like(y)
        before = out._version
        grads(torch.tanh(w))[k](out)
        assert out._version > before
