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
