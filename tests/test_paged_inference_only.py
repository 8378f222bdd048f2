"""The paged cache and attention have no backward pass: an operand that a gradient is asked of is refused (on the host model)."""
import pytest
import torch

from tests.hostmodel.model import in_child


@in_child
def test_operands_that_require_a_gradient_are_refused():
    from tests.hostmodel.backend import python_api_on_hostmodel

    with python_api_on_hostmodel():
        import comp_inference_amd as ci

        cache = ci.PagedKVCache(2, 32, 2, 64, device="cpu")
        table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
        x, q = torch.ones(1, 2, 64, dtype=torch.bfloat16), torch.ones(1, 4, 64, dtype=torch.bfloat16)
        wants = lambda t: t.clone().requires_grad_()  # noqa: E731
        calls = [lambda: ci.paged_kv_append(cache, wants(x), x, table, lens), lambda: ci.paged_kv_append(cache, x, wants(x), table, lens),
                 lambda: ci.paged_kv_append(cache, x, x, table, lens, q=wants(q)), lambda: ci.paged_attention(wants(q), cache, table, lens),
                 lambda: ci.paged_attention(wants(q) * 2, cache, table, lens)]
        for call in calls:
            with pytest.raises(RuntimeError, match="gradient"):
                call()
            with torch.no_grad():
                call()
            with torch.inference_mode():
                call()
        assert not ci.paged_attention(q, cache, table, lens).requires_grad
