"""Row offsets and lengths that no batch can have, in the paged cache's operators and attention: always reported, never
followed outside the arrays.  On the host model of the library, without a GPU."""
import pytest
import torch

from tests.hostmodel.model import in_child


@in_child
def test_offsets_that_fall_and_lengths_of_sequences_without_new_tokens_are_reported():
    """A sequence that ends before it begins has no row, so no workgroup comes by to report it; nor one whose length is
    outside the table."""
    from tests.hostmodel.backend import python_api_on_hostmodel

    with python_api_on_hostmodel():
        import comp_inference_amd as ci

        cache = ci.PagedKVCache(4, 32, 2, 64, device="cpu")
        x, q = torch.zeros(8, 2, 64, dtype=torch.bfloat16), torch.zeros(8, 4, 64, dtype=torch.bfloat16)
        table = torch.arange(3, dtype=torch.int32)[:, None]

        def calls(lens, start):
            lens, start = (torch.tensor(t, dtype=torch.int32) for t in (lens, start))
            yield "append", lambda: ci.paged_kv_append(cache, x, x, table, lens, start)
            yield "read", lambda: ci.paged_kv_read(cache, table, lens, start, tokens=8)
            for bounds in (dict(max_query_len=2), dict(max_query_len=2, max_seq_len=8), dict(max_query_len=64, max_seq_len=8)):
                yield f"attention {bounds}", lambda: ci.paged_attention(q, cache, table, lens, start, **bounds)  # noqa: B023

        for name, call in calls([5, 5, 5], [0, 5, 5, 8]):
            call()
            assert ci.device_status() == 0, name
        for lens, start in (([5, 5, 5], [0, 5, 3, 8]), ([5, 33, 3], [0, 5, 5, 8]), ([5, -1, 3], [0, 5, 5, 8])):
            for name, call in calls(lens, start):
                call()
                with pytest.raises(RuntimeError, match="do not exist"):
                    ci.device_status()
                    raise AssertionError((name, lens, start))
                assert ci.device_status() == 0
