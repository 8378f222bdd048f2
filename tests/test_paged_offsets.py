"""Row offsets and lengths that no batch can have, in the paged cache's operators and attention: always reported, never
followed outside the arrays.  On the host model of the library, without a GPU."""
import ctypes as C

import numpy as np
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


@pytest.mark.parametrize("rows,lens", [
    # few rows, tiles of four: a sequence of length l is l - 192 units of 128 keys; 2^32 + 384 together
    (512, [1 << 30] * 4 + [512, 1024]),
    # many rows, four tiles of 256: 2^26 - 22 places, or 42; 2^32 + 272 together
    (1024, [1 << 30] * 64 + [1024] * 40)])
@in_child
def test_work_that_passes_32_bits_by_rows_that_several_sequences_claim(rows, lens):
    """Offsets 0, n, 0, n, ..: every second sequence claims all the rows.  Together their work, over lengths of 2^30, is a
    little more than 32 bits count; a sum that wraps around would have the join read parts that no workgroup wrote, far
    outside the workspace.  Nothing is done for such a batch, and it is reported."""
    from comp_inference_amd import attention_hip as A
    from tests.hostmodel.model import Model

    m = Model(cus=8)
    L = m.lib
    L.ci_kv_cache_bytes.restype = C.c_uint64
    L.ci_paged_attention_workspace_bytes.restype = C.c_size_t
    dim, page, width = 64, 4096, 1 << 18
    query_len = 1 if rows == 512 else rows
    seqs = 2 * len(lens) - 1
    table = np.zeros((seqs, width), np.int32)
    nbytes = L.ci_kv_cache_bytes(1, page, 1, dim, 0)
    data = m.dev(np.zeros(nbytes, np.uint8))
    cache = A._Cache(data.ptr, nbytes, 1, page, 1, dim, 0)
    dt, dl = m.dev(table), m.dev(np.array([x for l in lens for x in (l, 0)][:seqs], np.int32))
    start = m.dev(np.array([0, rows] * len(lens), np.int32))
    q, out = m.dev(np.zeros((rows, 1, dim), np.uint16)), m.dev(np.full((rows, 1, dim), 7, np.uint16))
    r = lambda d: C.byref(A._Rows(d.ptr, dim, dim))  # noqa: E731
    batch = A._Batch(dt.ptr, width, width, dl.ptr, start.ptr, seqs, rows)
    n = L.ci_paged_attention_workspace_bytes(C.byref(cache), C.byref(batch), 1, 0, 0, query_len, 0)
    assert n
    ws = m.empty(n, np.uint8)
    m.call("ci_paged_attention", C.byref(cache), C.byref(batch), r(q), r(out), None, C.c_int64(1), 1, C.c_float(0.125), 0, 0, query_len, 0,
           ws.p, C.c_size_t(n), None)
    assert (out.get() == 7).all()
    status = C.c_uint32()
    assert L.ci_device_status(C.byref(status), None) != 0 and status.value == 2
    m.free_all()
