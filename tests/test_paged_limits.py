"""The paged cache at the ends of its range, on the host model: how much work one call of attention takes (the host's check that
32 bits count it, at its border; those calls get no further), and sequences of the greatest length."""
import ctypes as C

import numpy as np
import pytest

from tests.hostmodel.model import in_child
from tests.test_paged_refusals import _Args, _placed


@pytest.mark.parametrize("tokens,query_len,width", [
    # many rows: (2^25 / 256 + 2) tiles of 2 heads, so 0xFF000000 / 262148 = 16319 steps each, one for a page of 64 and two more
    (1 << 24, 0, 16317),
    # few rows, four to a tile: (2^17 / 4 + 2) tiles of 2 heads, so 0xFF000000 / 65540 = 65276 units of two pages, and two more
    (1 << 16, 1, 2 * 65274 + 1)])
@in_child
def test_more_work_than_a_list_counts_is_refused_at_the_border(tokens, query_len, width):
    from tests.hostmodel import build
    from tests.hostmodel.model import Model

    lib = Model(cus=256, lib_path=build.build()).lib
    for w, said in ((width, b"workspace"), (width + 1, b"several")):
        a = _Args()
        a.q, a.out = _placed(0), _placed(1 << 40)
        a.batch.num_tokens, a.batch.table_width, a.batch.table_stride = tokens, w, w
        a.max_query_len, a.workspace = query_len, None
        assert a.attend(lib) != 0
        assert said in lib.ci_last_error(), lib.ci_last_error()


@pytest.mark.parametrize("kind", [0, 1])
@in_child
def test_sequences_of_the_greatest_length(kind):
    """2^30 tokens, every page of the table the same one, under a window and in full view of the last rows' mask arithmetic: on
    the build with the compiler's undefined-behaviour checks, against plain sums."""
    from comp_inference_amd import attention_hip as A
    from tests.hostmodel import build
    from tests.hostmodel.model import Model
    from tests.test_hostmodel_paged import _bf16, _f64

    m = Model(cus=4, lib_path=build.build(undefined=True))
    L = m.lib
    L.ci_kv_cache_bytes.restype = C.c_uint64
    L.ci_paged_attention_workspace_bytes.restype = C.c_size_t
    rng = np.random.default_rng(kind)
    dim, page, length, window, sinks = 64, 4096, 1 << 30, 100, 5
    nbytes = L.ci_kv_cache_bytes(1, page, 1, dim, kind)
    data = m.dev(np.zeros(nbytes, np.uint8))
    cache = A._Cache(data.ptr, nbytes, 1, page, 1, dim, kind)
    table = m.dev(np.zeros((1, length // page), np.int32))
    rows = lambda d: C.byref(A._Rows(d.ptr, dim, dim))  # noqa: E731

    def batch(n, start=True, width=length // page, tokens=length):
        keep.append((m.dev(np.array([tokens], np.int32)), m.dev(np.array([0, n], np.int32))))
        return A._Batch(table.ptr, width, width, keep[-1][0].ptr, keep[-1][1].ptr if start else None, 1, n)

    keep = []
    k, v = (m.dev(_bf16(rng.standard_normal((page, 1, dim)))) for _ in range(2))
    whole = batch(page, width=1, tokens=page)
    m.call("ci_paged_kv_append", C.byref(cache), C.byref(whole), rows(k), rows(v), None, None, 0, None, 0, 0, None)
    # the last two tokens anew, at their positions near 2^30
    last = [m.dev(_bf16(rng.standard_normal((2, 1, dim)))) for _ in range(2)]
    m.call("ci_paged_kv_append", C.byref(cache), C.byref(batch(2)), rows(last[0]), rows(last[1]), None, None, 0, None, 0, 0, None)
    rk, rv = m.empty((page, 1, dim), np.uint16), m.empty((page, 1, dim), np.uint16)
    m.call("ci_paged_kv_read", C.byref(cache), C.byref(batch(page)), rows(rk), rows(rv), None)
    ks, vs = _f64(rk.get())[:, 0], _f64(rv.get())[:, 0]
    if kind == 0:
        assert np.array_equal(ks[-2:], _f64(last[0].get())[:, 0]) and np.array_equal(vs[:-2], _f64(v.get())[:-2, 0])
    for n, start, longest in ((1, False, 0), (3, True, 1), (300, True, 0), (700, True, 0)):
        q, out = m.dev(_bf16(rng.standard_normal((n, 1, dim)))), m.empty((n, 1, dim), np.uint16)
        b = batch(n, start)
        size = L.ci_paged_attention_workspace_bytes(C.byref(cache), C.byref(b), 1, window, sinks, longest, 0)
        ws = m.empty(max(size, 1), np.uint8)
        m.call("ci_paged_attention", C.byref(cache), C.byref(b), rows(q), rows(out), None, C.c_int64(1), 1, C.c_float(dim ** -0.5),
               window, sinks, longest, 0, ws.p if size else None, C.c_size_t(size), None)
        got = _f64(out.get())
        for i in {0, n // 2, n - 1}:
            p = length - n + i
            j = np.r_[0:sinks, p - window + 1:p + 1] % page
            s = ks[j] @ _f64(q.get())[i, 0] * dim ** -0.5
            w = np.exp(s - s.max())
            # (a rounding of each weight and of the result, 2^-8 each of sums of |v| around one; of each value read back in 4 bits)
            assert np.abs(got[i, 0] - w @ vs[j] / w.sum()).max() < 0.03, (n, i)
    status = C.c_uint32()
    assert L.ci_device_status(C.byref(status), None) == 0
    m.free_all()
