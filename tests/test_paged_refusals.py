"""What the paged cache and the attention over it refuse, on the CPU: through the C ABI (before any device is asked for
anything) and through the Python operators (on the host model of the library)."""
import ctypes as C

import pytest
import torch

from tests.hostmodel.model import in_child


class _Args:
    """Arguments a C caller would give, with pointers that are never followed: every call here is refused first."""

    def __init__(self):
        from comp_inference_amd import attention_hip as A

        self.cache = A._Cache(0x1000, 1 << 30, 8, 64, 2, 128, 0)
        self.batch = A._Batch(0x1000, 4, 4, 0x1000, 0x1000, 2, 10)
        self.k, self.v, self.q, self.out = (A._Rows(0x1000, 1024, 128) for _ in range(4))
        self.q_heads, self.rotary, self.rotary_rows, self.rotary_dim = 4, 0x1000, 100, 128
        self.scale, self.window, self.sinks, self.workspace, self.workspace_bytes = 0.1, 0, 0, 0x1000, 1 << 30
        self.max_query_len = self.max_seq_len = 0

    def append(self, lib):
        r = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return lib.ci_paged_kv_append(r(self.cache), r(self.batch), r(self.k), r(self.v), r(self.q), r(self.out), self.q_heads,
                                      C.c_void_p(self.rotary), self.rotary_rows, self.rotary_dim, None)

    def read(self, lib):
        r = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return lib.ci_paged_kv_read(r(self.cache), r(self.batch), r(self.k), r(self.v), None)

    def attend(self, lib):
        r = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return lib.ci_paged_attention(r(self.cache), r(self.batch), r(self.q), r(self.out), None, C.c_int64(4), self.q_heads,
                                      C.c_float(self.scale), self.window, self.sinks, self.max_query_len, self.max_seq_len,
                                      C.c_void_p(self.workspace), C.c_size_t(self.workspace_bytes), None)


COMMON = {
    "no_cache": (lambda a: setattr(a, "cache", None), b"null cache"),
    "no_batch": (lambda a: setattr(a, "batch", None), b"null batch"),
    "kind": (lambda a: setattr(a.cache, "kind", 2), b"kind"),
    "head_dim": (lambda a: setattr(a.cache, "head_dim", 96), b"head_dim"),
    "page_size": (lambda a: setattr(a.cache, "page_size", 48), b"page_size"),
    "page_size_small": (lambda a: setattr(a.cache, "page_size", 16), b"page_size"),
    "no_pages": (lambda a: setattr(a.cache, "num_pages", 0), b"num_pages"),
    "no_heads": (lambda a: setattr(a.cache, "kv_heads", 0), b"kv_heads"),
    "short_data": (lambda a: setattr(a.cache, "data_bytes", 8 * 64 * 2 * 128 * 4 - 1), b"holds"),
    "null_data": (lambda a: setattr(a.cache, "d_data", None), b"aligned"),
    "odd_data": (lambda a: setattr(a.cache, "d_data", 0x1008), b"aligned"),
    "no_table": (lambda a: setattr(a.batch, "d_block_table", None), b"block table"),
    "no_lens": (lambda a: setattr(a.batch, "d_seq_lens", None), b"lengths"),
    "no_columns": (lambda a: setattr(a.batch, "table_width", 0), b"columns"),
    "overlapping_rows": (lambda a: setattr(a.batch, "table_stride", 3), b"overlap"),
    "long_table": (lambda a: (setattr(a.batch, "table_width", 1 << 25), setattr(a.batch, "table_stride", 1 << 25)), b"2^30"),
    "rows_without_offsets": (lambda a: setattr(a.batch, "d_query_start", None), b"query_start"),
    "many_rows": (lambda a: setattr(a.batch, "num_tokens", 1 << 30), b"2^30"),
}
ROWS = {
    "null": lambda r: setattr(r, "d_data", None),
    "unaligned": lambda r: setattr(r, "d_data", 0x1008),
    "row_stride": lambda r: setattr(r, "row_stride", 1020),
    "head_stride": lambda r: setattr(r, "head_stride", 129),
    "backwards": lambda r: setattr(r, "row_stride", -1024),
}


@pytest.mark.parametrize("case", sorted(COMMON))
@pytest.mark.parametrize("entry", ["append", "read", "attend"])
def test_every_entry_point_checks_cache_and_batch(case, entry):
    from comp_inference_amd import _lib

    lib = _lib.lib()
    a = _Args()
    change, said = COMMON[case]
    change(a)
    assert getattr(a, entry)(lib) == 1
    assert said in lib.ci_last_error(), lib.ci_last_error()


@pytest.mark.parametrize("case", sorted(ROWS))
@pytest.mark.parametrize("entry,operands", [("append", "kvq"), ("append", ("out",)), ("read", "kv"), ("attend", ("q", "out"))])
def test_rows_are_checked(case, entry, operands):
    from comp_inference_amd import _lib

    lib = _lib.lib()
    for name in operands:
        a = _Args()
        ROWS[case](getattr(a, name))
        assert getattr(a, entry)(lib) == 1
        assert b"aligned" in lib.ci_last_error()


@pytest.mark.parametrize("entry,field,value,code,said", [
    ("append", "k", None, 1, b"null keys"), ("append", "out", None, 1, b"go together"), ("append", "q", None, 1, b"go together"),
    ("append", "q_heads", 0, 1, b"q_heads"), ("append", "rotary_dim", 24, 1, b"rotary_dim"), ("append", "rotary_dim", 0, 1, b"rotary_dim"),
    ("append", "rotary_dim", 144, 1, b"rotary_dim"), ("append", "rotary_rows", 0, 1, b"rows"), ("append", "rotary", 0x1004, 1, b"aligned"),
    ("read", "v", None, 1, b"null keys"),
    ("attend", "q", None, 1, b"null q"), ("attend", "out", None, 1, b"null q"), ("attend", "q_heads", 3, 1, b"q_heads"),
    ("attend", "q_heads", 0, 1, b"q_heads"), ("attend", "window", -1, 1, b"window"), ("attend", "sinks", -1, 1, b"window"),
    ("attend", "scale", 0.0, 1, b"scale"), ("attend", "scale", -0.1, 1, b"scale"), ("attend", "scale", float("nan"), 1, b"scale"),
    ("attend", "scale", float("inf"), 1, b"scale")])
def test_arguments_of_each_entry_point(entry, field, value, code, said):
    from comp_inference_amd import _lib

    lib = _lib.lib()
    a = _Args()
    setattr(a, field, value)
    assert getattr(a, entry)(lib) == code
    assert said in lib.ci_last_error(), lib.ci_last_error()


def _placed(at, row=1024, head=128):
    from comp_inference_amd import attention_hip as A

    return A._Rows(0x100000 + 2 * at, row, head)


@pytest.mark.parametrize("entry,change,refused", [
    ("attend", dict(q=_placed(0), out=_placed(0)), True),                         # in place
    ("attend", dict(q=_placed(0), out=_placed(1024)), True),                      # a row further
    ("attend", dict(q=_placed(9 * 1024), out=_placed(0)), True),                  # the last row
    ("attend", dict(q=_placed(9 * 1024 + 512), out=_placed(0, 1024)), False),     # in the last row's gap
    ("attend", dict(q=_placed(0), out=_placed(512)), False),                      # heads 4..7 of rows of eight
    ("attend", dict(q=_placed(512), out=_placed(0)), False),
    ("attend", dict(q=_placed(0), out=_placed(504)), True),
    ("attend", dict(q=_placed(0, 1536, 384), out=_placed(128, 1536, 384)), False),  # [tokens, heads, 3, dim]
    ("attend", dict(q=_placed(0, 1536, 384), out=_placed(8, 1536, 384)), True),
    ("attend", dict(q=_placed(0, 128, 1280), out=_placed(5120, 128, 1280)), False),  # heads outermost, one after the other
    ("attend", dict(q=_placed(0, 128, 1280), out=_placed(5112, 128, 1280)), True),
    ("append", dict(q=_placed(0), out=_placed(8), k=_placed(1 << 20), v=_placed(2 << 20)), True),
    ("append", dict(q=_placed(0), out=_placed(0, 1024, 136), k=_placed(1 << 20), v=_placed(2 << 20)), True),
    ("append", dict(q=_placed(0), out=_placed(3 << 20), k=_placed(3 << 20), v=_placed(2 << 20)), True),
    ("append", dict(q=_placed(0), out=_placed(3 << 20), k=_placed(1 << 20), v=_placed((3 << 20) + 384)), True),
    ("append", dict(q=_placed(0), out=_placed(0), k=_placed(512), v=_placed(768)), False),  # one buffer, queries in place
    ("read", dict(k=_placed(0), v=_placed(128)), True),
    ("read", dict(k=_placed(0), v=_placed(256)), False)])
def test_outputs_do_not_lie_on_other_operands(entry, change, refused):
    """(What is let through ends a check later, for want of a device here or of a workspace: the pointers are never followed.)"""
    from comp_inference_amd import _lib

    if not refused and torch.cuda.is_available():
        pytest.skip("a call that is not refused would run")
    lib = _lib.lib()
    a = _Args()
    a.workspace = None
    for name, rows in change.items():
        setattr(a, name, rows)
    assert getattr(a, entry)(lib) != 0
    assert (b"memory" in lib.ci_last_error()) == refused, lib.ci_last_error()


def test_more_work_than_a_list_counts_is_refused():
    from comp_inference_amd import _lib

    lib = _lib.lib()
    a = _Args()
    a.batch.num_tokens, a.batch.table_width, a.batch.table_stride = 1 << 24, 1 << 18, 1 << 18
    a.q, a.out = _placed(0), _placed(1 << 40)
    rc = a.attend(lib)
    assert rc != 0 and (b"several" in lib.ci_last_error() or not torch.cuda.is_available()), lib.ci_last_error()


def test_sizes_of_a_cache():
    from comp_inference_amd import attention_hip as A

    assert A._cache_bytes(10, 64, 8, 128, 0) == 10 * 64 * 8 * 128 * 2 * 2
    assert A._cache_bytes(10, 64, 8, 128, 1) == 10 * 64 * 8 * (128 + 8)
    assert A._cache_bytes(3, 32, 1, 64, 1) == 3 * 32 * (64 + 8)
    for bad in ((0, 64, 8, 128, 0), (1, 40, 8, 128, 0), (1, 8192, 8, 128, 0), (1, 64, 0, 128, 0), (1, 64, 8, 80, 0), (1, 64, 8, 128, 2)):
        assert A._cache_bytes(*bad) == 0


@in_child
def test_the_python_operators_refuse():
    from tests.hostmodel.backend import python_api_on_hostmodel

    with python_api_on_hostmodel():
        import comp_inference_amd as ci

        for bad in (dict(kind="fp8"), dict(page_size=48), dict(page_size=0), dict(head_dim=96), dict(kv_heads=0), dict(num_pages=-1)):
            with pytest.raises(ValueError):
                ci.PagedKVCache(**{**dict(num_pages=4, page_size=32, kv_heads=2, head_dim=64, device="cpu"), **bad})
        cache = ci.PagedKVCache(4, 32, 2, 64, device="cpu")
        x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
        q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
        table = torch.zeros(3, 2, dtype=torch.int32)
        lens = torch.ones(3, dtype=torch.int32)
        start = torch.arange(4, dtype=torch.int32)
        rot = ci.rotary_table(8, 64, device="cpu")
        good = dict(k=x, v=x, block_table=table, seq_lens=lens)
        ci.paged_kv_append(cache, **good)

        def refuse(error, said, fn, *args, **kw):
            with pytest.raises(error, match=said):
                fn(*args, **kw)

        for change, error, said in (
                (dict(k=x.half()), RuntimeError, "bfloat16"), (dict(v=x[:2]), ValueError, "shape"),
                (dict(k=torch.zeros(3, 2, 128, dtype=torch.bfloat16)), ValueError, "shape"),
                (dict(v=torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2]), RuntimeError, "stride"),
                (dict(k=torch.zeros(3, 2, 65, dtype=torch.bfloat16)[..., 1:]), RuntimeError, "stride"),
                (dict(block_table=table.long()), RuntimeError, "int32"), (dict(seq_lens=lens.long()), RuntimeError, "int32"),
                (dict(block_table=table[:2]), ValueError, "rows"), (dict(query_start=start[:3]), ValueError, "query_start"),
                (dict(seq_lens=lens[:2], block_table=table[:2]), ValueError, "query_start"),
                (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), RuntimeError, "contiguous"),
                (dict(q_out=q), ValueError, "without q"), (dict(q=q, q_out=q[:2]), ValueError, "shape"),
                (dict(rotary=rot.double()), RuntimeError, "float32"), (dict(rotary=rot[:, :24].contiguous()), ValueError, "multiple of 16"),
                (dict(rotary=rot[:, :32]), RuntimeError, "contiguous"),
                (dict(q=q, q_out=q[:1].expand(3, 4, 64)), RuntimeError, "overlap")):
            refuse(error, said, ci.paged_kv_append, cache, **{**good, **change})
        refuse(ValueError, "tokens", ci.paged_kv_read, cache, table, lens, start)
        refuse(ValueError, "query_start", ci.paged_kv_read, cache, table, lens, tokens=5)
        good = dict(q=q, cache=cache, block_table=table, seq_lens=lens)
        ci.paged_attention(**good)
        for change, error, said in (
                (dict(q=q[:, :3]), ValueError, "multiple"), (dict(q=q[:, :0]), ValueError, "multiple"),
                (dict(q=q.float()), RuntimeError, "bfloat16"), (dict(q=q[:2]), ValueError, "query_start"),
                (dict(out=q[:2]), ValueError, "shape"), (dict(out=q.float()), RuntimeError, "bfloat16"),
                (dict(out=q[:1].expand(3, 4, 64)), RuntimeError, "overlap"),
                (dict(window=-1), ValueError, "window"), (dict(sinks=-3), ValueError, "window"), (dict(scale=0.0), RuntimeError, "scale"),
                (dict(scale=float("nan")), RuntimeError, "scale"), (dict(window=1 << 31), ValueError, "window")):
            refuse(error, said, ci.paged_attention, **{**good, **change})
        with pytest.raises(ValueError):
            ci.rotary_table(4, 5, device="cpu")
        cache.data = cache.data.transpose(0, 1)
        refuse(RuntimeError, "contiguous", ci.paged_attention, **good)


def test_the_operators_refuse_cpu_tensors():
    import comp_inference_amd as ci

    cache = ci.PagedKVCache(2, 32, 1, 64, device="cpu")
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: ci.paged_kv_append(cache, x, x, table, lens), lambda: ci.paged_kv_read(cache, table, lens),
                 lambda: ci.paged_attention(x, cache, table, lens)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_the_rotary_table_is_exact_at_far_positions():
    import math

    import comp_inference_amd as ci

    t = ci.rotary_table(200001, 64, theta=500000.0, device="cpu")
    for p in (0, 1, 131071, 200000):
        for i in (0, 1, 17, 31):
            a = p * 500000.0 ** (-2.0 * i / 64)
            assert abs(float(t[p, i]) - math.cos(a)) < 1e-7 and abs(float(t[p, 32 + i]) - math.sin(a)) < 1e-7
