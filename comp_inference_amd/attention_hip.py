"""A paged key/value cache and attention over it on the GPU: what stands between the compressed linears of a decoder.

The reference has no counterpart (its models run the attention of the library they come from); the kernels are HIP
(csrc/kv_cache.hip, csrc/attention.hip), the cache's order in memory is csrc/paged.h.  A batch is given by three int32
tensors on the device: `block_table` [B, P] (the pages of each sequence), `seq_lens` [B] (tokens, the new ones included)
and `query_start` [B + 1] (which rows of q / k / v belong to which sequence; None: one row each).  The kernels read them,
so a captured graph may be replayed with new contents.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib
from ._lib import check, lib, ptr

KINDS = {"bf16": 0, "int4": 1}


class _Cache(C.Structure):
    """ci_kv_cache (include/comp_inference_hip.h)."""
    _fields_ = [("d_data", C.c_void_p), ("data_bytes", C.c_uint64), ("num_pages", C.c_uint32), ("page_size", C.c_uint32),
                ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("kind", C.c_uint32)]


class _Batch(C.Structure):
    """ci_kv_batch."""
    _fields_ = [("d_block_table", C.c_void_p), ("table_stride", C.c_uint32), ("table_width", C.c_uint32),
                ("d_seq_lens", C.c_void_p), ("d_query_start", C.c_void_p), ("num_seqs", C.c_uint32),
                ("num_tokens", C.c_uint32)]


class _Rows(C.Structure):
    """ci_rows."""
    _fields_ = [("d_data", C.c_void_p), ("row_stride", C.c_int64), ("head_stride", C.c_int64)]


def _cache_bytes(num_pages, page_size, kv_heads, head_dim, kind) -> int:
    fn = lib().ci_kv_cache_bytes
    fn.restype = C.c_uint64
    return int(fn(num_pages, page_size, kv_heads, head_dim, kind))


class PagedKVCache:
    """Keys and values of one layer in pages of `page_size` tokens (a power of two from 32 to 4096) for `kv_heads` heads of
    64 or 128 channels.  `kind`: "bf16", or "int4": per token and head sixteen levels between the row's minimum and its
    maximum (a code of 4 bits each, and a bf16 pair step, low), 27 % of the bytes at 128 channels.  `data` is the memory:
    its contents are in the order attention reads them (`paged_kv_read` gives rows).  Pages are handed out by the caller:
    a sequence owns the pages it appends to, pages that are only read may be shared."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, kind: str = "bf16", device="cuda"):
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {sorted(KINDS)}, not {kind!r}")
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = map(int, (num_pages, page_size, kv_heads, head_dim))
        self.kind = kind
        shape = (self.num_pages, self.page_size, self.kv_heads, self.head_dim)
        nbytes = 0 if min(shape) < 1 or max(shape) >= 1 << 31 else _cache_bytes(*shape, KINDS[kind])
        if nbytes == 0:
            raise ValueError("a cache has 1 to 2^31 - 1 pages of 32 to 4096 tokens (a power of two), 1 to 1024 heads of 64 or "
                             f"128 channels; not {num_pages} pages of {page_size}, {kv_heads} heads of {head_dim}")
        blocks = self.page_size // 32
        dtype = torch.bfloat16 if kind == "bf16" else torch.uint8
        per = nbytes // (self.num_pages * self.kv_heads * blocks * dtype.itemsize)
        self.data = torch.zeros(self.num_pages, self.kv_heads, blocks, per, dtype=dtype, device=device)

        self._bound = None

    def _struct(self):
        """The C descriptor by reference; made again when `data` is another memory."""
        d = self.data
        at = (d.data_ptr(), d.nbytes)
        if self._bound is None or self._bound[0] != at or not d.is_contiguous():
            if not d.is_contiguous():
                raise RuntimeError("the cache's data must stay contiguous")
            c = _Cache(*at, self.num_pages, self.page_size, self.kv_heads, self.head_dim,
                       KINDS[self.kind])
            self._bound = (at, c, C.byref(c))
        return self._bound[2]

    # A copy (copy.deepcopy, pickling) has memory of its own: the descriptor is made again there.
    def __getstate__(self):
        return {**self.__dict__, "_bound": None}


def rotary_table(positions: int, rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """fp32 [positions, rotary_dim]: cosines, then sines, of position * theta^(-2 i / rotary_dim), i < rotary_dim / 2.
    Angles are formed in 64 bits (a far position's angle in 32 bits is off by more than a turn's thousandth)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    inverse = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inverse
    return torch.cat((angle.cos(), angle.sin()), dim=1).to(torch.float32).to(device)


def _no_gradient(*operands):
    """There is no backward pass: a result without one would cut the graph silently."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in operands):
        raise RuntimeError("the paged cache and attention are for inference: an operand requires a gradient "
                           "(call under torch.no_grad(), or detach it)")


def _elsewhere(name: str, t, cache: PagedKVCache):
    return RuntimeError(f"{name} is on {t.device}, the cache on {cache.data.device}")


# These checks run in front of every launch of a token loop: each asks a tensor for its properties once, all conditions in
# one test, and only a call that is refused finds out which one it was.

def _batch(cache: PagedKVCache, index: int, block_table, seq_lens, query_start, tokens: int):
    """ci_kv_batch by reference."""
    seqs, start = seq_lens.numel(), None
    ok = (block_table.dtype is torch.int32 and seq_lens.dtype is torch.int32 and block_table.dim() == 2
          and seq_lens.dim() == 1 and block_table.get_device() == index and seq_lens.get_device() == index
          and seq_lens.is_contiguous())
    if query_start is not None:
        ok = (ok and query_start.dtype is torch.int32 and query_start.dim() == 1 and query_start.get_device() == index
              and query_start.numel() == seqs + 1 and query_start.is_contiguous())
        start = query_start.data_ptr()
    if ok:
        (rows, width), (step, inner) = block_table.shape, block_table.stride()
        if rows == seqs and (start is not None or tokens == seqs) and (inner == 1 or width <= 1) and 0 <= step < 1 << 32:
            return C.byref(_Batch(block_table.data_ptr(), step if seqs > 1 else width, width, seq_lens.data_ptr(), start,
                                  seqs, tokens))
    for name, t, dim in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("query_start", query_start, 1)):
        if t is not None and (t.dtype is not torch.int32 or t.dim() != dim):
            raise RuntimeError(f"{name} must be a {dim}-D int32 tensor")
        if t is not None and t.get_device() != index:
            raise _elsewhere(name, t, cache)
    if block_table.shape[0] != seqs or (query_start is not None and query_start.numel() != seqs + 1):
        raise ValueError(f"block_table must have {seqs} rows and query_start {seqs + 1} entries for {seqs} sequences")
    if query_start is None and tokens != seqs:
        raise ValueError(f"without query_start there is one new token per sequence: {tokens} rows, {seqs} sequences")
    raise RuntimeError("seq_lens and query_start must be contiguous, and the rows of block_table")


def _rows(name: str, t: torch.Tensor, cache: PagedKVCache, index: int, heads: int | None, tokens: int | None):
    """ci_rows by reference of [tokens, heads, head_dim] in bf16 with unit stride inside a head."""
    if t.dtype is torch.bfloat16 and t.dim() == 3 and t.get_device() == index:
        (n, h, d), (row, head, inner), at = t.shape, t.stride(), t.data_ptr()
        if d == cache.head_dim and (heads is None or h == heads) and (tokens is None or n == tokens):
            if (inner == 1 and not (at & 15 or (row | head) & 7)) or n == 0 or h == 0:
                return C.byref(_Rows(at, row, head))
            raise RuntimeError(f"{name} must have unit stride inside a head, 16-byte aligned rows and strides that are multiples of 8")
        raise ValueError(f"{name} has shape {(n, h, d)}; the other operands ask for ({tokens}, {heads}, {cache.head_dim})")
    if t.dtype is not torch.bfloat16 or t.dim() != 3:
        raise RuntimeError(f"{name} must be a 3-D bfloat16 tensor [tokens, heads, head_dim]")
    raise _elsewhere(name, t, cache)


def _output(name: str, given, tokens: int, heads: int, cache: PagedKVCache) -> torch.Tensor:
    if given is None:
        return torch.empty((tokens, heads, cache.head_dim), dtype=torch.bfloat16, device=cache.data.device)
    if given.dim() == 3 and given.numel():
        # (the strides that are used must lead from one head to another place)
        steps = sorted((s, n) for s, n in zip(given.stride(), given.shape) if n > 1)
        if any(s < (steps[i - 1][0] * steps[i - 1][1] if i else 1) for i, (s, _) in enumerate(steps)):
            raise RuntimeError(f"{name} must not overlap itself")
    return given


def _here(index: int):
    """The context in which kernels of device `index` are launched (none where it is the current one already)."""
    return _NOTHING if torch.cuda.current_device() == index else torch.cuda.device(index)


_NOTHING = contextlib.nullcontext()


def paged_kv_append(cache: PagedKVCache, k, v, block_table, seq_lens, query_start=None, q=None, rotary=None, q_out=None):
    """Stores the keys and values [T, kv_heads, head_dim] (bf16, any row and head strides that are multiples of 8) of a
    batch's new tokens: the last ones of every sequence.  With `rotary` (a table as `rotary_table` makes; channels d and
    d + rotary_dim / 2 form a pair, the channels behind rotary_dim stay) keys and queries are turned by their position's
    angle first, in 64 bits, rounded to 32 bits and then to bf16.  `q` [T, heads, head_dim] is turned the same way
    into `q_out` (`q` itself, or memory of its own; made if not given), which is returned.  Rows behind the last sequence, and
    sequences of length 0, are left as they were.  Tokens, pages and table rows that do not exist are left out and
    reported by `device_status`.  No gradients: operands that require one are refused."""
    _lib.require_device(cache.data)
    _no_gradient(k, v, q)
    index, H = cache.data.get_device(), cache.kv_heads
    kr = _rows("k", k, cache, index, H, None)
    tokens = k.shape[0]
    vr = _rows("v", v, cache, index, H, tokens)
    b = _batch(cache, index, block_table, seq_lens, query_start, tokens)
    qr = orows = None
    heads = positions = turned = 0
    table = None
    if q is not None:
        qr = _rows("q", q, cache, index, None, tokens)
        heads = q.shape[1]
        q_out = _output("q_out", q_out, tokens, heads, cache)
        orows = _rows("q_out", q_out, cache, index, heads, tokens)
    elif q_out is not None:
        raise ValueError("q_out without q")
    if rotary is not None:
        if rotary.dtype is not torch.float32 or rotary.dim() != 2 or not rotary.is_contiguous():
            raise RuntimeError("rotary must be a contiguous 2-D float32 tensor [positions, rotary_dim]")
        if rotary.get_device() != index:
            raise _elsewhere("rotary", rotary, cache)
        positions, turned = rotary.shape
        if turned == 0 or turned % 16 or turned > cache.head_dim:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim, not {turned}")
        table = C.c_void_p(rotary.data_ptr())
    c = cache._struct()
    with _here(index):
        check(lib().ci_paged_kv_append(c, b, kr, vr, qr, orows, heads, table, positions, turned,
                                       _lib.stream_handle(cache.data.device)))
    return q_out


def paged_kv_read(cache: PagedKVCache, block_table, seq_lens, query_start=None, tokens=None, k_out=None, v_out=None):
    """(keys, values) [tokens, kv_heads, head_dim] in bf16 of the last tokens of every sequence, as the cache holds them:
    `query_start` cuts the rows as for `paged_kv_append`.  `tokens`: rows in all (needed with `query_start` unless the
    outputs are given; reading it from the device would wait for it)."""
    _lib.require_device(cache.data)
    index, H = cache.data.get_device(), cache.kv_heads
    if tokens is None:
        if query_start is not None and k_out is None:
            raise ValueError("tokens (the number of rows) is needed with query_start")
        tokens = seq_lens.numel() if query_start is None else k_out.shape[0]
    tokens = int(tokens)
    k_out, v_out = _output("k_out", k_out, tokens, H, cache), _output("v_out", v_out, tokens, H, cache)
    kr, vr = _rows("k_out", k_out, cache, index, H, tokens), _rows("v_out", v_out, cache, index, H, tokens)
    b = _batch(cache, index, block_table, seq_lens, query_start, tokens)
    c = cache._struct()
    with _here(index):
        check(lib().ci_paged_kv_read(c, b, kr, vr, _lib.stream_handle(cache.data.device)))
    return k_out, v_out


def paged_attention(q, cache: PagedKVCache, block_table, seq_lens, query_start=None, window: int = 0, sinks: int = 0,
                    scale=None, max_query_len: int = 0, max_seq_len: int = 0, out=None, return_lse: bool = False):
    """softmax(scale * q k^T) v over the visible keys of every query's sequence; q [T, heads, head_dim] in bf16, heads a
    multiple of the cache's kv heads.  The query at position p sees key j when j <= p and, with a `window` > 0, p - j <
    window or j < `sinks`.  A row that sees nothing (a sequence of length 0) gets zeros, one whose scores are all -inf is
    NaN; rows behind the last sequence are not written.  With a window, pages that hold no key a new token sees need not be
    named in `block_table` (any entry will do).  `out` shares no memory with q.  `scale`: 1 / sqrt(head_dim) if not given;
    positive.  `max_query_len`, `max_seq_len`: what the caller knows about the longest sequence (0: nothing); they choose
    kernels, the results do not rest on them.  `return_lse`: also fp32 [T, heads], the natural logarithm of the sum of
    exp(scores).  Scores, sums and the output are held in 32
    bits; the weights are rounded to bf16 for the product with v.  No gradients: a q that requires one is refused."""
    _lib.require_device(cache.data)
    _no_gradient(q)
    dev = cache.data.device
    index = cache.data.get_device()
    qr = _rows("q", q, cache, index, None, None)
    tokens, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads are no multiple of {cache.kv_heads} kv heads")
    out = _output("out", out, tokens, heads, cache)
    orows = _rows("out", out, cache, index, heads, tokens)
    b = _batch(cache, index, block_table, seq_lens, query_start, tokens)
    limit = (1 << 31) - 1
    window, sinks = int(window), int(sinks)
    if not (0 <= window <= limit and 0 <= sinks <= limit):
        raise ValueError("window and sinks must be 0 to 2^31 - 1")
    max_query_len, max_seq_len = min(max(int(max_query_len), 0), limit), min(max(int(max_seq_len), 0), limit)
    lse = torch.empty(tokens, heads, dtype=torch.float32, device=dev) if return_lse else None
    c = cache._struct()
    library = lib()
    library.ci_paged_attention_workspace_bytes.restype = C.c_size_t
    with _here(index):
        need = library.ci_paged_attention_workspace_bytes(c, b, heads, window, sinks, max_query_len, max_seq_len)
        # (a workspace of the call's own: two captured graphs never share one)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(library.ci_paged_attention(
            c, b, qr, orows, ptr(lse), C.c_int64(heads), heads,
            C.c_float(cache.head_dim ** -0.5 if scale is None else float(scale)), window, sinks, max_query_len, max_seq_len,
            ptr(ws), C.c_size_t(need), _lib.stream_handle(dev)))
    return (out, lse) if return_lse else out
