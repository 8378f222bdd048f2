"""The paged cache's and the attention's kernels on the host model: the tests written for the GPU
(tests/test_gpu_paged.py), on the plain model, and a part of them with every memory access instrumented (wavefronts that
touch the same LDS byte with no barrier in between) and with the compiler's undefined-behaviour checks; and cases in the
model's own memory, where every array ends at an inaccessible page and nothing unwritten may be read."""
import ctypes as C
import os
import re
import subprocess
import sys

import numpy as np
import pytest

from tests.hostmodel.model import Model, in_child

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
JOBS = str(max(1, min(7, (os.cpu_count() or 2) - 1)))


def _suite(lib=None, pick=None, least=1):
    from tests.hostmodel import build

    env = dict(os.environ, OMP_NUM_THREADS="1", PYTHONPATH=ROOT)
    path = build.build(**{lib: True}) if lib else None
    build.build()  # (the children find the libraries up to date)
    if path:
        env["CI_HOSTMODEL_LIB"] = path
    cmd = [sys.executable, "-m", "pytest", "tests/test_gpu_paged.py", "-m", "gpu", "-q", "-p", "tests.hostmodel.pytest_plugin",
           "--timeout", "900", "-p", "no:cacheprovider", "-n", JOBS] + (["-k", pick] if pick else [])
    p = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=1800)
    assert p.returncode == 0, p.stdout[-6000:] + p.stderr[-1000:]
    m = re.search(r"(\d+) passed", p.stdout)
    assert m and int(m.group(1)) >= least, p.stdout[-1500:]


def test_the_gpu_tests_on_the_host_model():
    _suite(least=180)


PART = "one_token or behind or special or (lens2-news2-64-3 and append) or (33-70-24-2 and single) or (50-5-lens1 and 6-2) or exist"


def test_a_part_of_them_with_ordering_checked():
    _suite("order", PART, 15)


def test_a_part_of_them_with_undefined_behaviour_checked():
    _suite("undefined", PART, 15)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("build", [None, "order"])
def test_arrays_that_end_at_an_inaccessible_page(kind, dim, build):
    _arrays(kind, dim, build)


def _bf16(a):
    u = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def _f64(b):
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@in_child
def _arrays(kind, dim, build):
    """Append, read and attention (single tokens, cut items, prompts; windows) with every operand ending (or beginning)
    where memory does and, in the instrumented build, every byte of workspace and outputs unwritten at first."""
    from comp_inference_amd import attention_hip as A
    from tests.hostmodel import build as B

    for end in (True, False):
        m = Model(cus=4, end_at_guard=end, lib_path=B.build(order=True) if build else None)
        L = m.lib
        L.ci_kv_cache_bytes.restype = C.c_uint64
        L.ci_paged_attention_workspace_bytes.restype = C.c_size_t
        rng = np.random.default_rng(dim + kind)
        heads, kv, page = 6, 2, 32
        for lens, news in (([700, 33], None), ([33, 100], [33, 90])):
            seqs = len(lens)
            need = [-(-l // page) for l in lens]
            pages = sum(need)
            table = np.full((seqs, max(need)), -1, np.int32)
            order, at = rng.permutation(pages), 0
            for b, n in enumerate(need):
                table[b, :n] = order[at:at + n]
                at += n
            nbytes = L.ci_kv_cache_bytes(pages, page, kv, dim, kind)
            data = m.dev(np.zeros(nbytes, np.uint8))
            cache = A._Cache(data.ptr, nbytes, pages, page, kv, dim, kind)
            total = sum(lens)
            k, v = _bf16(rng.standard_normal((total, kv, dim))), _bf16(rng.standard_normal((total, kv, dim)))
            dk, dv = m.dev(k), m.dev(v)
            dt, dl = m.dev(table), m.dev(np.array(lens, np.int32))
            cut = lambda ns: m.dev(np.concatenate([[0], np.cumsum(ns)]).astype(np.int32))  # noqa: E731
            whole = cut(lens)
            rows = lambda d, h: A._Rows(d.ptr, h * dim, dim)  # noqa: E731
            every = A._Batch(dt.ptr, table.shape[1], table.shape[1], dl.ptr, whole.ptr, seqs, total)
            m.call("ci_paged_kv_append", C.byref(cache), C.byref(every), C.byref(rows(dk, kv)), C.byref(rows(dv, kv)), None, None, 0,
                   None, 0, 0, None)
            rk, rv = m.empty((total, kv, dim), np.uint16), m.empty((total, kv, dim), np.uint16)
            m.call("ci_paged_kv_read", C.byref(cache), C.byref(every), C.byref(rows(rk, kv)), C.byref(rows(rv, kv)), None)
            if kind == 0:
                assert np.array_equal(rk.get(), k) and np.array_equal(rv.get(), v)
            else:
                assert np.abs(_f64(rk.get()) - _f64(k)).max() < 0.4
            T = seqs if news is None else sum(news)
            q = m.dev(_bf16(rng.standard_normal((T, heads, dim))))
            start = None if news is None else cut(news)
            batch = A._Batch(dt.ptr, table.shape[1], table.shape[1], dl.ptr, start.ptr if start else None, seqs, T)
            for window, sinks in ((0, 0), (40, 3)):
                for longest in (0, 1):
                    args = (heads, window, sinks, longest, 0)
                    n = L.ci_paged_attention_workspace_bytes(C.byref(cache), C.byref(batch), *args)
                    ws, out = m.empty(max(n, 1), np.uint8), m.empty((T, heads, dim), np.uint16)
                    lse = m.empty((T, heads), np.float32)
                    m.call("ci_paged_attention", C.byref(cache), C.byref(batch), C.byref(rows(q, heads)), C.byref(rows(out, heads)),
                           lse.p, C.c_int64(heads), heads, C.c_float(dim ** -0.5), window, sinks, longest, 0,
                           ws.p if n else None, C.c_size_t(n), None)
                    got, ks, vs = _f64(out.get()), _f64(rk.get()), _f64(rv.get())
                    at = 0
                    for b, l in enumerate(lens):
                        first = sum(lens[:b])
                        nn = 1 if news is None else news[b]
                        for i in {0, nn // 2, nn - 1}:
                            p = l - nn + i
                            j = np.arange(p + 1)
                            j = j[(p - j < window) | (j < sinks)] if window else j
                            for h in (0, heads - 1):
                                s = ks[first + j, h // 3] @ _f64(q.get())[at + i, h] * dim ** -0.5
                                w = np.exp(s - s.max())
                                want = w @ vs[first + j, h // 3] / w.sum()
                                # (a rounding of each weight, of each value read back, of the result: 2^-8 each, times
                                # sums of |v| below 4, and scores off by a key's rounding)
                                assert np.abs(got[at + i, h] - want).max() < 0.05, (kind, dim, window, longest, b, i, h)
                        at += nn
        m.free_all()
