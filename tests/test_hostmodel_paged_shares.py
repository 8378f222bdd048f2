"""The newer GPU tests of the paged cache on the host model of the library: prompts cut into shares, values that are no
numbers, rows without weight, 4-bit accuracy; a part of them with the ordering between wavefronts checked and with the
compiler's undefined-behaviour checks.  The log of launches shows that shares of many rows are joined there."""
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
FILES = ["tests/test_gpu_paged_shares.py", "tests/test_gpu_paged_wild.py", "tests/test_gpu_paged_no_weight.py", "tests/test_gpu_paged_four_bits.py"]


def _run(files, log, lib=None, pick=None, least=1):
    """Runs tests on the model; the names of the kernels launched."""
    from tests.hostmodel import build

    path = build.build(**{lib: True}) if lib else None
    build.build()  # (the children find the libraries up to date)
    env = dict(os.environ, OMP_NUM_THREADS="1", PYTHONPATH=ROOT, CI_HOSTMODEL_LAUNCH_LOG=str(log))
    if path:
        env["CI_HOSTMODEL_LIB"] = path
    cmd = [sys.executable, "-m", "pytest", *files, "-m", "gpu", "-q", "-p", "tests.hostmodel.pytest_plugin", "--timeout", "900",
           "-p", "no:cacheprovider", "-n", JOBS] + (["-k", pick] if pick else [])
    p = subprocess.run(cmd, cwd=ROOT, env=env, capture_output=True, text=True, timeout=1800)
    assert p.returncode == 0, p.stdout[-6000:] + p.stderr[-1000:]
    m = re.search(r"(\d+) passed", p.stdout)
    assert m and int(m.group(1)) >= least, p.stdout[-1500:]
    return open(log).read()


def _joins(log):
    return log.count("attend_rows_join_kernel")


MOST = "not (shares and (mixed or (ragged and 128))) and not (see_them and rows and 128)"  # (the longest ones; minutes)


def test_the_newer_gpu_tests_on_the_host_model(tmp_path):
    log = _run(FILES, tmp_path / "launches", pick=MOST, least=80)
    assert _joins(log) >= 50, _joins(log)


PART = "(cut_into_shares and parts) or (see_them and few) or (alone and few_in_shares and 64) or (only and few_several)"


def test_a_part_of_them_with_ordering_checked(tmp_path):
    assert _joins(_run(FILES, tmp_path / "launches", "order", PART, 20)) >= 16


def test_a_part_of_them_with_undefined_behaviour_checked(tmp_path):
    assert _joins(_run(FILES, tmp_path / "launches", "undefined", PART, 20)) >= 16


@pytest.mark.parametrize("kind", [0, 1])
@in_child
def test_no_part_is_joined_that_was_not_written(kind):
    """Batches whose cuts fall anywhere in a tile, near its ends too, where they are moved: on the build that knows which
    bytes of the workspace have been written; against plain sums at a few rows."""
    from comp_inference_amd import attention_hip as A
    from tests.hostmodel import build
    from tests.test_hostmodel_paged import _bf16, _f64

    m = Model(cus=8, lib_path=build.build(order=True))
    L = m.lib
    L.ci_kv_cache_bytes.restype = C.c_uint64
    L.ci_paged_attention_workspace_bytes.restype = C.c_size_t
    dim, page = 64, 64
    for n, keys in ((520, 2300), (777, 2211), (1030, 2600)):
        rng = np.random.default_rng(n + kind)
        pages = -(-keys // page)
        nbytes = L.ci_kv_cache_bytes(pages, page, 1, dim, kind)
        data = m.dev(np.zeros(nbytes, np.uint8))
        cache = A._Cache(data.ptr, nbytes, pages, page, 1, dim, kind)
        dt, dl = m.dev(rng.permutation(pages).astype(np.int32)[None]), m.dev(np.array([keys], np.int32))
        dk, dv = (m.dev(_bf16(rng.standard_normal((keys, 1, dim)))) for _ in range(2))
        rows = lambda d: C.byref(A._Rows(d.ptr, dim, dim))  # noqa: E731
        whole, start = m.dev(np.array([0, keys], np.int32)), m.dev(np.array([0, n], np.int32))
        every = A._Batch(dt.ptr, pages, pages, dl.ptr, whole.ptr, 1, keys)
        m.call("ci_paged_kv_append", C.byref(cache), C.byref(every), rows(dk), rows(dv), None, None, 0, None, 0, 0, None)
        rk, rv = m.empty((keys, 1, dim), np.uint16), m.empty((keys, 1, dim), np.uint16)
        m.call("ci_paged_kv_read", C.byref(cache), C.byref(every), rows(rk), rows(rv), None)
        q, out = m.dev(_bf16(rng.standard_normal((n, 1, dim)))), m.empty((n, 1, dim), np.uint16)
        batch = A._Batch(dt.ptr, pages, pages, dl.ptr, start.ptr, 1, n)
        size = L.ci_paged_attention_workspace_bytes(C.byref(cache), C.byref(batch), 1, 0, 0, 0, 0)
        assert size
        ws = m.empty(size, np.uint8)
        m.call("ci_paged_attention", C.byref(cache), C.byref(batch), rows(q), rows(out), None, C.c_int64(1), 1, C.c_float(dim ** -0.5),
               0, 0, 0, 0, ws.p, C.c_size_t(size), None)
        got, ks, vs = _f64(out.get()), _f64(rk.get()), _f64(rv.get())
        for i in (0, 255, 256, n // 2, n - 1):
            p = keys - n + i
            s = ks[:p + 1, 0] @ _f64(q.get())[i, 0] * dim ** -0.5
            w = np.exp(s - s.max())
            # (a rounding of each weight and of the result, 2^-8 each of sums of |v| around one; scores off by a key's rounding)
            assert np.abs(got[i, 0] - w @ vs[:p + 1, 0] / w.sum()).max() < 0.03, (n, keys, i)
        m.free_all()
