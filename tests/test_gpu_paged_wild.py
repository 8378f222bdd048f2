"""Attention over the paged cache beside values that are no numbers: a row is an infinity or NaN in exactly the channels in
which a key it sees is, whatever the other rows of its tile see, by every kernel; and such values do not make a call take
hundreds of times its time."""
import math

import pytest
import torch

import paged_ref as R
from test_gpu_paged import DEV, Filled, _ci

pytestmark = pytest.mark.gpu

CALLS = [
    # many rows: whole tiles, and (over 2048 keys) tiles cut into shares; rows enough for a card of 256 CUs
    pytest.param([1100], [1100], 16, 8, {}, id="rows"),
    pytest.param([2500], [1300], 14, 7, {}, id="rows_in_shares"),
    # few rows: whole, and items cut and joined, several tokens in a tile
    pytest.param([90, 33], [30, 33], 4, 2, dict(max_query_len=2, max_seq_len=100), id="few"),
    pytest.param([1500, 700], [9, 30], 4, 2, dict(max_query_len=2), id="few_in_shares"),
    pytest.param([1500, 700], [9, 30], 4, 2, dict(max_query_len=12), id="few_in_shares_32"),
]


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news,heads,kv_heads,bounds", CALLS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_infinities_and_nan_reach_the_rows_that_see_them(kind, dim, lens, news, heads, kv_heads, bounds, window, sinks):
    ci = _ci()
    f = Filled(lens, news, heads, kv_heads, dim, kind, page=32, seed=17)
    v, at, parts = [x.clone() for x in f.v], 0, []
    inf, nan = math.inf, math.nan
    for b, (l, n) in enumerate(zip(lens, news)):
        # the first token (heads of 64; a 4-bit row with a NaN is NaN throughout, so no row would be left there); two neighbours
        # in the middle of the new ones, whose infinities cancel where both are seen; the last
        for t, four in ((0, [1.0, 1.0, nan, 1.0]), (l - n + n // 2, [inf, -inf, 1.0, 1.0]), (l - n + n // 2 + 1, [-inf, -inf, 1.0, 1.0]),
                        (l - 1, [1.0, 1.0, 1.0, inf])):
            if t == 0 and dim == 128:
                continue
            row = torch.tensor(four * (dim // 4), dtype=torch.bfloat16)
            v[b][t] = torch.where(torch.isfinite(row), v[b][t], row)
    whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(f.cache, torch.cat(f.k).to(DEV), torch.cat(v).to(DEV), f.table, f.seq, whole)
    got, lse = ci.paged_attention(f.q.to(DEV), *f.args(), window=window, sinks=sinks, return_lse=True, **bounds)
    got, lse = got.double().cpu(), lse.double().cpu()
    for b, (l, n) in enumerate(zip(lens, news)):
        k, x = R.stored(f.k[b], kind), R.stored(v[b], kind)
        finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
        want, want_lse, mass, worst = R.attention(f.q[at:at + n], k, finite, l - n, dim ** -0.5, window, sinks)
        if kind == "int4":  # (a code times its step, beside the low; rows that are no numbers hold neither)
            y = torch.where(torch.isfinite(v[b].float()).all(-1, keepdim=True), v[b], torch.zeros_like(v[b]))
            step, _ = R.pairs(y)
            mass = mass + R.attention(f.q[at:at + n], k, (R.codes(y) * step).double(), l - n, dim ** -0.5, window, sinks)[0]
        bound = R.attention_bound(want, mass, worst, dim)
        seen = R.visible(l - n + torch.arange(n), l, window, sinks).double()
        kinds = [(seen @ m.double().reshape(l, -1)).reshape(n, kv_heads, dim).repeat_interleave(heads // kv_heads, 1) > 0
                 for m in (x == inf, x == -inf, x.isnan())]
        none = kinds[2] | (kinds[0] & kinds[1])
        y, part = got[at:at + n], lse[at:at + n]
        assert torch.equal(y.isnan(), none)
        assert (y[kinds[0] & ~none] == inf).all() and (y[kinds[1] & ~none] == -inf).all()
        rest = ~(kinds[0] | kinds[1] | none)
        parts.append(rest)
        off = ((y - want).abs() - bound)[rest]
        assert not off.numel() or float(off.max()) <= 0
        assert torch.allclose(part, want_lse, rtol=0, atol=1e-3)
        at += n
    assert any(p.any() for p in parts) or (kind == "int4" and dim == 64)
    assert ci.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news,heads,kv_heads,bounds", CALLS)
def test_an_infinity_without_weight_is_no_number(dim, lens, news, heads, kv_heads, bounds):
    """A key whose score is minus infinity weighs nothing, and nothing times an infinity is no number: rows that see it are NaN
    where its value is infinite, and only there; a key with a weight and an infinity leaves infinities."""
    ci = _ci()
    f = Filled(lens, news, heads, kv_heads, dim, "bf16", page=32, seed=23)
    q = f.q.clone()
    q[..., 5] = q[..., 5].abs() + 0.5
    k, v, at = [x.clone() for x in f.k], [x.clone() for x in f.v], 0
    where = [l - n + n // 2 for l, n in zip(lens, news)]
    for b, t in enumerate(where):
        k[b][t, :, 5] = -math.inf
        v[b][t, :, 8] = math.inf
        v[b][t, :, 9] = -math.inf
        v[b][max(t - 1, 0), :, 10] = math.inf
    whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(f.cache, torch.cat(k).to(DEV), torch.cat(v).to(DEV), f.table, f.seq, whole)
    got = ci.paged_attention(q.to(DEV), *f.args(), **bounds).cpu()
    for l, n, t in zip(lens, news, where):
        p = torch.arange(l - n, l)
        y = got[at:at + n]
        assert y[p >= t][..., 8:10].isnan().all() and (y[p >= t - 1][..., 10] == math.inf).all()
        rest = y.clone()
        rest[p >= t, :, 8:10] = 0
        rest[p >= t - 1, :, 10] = 0
        assert torch.isfinite(rest).all()
        at += n
    assert ci.device_status() == 0


def _microseconds(call, times=5):
    call()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(times):
        call()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) * 1e3 / times


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("lens,news,heads,kv_heads,least", [([1500], [1500], 16, 8, 30.0), ([20000], [1], 32, 8, 5.0),
                                                            ([20000], [6], 32, 8, 5.0)])
def test_a_nan_at_the_first_token_costs_little_time(kind, lens, news, heads, kv_heads, least):
    """Every row sees it, so every row is NaN in that channel, and is computed a second time at a lower rate: three to five
    times the call for a prompt, at most twice for few rows (whose other wavefronts see numbers alone).  Rows done one by one
    took two hundred times the call."""
    ci = _ci()
    if type(torch.cuda.current_stream()).__name__ == "_Stream":
        pytest.skip("needs a GPU's time")
    f = Filled(lens, news, heads, kv_heads, 128, kind, seed=5)
    q = f.q.to(DEV)
    call = lambda: ci.paged_attention(q, *f.args(), max_query_len=max(news))  # noqa: E731
    before = _microseconds(call)
    v = [x.clone() for x in f.v]
    v[0][0, :, 7] = math.nan
    whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(f.cache, torch.cat(f.k).to(DEV), torch.cat(v).to(DEV), f.table, f.seq, whole)
    after = _microseconds(call)
    assert call()[..., 7].isnan().all()
    assert after < least * max(before, 20.0), (before, after)
