"""Rows of attention over the paged cache that give no key a weight: those that see keys, all with scores of minus infinity,
are NaN, as the formula says; those that see no key are zeros."""
import math

import pytest
import torch

import paged_ref as R
from test_gpu_paged import DEV, _ci, _compare
from test_gpu_paged_wild import CALLS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news,heads,kv_heads,bounds", CALLS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_scores_of_minus_infinity_alone(dim, lens, news, heads, kv_heads, bounds, window, sinks):
    """A channel of the keys before a token is minus infinity, queries are positive there: rows before that token have no
    other score, the rows from it on give those keys no weight."""
    ci = _ci()
    table, seq, start, pages = R.layout(lens, news, 32, seed=3)
    table, seq, start = table.to(DEV), seq.to(DEV), start.to(DEV)
    cache = ci.PagedKVCache(pages, 32, kv_heads, dim, device=DEV)
    k = [R.normal(l, kv_heads, dim, seed=11 + i) for i, l in enumerate(lens)]
    v = [R.normal(l, kv_heads, dim, seed=21 + i) for i, l in enumerate(lens)]
    q = R.normal(sum(news), heads, dim, seed=31)
    q[..., 5] = q[..., 5].abs() + 0.5
    cut = [l - n + n // 2 for l, n in zip(lens, news)]
    for x, t in zip(k, cut):
        x[:t, :, 5] = -math.inf
    whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(cache, torch.cat(k).to(DEV), torch.cat(v).to(DEV), table, seq, whole)
    got, lse = ci.paged_attention(q.to(DEV), cache, table, seq, start, window=window, sinks=sinks, return_lse=True, **bounds)
    at = 0
    for b, (l, n, t) in enumerate(zip(lens, news, cut)):
        none = t - (l - n)  # rows before the token
        assert got[at:at + none].isnan().all() and (lse[at:at + none] == -math.inf).all()
        rest = slice(at + none, at + n)
        want, want_lse, mass, worst = R.attention(q[rest], k[b][t:].double(), v[b][t:].double(), 0, dim ** -0.5, window, 0)
        _compare(got[rest], want, R.attention_bound(want, mass, worst, dim))
        assert torch.allclose(lse[rest].double().cpu(), want_lse, rtol=0, atol=1e-3)
        at += n
    assert ci.device_status() == 0
    # a sequence none of whose pages exist sees no key: zeros
    table[0] = -1
    got, lse = ci.paged_attention(q.to(DEV), cache, table, seq, start, window=window, sinks=sinks, return_lse=True, **bounds)
    assert not got[:news[0]].any() and (lse[:news[0]] == -math.inf).all()
    with pytest.raises(RuntimeError, match="do not exist"):
        ci.device_status()


def test_single_tokens_and_a_last_page_that_is_gone():
    """One token each: scores of minus infinity alone, in one workgroup and cut into parts; with the newest page gone the
    keys of the others are still seen."""
    ci = _ci()
    lens, H, D = [40, 1500, 70], 2, 128
    table, seq, _, pages = R.layout(lens, [1, 1, 1], 32, seed=4)
    table, seq = table.to(DEV), seq.to(DEV)
    cache = ci.PagedKVCache(pages, 32, H, D, device=DEV)
    k = torch.full((sum(lens), H, D), 1.0, dtype=torch.bfloat16)
    k[..., 9] = -math.inf
    whole = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(cache, k.to(DEV), R.normal(sum(lens), H, D, seed=1).to(DEV), table, seq, whole)
    q = torch.ones(3, 4 * H, D, dtype=torch.bfloat16).to(DEV)
    for kw in ({}, dict(max_seq_len=100), dict(window=33)):
        assert ci.paged_attention(q, cache, table, seq, **kw).isnan().all()
    assert ci.device_status() == 0
    table[2, 2] = -1
    assert ci.paged_attention(q, cache, table, seq).isnan().all()
    table[2, :2] = pages
    got = ci.paged_attention(q, cache, table, seq)
    assert got[:2].isnan().all() and not got[2].any()
    with pytest.raises(RuntimeError, match="do not exist"):
        ci.device_status()
