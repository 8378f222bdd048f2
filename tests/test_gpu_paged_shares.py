"""Attention over the paged cache with many rows and more than 2048 keys: tiles of 256 rows whose steps are cut into shares
between workgroups and joined.  Sizes follow the compute units, so that a card of 256 takes this path and the host model of 8
does (tests/test_hostmodel_paged_shares.py asserts the launches)."""
import math

import pytest
import torch

import paged_ref as R
from test_gpu_paged import DEV, Filled, _ci, _compare

pytestmark = pytest.mark.gpu


def _kv_heads(tokens, group):
    """Heads of the cache enough for the kernel for many rows: its tiles are to number a quarter of the compute units."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    heads = 1
    while tokens * group * heads < 64 * cus:
        heads += 1 if heads < 4 else 2
    return heads


# lengths and new tokens, query heads of a kv head
RAGGED = ([4200, 2100, 1], [600, 300, 1], 4)   # ten tiles, five (one in the middle), one of four rows; some cut, some not
PARTS = ([5000], [70], 8)                      # three tiles, every one cut several times
WHOLE = ([2331], [2331], 1)                    # a prompt from its first token: tiles of 4 to 37 steps
MIXED = ([3000] + [700] * 5, [130] + [1] * 5, 6)  # one part of a prompt among single tokens


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news,group", [pytest.param(*RAGGED, id="ragged"), pytest.param(*PARTS, id="parts"),
                                             pytest.param(*WHOLE, id="whole"), pytest.param(*MIXED, id="mixed")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2100, 70)])
def test_prompts_cut_into_shares(kind, dim, lens, news, group, window, sinks):
    ci = _ci()
    heads = _kv_heads(sum(news), group)
    f = Filled(lens, news, group * heads, heads, dim, kind, page=32, seed=7, scale=1.5)
    q = f.q.to(DEV)
    got, lse = ci.paged_attention(q, *f.args(), window=window, sinks=sinks, return_lse=True)
    want, want_lse, bound = f.expect(window, sinks)
    _compare(got, want, bound)
    assert torch.allclose(lse.double().cpu(), want_lse, rtol=0, atol=1e-3)
    # the same bits again, and with pages taken out that no new token sees
    table = f.table.clone()
    if window:
        for b, (l, n) in enumerate(zip(lens, news)):
            at = torch.arange(table.shape[1]) * 32
            table[b, ((at >= sinks) & (at + 31 < l - n - window + 1)).to(DEV)] = -1
        assert (table != f.table).any() or lens == WHOLE[0]
    again = ci.paged_attention(q, f.cache, table, f.seq, f.start, window=window, sinks=sinks)
    assert torch.equal(again, got)
    assert ci.device_status() == 0


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_pages_that_do_not_exist_inside_shares(kind):
    """A page in the middle of a long sequence is none of the cache's: its keys are seen by nobody, and it is reported."""
    ci = _ci()
    lens, news, group = PARTS
    heads = _kv_heads(sum(news), group)
    f = Filled(lens, news, group * heads, heads, 128, kind, page=64, seed=9)
    f.table[0, 20] = f.cache.num_pages + 5
    got = ci.paged_attention(f.q.to(DEV), *f.args())
    with pytest.raises(RuntimeError, match="do not exist"):
        ci.device_status()
    there = torch.cat((torch.arange(0, 20 * 64), torch.arange(21 * 64, lens[0])))
    f.k[0], f.v[0], f.lens = f.k[0][there], f.v[0][there], [len(there)]
    want, _, bound = f.expect()
    _compare(got, want, bound)


def test_a_captured_call_in_shares():
    """Replays with other contents, lengths and pages, eager work between them."""
    ci = _ci()
    if type(torch.cuda.current_stream()).__name__ == "_Stream":
        pytest.skip("needs streams")
    lens, news, group = RAGGED
    heads = _kv_heads(sum(news), group)
    a = Filled(lens, news, group * heads, heads, 64, "bf16", page=32, seed=11)
    b = Filled([l - 37 if l > 40 else l for l in lens], news, group * heads, heads, 64, "bf16", page=32, seed=12)
    q, seq = a.q.to(DEV), a.seq.clone()
    table = torch.zeros(3, max(a.table.shape[1], b.table.shape[1]), dtype=torch.int32, device=DEV)
    cache = ci.PagedKVCache(max(a.cache.num_pages, b.cache.num_pages), 32, heads, 64, device=DEV)

    def fill(f):
        q.copy_(f.q), seq.copy_(f.seq), table.fill_(-1)
        table[:, :f.table.shape[1]] = f.table
        cache.data[:f.cache.num_pages] = f.cache.data

    fill(a)
    call = lambda: ci.paged_attention(q, cache, table, seq, a.start)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for f in (b, a, b):
        fill(f)
        out.fill_(math.nan)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        want, _, bound = f.expect()
        _compare(out, want, bound)
        torch.randn(1 << 20, device=DEV).sum().item()
