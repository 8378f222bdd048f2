"""The paged key/value cache and attention over it (comp_inference_amd/attention_hip.py) against plain forms in 64 bits
(tests/paged_ref.py): stored rows and codes exactly, attention within bounds derived from its roundings."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ci():
    import comp_inference_amd as ci

    return ci


def _put(*tensors):
    return [t.to(DEV) for t in tensors]


class Filled:
    """A cache that holds given keys and values (made by appending whole sequences), and its batch."""

    def __init__(self, lens, news, heads, kv_heads, dim, kind, page=64, seed=0, scale=1.0, fill=None):
        ci = _ci()
        table, seq, start, pages = R.layout(lens, news, page, seed=seed)
        self.cache = ci.PagedKVCache(pages, page, kv_heads, dim, kind=kind, device=DEV)
        if fill is not None:
            self.cache.data.view(torch.uint8).fill_(fill)
        self.k = [R.normal(l, kv_heads, dim, seed=seed + 7 * i + 1, scale=scale) for i, l in enumerate(lens)]
        self.v = [R.normal(l, kv_heads, dim, seed=seed + 7 * i + 2) for i, l in enumerate(lens)]
        self.q = R.normal(sum(news), heads, dim, seed=seed + 3, scale=scale)
        self.lens, self.news, self.kind, self.dim = lens, news, kind, dim
        self.table, self.seq, self.start = _put(table, seq, start)
        if sum(lens):
            whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
            ci.paged_kv_append(self.cache, torch.cat(self.k).to(DEV), torch.cat(self.v).to(DEV), self.table, self.seq, whole)

    def args(self, rows=True):
        return (self.cache, self.table, self.seq) + ((self.start,) if rows else ())

    def expect(self, window=0, sinks=0, scale=None):
        """(out, lse, bound) of every row."""
        out, lse, bound = [], [], []
        at = 0
        for b, (l, n) in enumerate(zip(self.lens, self.news)):
            k, v = R.stored(self.k[b], self.kind), R.stored(self.v[b], self.kind)
            o, s, mass, worst = R.attention(self.q[at:at + n], k, v, l - n, scale or self.dim ** -0.5, window, sinks)
            if self.kind == "int4":  # what is summed is a code times its step, beside the low
                step, low = R.pairs(self.v[b])
                mass = mass + R.attention(self.q[at:at + n], k, (R.codes(self.v[b]) * step).double(), l - n,
                                          scale or self.dim ** -0.5, window, sinks)[0]
            out.append(o), lse.append(s), bound.append(R.attention_bound(o, mass, worst, self.dim))
            at += n
        return torch.cat(out), torch.cat(lse), torch.cat(bound)


def _compare(got, want, bound, what=""):
    got = got.double().cpu()
    off = (got - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert float(off.max()) <= 0, (what, float(off.max()), off.argmax().item(), float((got - want).abs().max()))


# ---- the cache ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("dim,kv_heads,heads,page,rotary_dim", [
    (128, 2, 4, 64, 128), (64, 3, 3, 32, 64), (128, 1, 5, 128, 32), (64, 5, 10, 256, 16), (64, 70, 70, 32, None)])
@pytest.mark.parametrize("lens,news", [([1], [1]), ([33, 5, 70], [33, 2, 41]), ([40, 64, 31, 97], [9, 0, 31, 66])])
def test_append_and_read(kind, dim, kv_heads, heads, page, rotary_dim, lens, news):
    """Parts of blocks, whole blocks and several, rows of a packed tensor; what the cache held before stays."""
    ci = _ci()
    table, seq, start, pages = _layout_on_device(lens, news, page)
    cache = ci.PagedKVCache(pages, page, kv_heads, dim, kind=kind, device=DEV)
    old = [max(l - n, 0) for l, n in zip(lens, news)]
    old_k, old_v = R.normal(sum(old), kv_heads, dim, seed=11), R.normal(sum(old), kv_heads, dim, seed=12)
    cut = lambda ns: torch.tensor([0] + ns).cumsum(0).to(torch.int32).to(DEV)  # noqa: E731
    if sum(old):
        ci.paged_kv_append(cache, old_k.to(DEV), old_v.to(DEV), table, torch.tensor(old, dtype=torch.int32).to(DEV), cut(old))
    T = sum(news)
    packed = R.normal(T, heads + 2 * kv_heads, dim, seed=13)
    q, k, v = packed.split((heads, kv_heads, kv_heads), 1)
    gq, gk, gv = packed.to(DEV).split((heads, kv_heads, kv_heads), 1)
    rotary = None if rotary_dim is None else ci.rotary_table(max(lens) + 3, rotary_dim, theta=500000.0, device=DEV)
    got_q = ci.paged_kv_append(cache, gk, gv, table, seq, start, q=gq, rotary=rotary)
    pos = torch.cat([torch.arange(l - n, l) for l, n in zip(lens, news)])
    want_k = k if rotary is None else R.rotate(k, pos, rotary.cpu())
    want_q = q if rotary is None else R.rotate(q, pos, rotary.cpu())
    assert torch.equal(got_q.cpu(), want_q)
    # everything the cache now holds, sequence after sequence
    got_k, got_v = ci.paged_kv_read(cache, table, seq, cut(lens), tokens=sum(lens))
    want = []
    for x, o in ((want_k, old_k), (v, old_v)):
        parts, a, b = [], 0, 0
        for n, m in zip(old, news):
            parts += [o[a:a + n], x[b:b + m]]
            a, b = a + n, b + m
        want.append(R.stored(torch.cat(parts), kind).float().to(torch.bfloat16))
    assert torch.equal(got_k.cpu(), want[0]) and torch.equal(got_v.cpu(), want[1])
    assert ci.device_status() == 0


def _layout_on_device(lens, news, page, seed=5):
    table, seq, start, pages = R.layout(lens, news, page, seed=seed)
    return (*_put(table, seq, start), pages)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
def test_append_one_token_each(kind):
    """The form of a decode step: no row offsets, one row per sequence, a place of length 0 among them; token after token
    gives what the whole sequence at once gives, bit for bit."""
    ci = _ci()
    lens, page, H, D = [37, 0, 5, 64], 32, 3, 128
    table, seq, _, pages = _layout_on_device(lens, [0] * 4, page)
    k, v = R.normal(max(lens), 4, H, D, seed=1), R.normal(max(lens), 4, H, D, seed=2)
    rotary = ci.rotary_table(80, D, device=DEV)
    step = ci.PagedKVCache(pages, page, H, D, kind=kind, device=DEV)
    for t in range(max(lens)):
        at = torch.tensor([t + 1 if t < l else 0 for l in lens], dtype=torch.int32).to(DEV)
        q = R.normal(4, 6, D, seed=100 + t)
        gq = torch.full((4, 6, D), 7.0, dtype=torch.bfloat16, device=DEV)
        ci.paged_kv_append(step, k[t].to(DEV), v[t].to(DEV), table, at, q=q.to(DEV), rotary=rotary, q_out=gq)
        turned = R.rotate(q, torch.full((4,), t), rotary.cpu())
        for b, l in enumerate(lens):
            assert torch.equal(gq[b].cpu(), turned[b] if t < l else torch.full((6, D), 7.0, dtype=torch.bfloat16))
    whole = ci.PagedKVCache(pages, page, H, D, kind=kind, device=DEV)
    rows = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(whole, torch.cat([k[:l, b] for b, l in enumerate(lens)]).to(DEV),
                       torch.cat([v[:l, b] for b, l in enumerate(lens)]).to(DEV), table, seq, rows, rotary=rotary)
    assert torch.equal(step.data.view(torch.uint8).cpu(), whole.data.view(torch.uint8).cpu())
    assert ci.device_status() == 0


def test_four_bit_rows_that_are_special():
    """Constant rows, rows with values on the border of two codes, tiny and huge ranges, infinities and NaN."""
    ci = _ci()
    D, rows = 64, []
    rows.append(torch.full((D,), 1.5))
    rows.append(torch.zeros(D))
    rows.append(torch.arange(D) % 16 * 1.0)                        # every code exactly
    rows.append(torch.arange(D) % 31 * 0.5)                        # every second value on a border
    rows.append(torch.cat((torch.tensor([-7.5, 7.5, 1e-30, -1e-30]), torch.zeros(D - 4))))  # beside a border
    rows.append(torch.linspace(-1e-38, 2e-38, D))
    rows.append(torch.linspace(-3e-40, 3e-40, D))                  # below the smallest normal number
    rows.append(torch.linspace(-1, 1, D) * 3e38)                  # maximum - minimum beyond 32 bits
    rows.append(torch.linspace(1000.0, 1001.0, D))
    rows.append(torch.cat((torch.tensor([math.inf]), torch.zeros(D - 1))))
    rows.append(torch.cat((torch.tensor([math.nan, -math.inf]), torch.ones(D - 2))))
    x = torch.stack(rows).to(torch.bfloat16)[:, None]
    n = x.shape[0]
    table, seq, start, pages = _layout_on_device([n], [n], 32)
    cache = ci.PagedKVCache(pages, 32, 1, D, kind="int4", device=DEV)
    ci.paged_kv_append(cache, x.to(DEV), x.flip(0).contiguous().to(DEV), table, seq, start)
    k, v = ci.paged_kv_read(cache, table, seq, start, tokens=n)
    want = R.stored(x, "int4").float().to(torch.bfloat16)
    assert torch.equal(k.cpu().nan_to_num(7e30), want.nan_to_num(7e30))
    assert torch.equal(v.cpu().nan_to_num(7e30), want.flip(0).nan_to_num(7e30))


def test_what_does_not_exist_is_left_out_and_reported():
    """Pages outside the cache, positions beyond the rotary table, lengths beyond the block table, row offsets outside the
    rows: nothing is stored for them, nothing else changes, and the device status says so."""
    ci = _ci()
    H, D, page = 2, 64, 32
    table, seq, start, pages = _layout_on_device([40, 40], [40, 40], page)
    k, v = _put(R.normal(80, H, D, seed=1), R.normal(80, H, D, seed=2))
    good = ci.PagedKVCache(pages, page, H, D, device=DEV)
    ci.paged_kv_append(good, k, v, table, seq, start)
    assert ci.device_status() == 0

    def run(table=table, seq=seq, start=start, **kw):
        cache = ci.PagedKVCache(pages, page, H, D, device=DEV)
        ci.paged_kv_append(cache, k, v, table, seq, start, **kw)
        with pytest.raises(RuntimeError, match="do not exist"):
            ci.device_status()
        assert ci.device_status() == 0
        return cache

    def held(cache, row, tokens):
        return ci.paged_kv_read(cache, table[row:row + 1], torch.tensor([tokens], dtype=torch.int32).to(DEV),
                                torch.tensor([0, tokens], dtype=torch.int32).to(DEV), tokens=tokens)[0].cpu()

    for bad in (-1, pages, 1 << 30):
        t = table.clone()
        t[0, 1] = bad
        cache = run(table=t)
        assert torch.equal(held(cache, 0, 32), k[:32].cpu()) and torch.equal(held(cache, 1, 40), k[40:].cpu())
        assert not cache.data[table[0, 1].item()].any()
    cache = run(rotary=ci.rotary_table(33, D, device=DEV))
    assert not held(cache, 0, 40)[33:].any() and held(cache, 0, 40)[:33].any()
    cache = run(seq=torch.tensor([40, page * table.shape[1] + 40], dtype=torch.int32).to(DEV))
    assert torch.equal(held(cache, 0, 40), k[:40].cpu())
    cache = run(start=torch.tensor([0, 40, 120], dtype=torch.int32).to(DEV))
    assert torch.equal(held(cache, 0, 40), k[:40].cpu())
    run(start=torch.tensor([-5, 40, 80], dtype=torch.int32).to(DEV))
    # attention: a page that is none of the cache's is a run of keys nobody sees
    q = R.normal(2, 4, D, seed=3).to(DEV)
    t = table.clone()
    t[0, 0] = pages + 3
    got = ci.paged_attention(q, good, t, seq)
    with pytest.raises(RuntimeError, match="do not exist"):
        ci.device_status()
    want, _, mass, worst = R.attention(q[:1].cpu(), k[32:40].double().cpu(), v[32:40].double().cpu(), 7, D ** -0.5)
    _compare(got[:1], want, R.attention_bound(want, mass, worst, D))
    same = ci.paged_attention(q, good, table, seq)
    assert torch.equal(got[1], same[1])
    with torch.no_grad():
        big = ci.paged_attention(q, good, table, torch.tensor([1 << 30, 40], dtype=torch.int32).to(DEV))
    with pytest.raises(RuntimeError, match="do not exist"):
        ci.device_status()
    assert torch.equal(big[1], same[1])


def test_rows_behind_the_last_sequence_are_left_alone():
    ci = _ci()
    H, D = 2, 128
    for kind in ("bf16", "int4"):
        f = Filled([50, 33], [20, 3], 4, H, D, kind)
        T = 30  # 23 rows belong to a sequence
        q = torch.cat((f.q, torch.full((7, 4, D), math.nan, dtype=torch.bfloat16))).to(DEV)
        out = torch.full((T, 4, D), 5.0, dtype=torch.bfloat16, device=DEV)
        ci.paged_attention(q, *f.args(), out=out)
        assert (out[23:] == 5.0).all()
        want, _, bound = f.expect()
        _compare(out[:23], want, bound)
        before = f.cache.data.clone()
        turned = torch.full((T, 4, D), 5.0, dtype=torch.bfloat16, device=DEV)
        k = torch.cat([x[-n:] for x, n in zip(f.k, f.news)] + [torch.full((7, H, D), math.nan, dtype=torch.bfloat16)]).to(DEV)
        v = torch.cat([x[-n:] for x, n in zip(f.v, f.news)] + [torch.full((7, H, D), math.nan, dtype=torch.bfloat16)]).to(DEV)
        ci.paged_kv_append(f.cache, k, v, f.table, f.seq, f.start, q=q, q_out=turned)
        assert (turned[23:] == 5.0).all() and torch.equal(turned[:23].cpu(), f.q)
        assert torch.equal(f.cache.data.view(torch.uint8), before.view(torch.uint8))
        rk, rv = torch.full((2, T, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
        ci.paged_kv_read(f.cache, f.table, f.seq, f.start, k_out=rk, v_out=rv)
        assert (rk[23:] == 5.0).all() and (rv[23:] == 5.0).all()
        assert ci.device_status() == 0


# ---- attention: single tokens -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (16, 2), (24, 2), (40, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3), (1, 0), (33, 70)])
def test_single_tokens(kind, dim, heads, kv_heads, window, sinks):
    """Group sizes from one query head per kv head to more than a tile's rows; lengths of one, at and around the ends of
    blocks; windows that end inside a block and sinks that reach into the window."""
    ci = _ci()
    lens = [1, 31, 32, 33, 100, 260]
    f = Filled(lens, [1] * len(lens), heads, kv_heads, dim, kind, page=64, seed=dim + heads, scale=2.0)
    got, lse = ci.paged_attention(f.q.to(DEV), *f.args(rows=False), window=window, sinks=sinks, return_lse=True)
    want, want_lse, bound = f.expect(window, sinks)
    _compare(got, want, bound)
    assert torch.allclose(lse.double().cpu(), want_lse, rtol=0, atol=1e-3)
    # the same rows named by offsets, and with bounds on the lengths: other kernels of the same sums
    rows = ci.paged_attention(f.q.to(DEV), *f.args(), window=window, sinks=sinks, max_query_len=1, max_seq_len=260)
    _compare(rows, want, bound)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([2000], 8, 2, 128), ([700, 1, 1500, 64, 900], 3, 3, 64),
                                                     ([1100] * 3, 32, 2, 64)])
def test_items_that_are_cut(kind, lens, heads, kv_heads, dim):
    """Long sequences among short ones: their keys are shared out between workgroups and joined."""
    ci = _ci()
    f = Filled(lens, [1] * len(lens), heads, kv_heads, dim, kind, page=32, seed=3, scale=2.0)
    for window, sinks in ((0, 0), (600, 10)):
        got, lse = ci.paged_attention(f.q.to(DEV), *f.args(rows=False), window=window, sinks=sinks, return_lse=True)
        want, want_lse, bound = f.expect(window, sinks)
        _compare(got, want, bound)
        assert torch.allclose(lse.double().cpu(), want_lse, rtol=0, atol=1e-3)


def test_more_sequences_than_threads_of_a_workgroup():
    ci = _ci()
    lens = [1 + (i * 37) % 90 for i in range(300)]
    for news, bound_on in (([1] * 300, {}), ([1 + i % 2 if lens[i] > 1 else 1 for i in range(300)], dict(max_query_len=2))):
        f = Filled(lens, news, 2, 1, 64, "bf16", page=32, seed=8)
        want, _, bound = f.expect()
        for kw in ({}, dict(max_seq_len=90)):
            got = ci.paged_attention(f.q.to(DEV), *f.args(rows=sum(news) != 300), **bound_on, **kw)
            _compare(got, want, bound)


def test_empty_places_and_empty_calls():
    ci = _ci()
    for kind in ("bf16", "int4"):
        f = Filled([5, 0, 40], [1, 0, 1], 4, 2, 64, kind)
        q = torch.cat((f.q[:1], torch.full((1, 4, 64), 3.0, dtype=torch.bfloat16), f.q[1:])).to(DEV)
        got, lse = ci.paged_attention(q, *f.args(rows=False), return_lse=True)
        want, _, bound = f.expect()
        _compare(got[[0, 2]], want, bound)
        assert not got[1].any() and (lse[1] == -math.inf).all()
        assert ci.device_status() == 0
        empty = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
        none = torch.empty(0, dtype=torch.int32, device=DEV)
        assert ci.paged_attention(empty, f.cache, f.table[:0], none).shape == (0, 4, 64)
        assert ci.paged_kv_append(f.cache, empty[:, :2], empty[:, :2], f.table[:0], none) is None
        assert ci.paged_kv_read(f.cache, f.table[:0], none)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("fill", [0xFF, 0x7F])
def test_memory_behind_a_sequence_need_not_hold_numbers(kind, fill):
    """Pages filled with NaN and infinities before the sequences are stored: nothing of them reaches a result, for single
    tokens and for prompts, also where a page or a block ends behind the sequence and where a window begins inside one."""
    ci = _ci()
    f = Filled([1, 33, 95], [1, 1, 1], 4, 2, 128, kind, fill=fill)
    for kw in ({}, dict(window=20, sinks=2)):
        got = ci.paged_attention(f.q.to(DEV), *f.args(rows=False), **kw)
        want, _, bound = f.expect(**kw)
        _compare(got, want, bound)
    g = Filled([33, 300], [33, 290], 4, 2, 128, kind, fill=fill)
    for kw in ({}, dict(window=50, sinks=2)):
        want, _, bound = g.expect(**kw)
        for n in (0, 2):
            got = ci.paged_attention(g.q.to(DEV), *g.args(), max_query_len=n, **kw)
            _compare(got, want, bound)


# ---- attention: many rows ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (6, 2, 128), (8, 1, 64)])
@pytest.mark.parametrize("lens,news", [([130], [130]), ([300, 1, 47], [70, 1, 47])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5), (7, 0)])
def test_prompts(kind, heads, kv_heads, dim, lens, news, window, sinks):
    """Whole prompts and later parts of them, ragged, with groups that do not divide a tile; by the kernel for many rows
    and, told that sequences are short, by the kernel for few."""
    ci = _ci()
    f = Filled(lens, news, heads, kv_heads, dim, kind, seed=21, scale=1.5)
    want, want_lse, bound = f.expect(window, sinks)
    for longest in (max(news), 2):
        got, lse = ci.paged_attention(f.q.to(DEV), *f.args(), window=window, sinks=sinks, max_query_len=longest,
                                      return_lse=True)
        _compare(got, want, bound)
        assert torch.allclose(lse.double().cpu(), want_lse, rtol=0, atol=1e-3)


def test_a_prompt_that_fills_the_chip():
    """Enough rows for the kernel that shares keys between wavefronts on a card of 256 CUs."""
    ci = _ci()
    for kind in ("bf16", "int4"):
        f = Filled([1030, 777], [1030, 500], 16, 8, 128, kind, seed=31)
        for kw in ({}, dict(window=300, sinks=9)):
            got = ci.paged_attention(f.q.to(DEV), *f.args(), **kw)
            want, _, bound = f.expect(**kw)
            _compare(got, want, bound, (kind, kw))


def test_scale_strides_and_outputs():
    """A scale of one's own; queries and outputs as slices of wider tensors, heads before rows; a table that is a slice."""
    ci = _ci()
    f = Filled([90, 60], [40, 60], 6, 2, 128, "bf16", seed=41)
    packed = torch.full((100, 11, 160), 9.0, dtype=torch.bfloat16, device=DEV)
    q = packed[:, 2:8, 8:136]
    q.copy_(f.q)
    wide = torch.full((3, f.table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    wide[:2, :f.table.shape[1]] = f.table
    out = torch.full((6, 100, 128), 2.0, dtype=torch.bfloat16, device=DEV)
    got = ci.paged_attention(q, f.cache, wide[:2, :f.table.shape[1]], f.seq, f.start, scale=0.05, out=out.transpose(0, 1))
    want, _, bound = f.expect(scale=0.05)
    _compare(got, want, bound)
    assert got.data_ptr() == out.data_ptr()
    k = torch.cat(f.k).to(DEV).transpose(0, 1).contiguous().transpose(0, 1)  # heads before rows
    v = torch.cat(f.v).to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    rows = torch.tensor([0, 90, 150], dtype=torch.int32, device=DEV)
    again = ci.PagedKVCache(f.cache.num_pages, 64, 2, 128, device=DEV)
    ci.paged_kv_append(again, k, v, wide[:2, :f.table.shape[1]], f.seq, rows)
    assert torch.equal(again.data, f.cache.data)
    # queries turned in place are the ones turned into another tensor
    table = ci.rotary_table(100, 128, device=DEV)
    one = ci.paged_kv_append(again, k[:100], v[:100], f.table, f.seq, f.start, q=q, rotary=table)
    two = ci.paged_kv_append(again, k[:100], v[:100], f.table, f.seq, f.start, q=q, rotary=table, q_out=q)
    assert two.data_ptr() == q.data_ptr() and torch.equal(one, two)
    assert (packed[:, :2] == 9.0).all() and (packed[:, 8:] == 9.0).all() and (packed[:, :, 136:] == 9.0).all()


def test_scores_far_apart_and_beyond_numbers():
    """Scores of thousands (all weight on one key), a score of infinity (NaN, as the formula says), keys of minus infinity
    (no weight); the other rows are not touched by them."""
    ci = _ci()
    f = Filled([64, 64, 64], [1, 1, 1], 2, 2, 64, "bf16", seed=51)
    k = [x.clone() for x in f.k]
    k[0] = (k[0].float() * 300).to(torch.bfloat16)
    q = f.q.clone()
    q[1] = q[1].abs()
    k[1][40] = math.inf
    k[2][3] = -math.inf
    q[2] = q[2].abs()
    rows = torch.tensor([0, 64, 128, 192], dtype=torch.int32, device=DEV)
    ci.paged_kv_append(f.cache, torch.cat(k).to(DEV), torch.cat(f.v).to(DEV), f.table, f.seq, rows)
    got = ci.paged_attention(q.to(DEV), *f.args(rows=False)).double().cpu()
    assert got[1].isnan().all()
    for b in (0, 2):
        want, _, mass, worst = R.attention(q[b:b + 1], k[b].double(), f.v[b].double(), 63, 64 ** -0.5)
        worst = worst if math.isfinite(worst) else 100.0
        _compare(got[b:b + 1], want, R.attention_bound(want, mass, worst, 64))


def test_other_streams_and_graphs():
    """Operators on a stream of their own; a captured step (append, then attention that cuts items) replayed with new
    contents, lengths and pages, eager work in between; two captured steps replayed in turn share nothing."""
    ci = _ci()
    if not torch.cuda.is_available() or DEV != "cuda" or type(torch.cuda.current_stream()).__name__ == "_Stream":
        pytest.skip("needs streams")
    H, G, D, page, B = 8, 2, 128, 32, 3
    lens = [900, 33, 400]
    table, _, _, pages = _layout_on_device([l + 8 for l in lens], [1] * B, page)
    graphs = []
    for kind in ("bf16", "int4"):
        cache = ci.PagedKVCache(pages, page, G, D, kind=kind, device=DEV)
        f = dict(cache=cache, kind=kind, seq=torch.tensor(lens, dtype=torch.int32, device=DEV),
                 qkv=torch.zeros(B, H + 2 * G, D, dtype=torch.bfloat16, device=DEV), rotary=ci.rotary_table(1000, D, device=DEV))
        f["k"] = [R.normal(l - 1, G, D, seed=60 + b) for b, l in enumerate(lens)]
        f["v"] = [R.normal(l - 1, G, D, seed=70 + b) for b, l in enumerate(lens)]
        rows = torch.tensor([0] + [l - 1 for l in lens]).cumsum(0).to(torch.int32).to(DEV)
        ci.paged_kv_append(cache, torch.cat(f["k"]).to(DEV), torch.cat(f["v"]).to(DEV), table, f["seq"] - 1, rows)

        def step(f=f):
            q = ci.paged_kv_append(f["cache"], f["qkv"][:, H:H + G], f["qkv"][:, H + G:], table, f["seq"], q=f["qkv"][:, :H],
                                   rotary=f["rotary"])
            return ci.paged_attention(q, f["cache"], table, f["seq"])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f["eager"] = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f["out"] = step()
        f["graph"], f["step"] = g, step
        graphs.append(f)
    for t in range(4):
        for f in graphs:
            f["qkv"].copy_(R.normal(B, H + 2 * G, D, seed=80 + t).to(DEV))
            if t:
                f["seq"].add_(1)
            f["out"].fill_(7.0)
        for f in graphs:
            f["graph"].replay()
        torch.cuda.synchronize()
        for f in graphs:
            qkv = f["qkv"].cpu()
            pos = f["seq"].cpu().long() - 1
            for b in range(B):
                at = pos[b:b + 1]
                turn = lambda x: R.rotate(x[None], at, f["rotary"].cpu())  # noqa: E731
                f["k"][b] = torch.cat((f["k"][b], turn(qkv[b, H:H + G])))
                f["v"][b] = torch.cat((f["v"][b], qkv[b, H + G:][None]))
                k, v = R.stored(f["k"][b], f["kind"]), R.stored(f["v"][b], f["kind"])
                want, _, mass, worst = R.attention(turn(qkv[b, :H]), k, v, int(at), D ** -0.5)
                if f["kind"] == "int4":
                    mass = 2 * mass + R.attention(turn(qkv[b, :H]), k, R.pairs(f["v"][b])[1].abs().expand(v.shape), int(at), D ** -0.5)[0]
                _compare(f["out"][b:b + 1], want, R.attention_bound(want, mass, worst, D), (t, b, f["kind"]))
            assert torch.equal(f["out"], f["step"]())  # eager work between the replays, the same bits
        junk = torch.randn(1 << 20, device=DEV)  # (so does this)
        junk.sum().item()


def test_results_do_not_hang_on_timing():
    """The same call many times over gives the same bits (shares and joins are in a fixed order)."""
    ci = _ci()
    f = Filled([700, 3, 1300], [1, 1, 1], 4, 1, 128, "bf16", seed=91)
    first = ci.paged_attention(f.q.to(DEV), *f.args(rows=False))
    for _ in range(5):
        assert torch.equal(first, ci.paged_attention(f.q.to(DEV), *f.args(rows=False)))


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("lens,news,longest", [([90], [90], 0), ([40, 300], [3, 6], 2), ([1500], [1500], 0), ([900], [2], 2)])
def test_what_a_row_does_not_see_may_be_anything(kind, lens, news, longest):
    """Keys and values of infinities and NaN at tokens that some rows of a tile see and others do not: those others get what
    they get without them, and the rows that see a NaN are NaN."""
    ci = _ci()
    heads, G, D, window, sinks = 4, 2, 64, 20, 1
    f = Filled(lens, news, heads, G, D, kind, seed=61)
    where = [l - n + n // 2 for l, n in zip(lens, news)]  # a token in the middle of the new ones
    k, v = [x.clone() for x in f.k], [x.clone() for x in f.v]
    for b, t in enumerate(where):
        v[b][t] = torch.tensor([math.inf, -math.inf, math.nan, 1.0] * (D // 4), dtype=torch.bfloat16)
        if b % 2:
            k[b][t] = math.nan
    whole = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)
    ci.paged_kv_append(f.cache, torch.cat(k).to(DEV), torch.cat(v).to(DEV), f.table, f.seq, whole)
    for kw in ({}, dict(window=window, sinks=sinks)):
        want, _, bound = f.expect(**kw)
        got = ci.paged_attention(f.q.to(DEV), *f.args(), max_query_len=longest, **kw).double().cpu()
        at = 0
        for l, n, t in zip(lens, news, where):
            p = torch.arange(l - n, l)
            sees = (p >= t) & ((p - t < window) | (t < sinks)) if kw else p >= t
            rows = slice(at, at + n)
            clean = got[rows][~sees]
            off = (clean - want[rows][~sees]).abs() - bound[rows][~sees]
            assert not len(off) or float(off.max()) <= 0, (kw, float(off.max()))
            assert not torch.isfinite(got[rows][sees][..., 2::4]).any()  # (the channels whose value is NaN)
            at += n
    assert ci.device_status() == 0


@pytest.mark.parametrize("kind", ["bf16", "int4"])
@pytest.mark.parametrize("lens,news,longest", [([700], [300], 0), ([700, 1450], [300, 260], 0), ([410, 100], [3, 1], 3)])
@pytest.mark.parametrize("window,sinks", [(50, 0), (50, 5), (97, 40), (20, 0)])
def test_pages_before_the_window_may_be_gone(kind, lens, news, longest, window, sinks):
    """Pages of 32 tokens that hold no key a new token sees are taken out of the table: the results stay, and nothing that
    does not exist is reported."""
    ci = _ci()
    f = Filled(lens, news, 8, 2, 64, kind, page=32, seed=71)
    kw = dict(window=window, sinks=sinks, max_query_len=longest)
    whole = ci.paged_attention(f.q.to(DEV), *f.args(), **kw)
    table = f.table.clone()
    for b, (l, n) in enumerate(zip(lens, news)):
        gone = torch.arange(table.shape[1]) * 32
        gone = (gone >= sinks) & (gone + 31 < l - n - window + 1)
        table[b, gone.to(DEV)] = -1
        assert gone.any() or l == 100
    got = ci.paged_attention(f.q.to(DEV), f.cache, table, f.seq, f.start, **kw)
    assert torch.equal(got, whole)
    assert ci.device_status() == 0
