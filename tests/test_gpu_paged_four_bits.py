"""How exact attention over four bits is: the bound counts what is rounded and nothing else -- a weight times its step, once,
against a code's distance from the middle of the codes -- on values whose middles are large and whose output is small, where
rounding the middles, or rounding against the code itself, is seen: oracles that round so are outside the bound."""
import math

import pytest
import torch

import paged_ref as R
from test_gpu_paged import DEV, _ci, _layout_on_device

pytestmark = pytest.mark.gpu


def _bf16(x):
    return x.to(torch.bfloat16).double()


def _values(dim):
    """Two kinds of rows (bf16), [2, dim]: the same slope of 0.97 from end to end, far above zero and further below it, so that
    the average is near zero at the upper end, and both middles are rounded upwards by as much as can be had."""
    slope = torch.linspace(-0.97, 0.97, dim, dtype=torch.float64)

    def error(at):
        row = (at + slope).to(torch.bfloat16)[None]
        step, low = R.pairs(row)
        middle = low + 7.5 * step
        return float(_bf16(middle) - middle)

    up = max((2.0 + i / 64 for i in range(30)), key=error)
    down = max((-2.0 - i / 64 - 1.94 for i in range(-20, 20)), key=lambda x: error(x) - 0.01 * abs(x + up + 1.94))
    return torch.stack([(up + slope).to(torch.bfloat16), (down + slope).to(torch.bfloat16)])


def _case(dim, keys):
    """A query, keys and values: one key in four weighs 1 (one of those that any column of a tile works on, so that their weights
    count from it), all others the same p < 1, chosen so that p * step is rounded by nearly half a step of bf16.  Constant keys
    are stored exactly."""
    rows = _values(dim)
    v = rows[torch.arange(keys) // 8 % 2][:, None].contiguous()
    step, _ = R.pairs(rows[:1])
    q = torch.full((dim,), 1.0 / 64, dtype=torch.bfloat16)
    scale = dim ** -0.5
    unit = scale * dim / 64  # score of a constant key of 1

    def rounded(low):
        s = math.exp(unit * (low - 1.0)) * float(step)
        return abs(float(_bf16(torch.tensor(s, dtype=torch.float64))) / s - 1.0)

    low = max((1.0 - i / 256 for i in range(1, 128)), key=rounded)
    assert rounded(low) > 0.9 * R.HALF_STEP
    k = torch.full((keys, 1, dim), low, dtype=torch.bfloat16)
    k[torch.isin(torch.arange(keys) % 8, torch.tensor([0, 2]))] = 1.0
    return q, k, v


def _judge(q, k, v, n):
    """Of the last n rows: the result in 64 bits, the bound, and what the two coarser ways of rounding would give."""
    keys, dim = v.shape[0], v.shape[2]
    step, low = (x[:, 0] for x in R.pairs(v))
    code = R.codes(v)[:, 0]
    score = (k.double()[:, 0] @ q.double()) * dim ** -0.5
    worst = float((k.double().abs()[:, 0] @ q.double().abs()).max()) * dim ** -0.5
    p = torch.exp(score - score[0])
    seen = (torch.arange(keys)[None] <= torch.arange(keys - n, keys)[:, None]).double()
    total = seen @ p
    mean = lambda x: (seen @ x) / total[:, None]  # noqa: E731
    exact = mean(p[:, None] * (low + code * step))
    r = _bf16(p[:, None] * step)
    coarse = [mean(p[:, None] * low + r * code),                            # rounded against the code
              mean(p[:, None] * _bf16(low + 7.5 * step) + r * (code - 7.5))]  # middles rounded
    # weights times steps rounded once, against the distance from the middle; scores as paged_ref.attention_bound has them (4-bit
    # operands 128 + code through 32-bit sums), on everything a weight multiplies; the sums of the values, one 32-bit rounding per
    # key of at most 143 steps and the low; the output
    off = dim * 16 * worst * 2.0 ** -24 + 2.0 ** -21 * (worst + 1.0)
    bound = (R.HALF_STEP * mean(p[:, None] * step * (code - 7.5).abs()) + 2 * off * mean(p[:, None] * (low + code * step).abs())
             + keys * 2.0 ** -24 * mean(p[:, None] * (143 * step + low.abs())) + R.HALF_STEP * exact.abs())
    return exact, bound * 1.02, coarse


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys,n,heads,kv_heads,bounds", [
    pytest.param(70, 1, 4, 1, {}, id="few"), pytest.param(100, 5, 6, 2, dict(max_query_len=8), id="few_several"),
    pytest.param(300, 300, 64, 8, {}, id="many"), pytest.param(2400, 290, 64, 8, {}, id="many_in_shares")])
def test_only_the_weights_are_rounded(dim, keys, n, heads, kv_heads, bounds):
    ci = _ci()
    q, k, v = _case(dim, keys)
    exact, bound, coarse = _judge(q, k, v, n)
    if keys <= 300:  # (over many more keys the 32-bit sums have their share of the bound)
        # (middles are a matter of the kernel for many rows; a row that sees one kind of values shows them best)
        for c in coarse[:2 if n == keys else 1]:
            assert float(((c - exact).abs() / bound).max()) > 1.2, "the bound lets a coarser rounding through"
    table, seq, start, pages = _layout_on_device([keys], [n], 64)
    cache = ci.PagedKVCache(pages, 64, kv_heads, dim, kind="int4", device=DEV)
    rows = torch.tensor([0, keys], dtype=torch.int32).to(DEV)
    ci.paged_kv_append(cache, k.expand(keys, kv_heads, dim).contiguous().to(DEV), v.expand(keys, kv_heads, dim).contiguous().to(DEV), table, seq, rows)
    got = ci.paged_attention(q.expand(n, heads, dim).contiguous().to(DEV), cache, table, seq, start, **bounds).double().cpu()
    off = (got - exact[:, None]).abs() - bound[:, None]
    assert float(off.max()) <= 0, float(off.max())
