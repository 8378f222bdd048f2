"""Plain forms in 64 bits of the paged cache and the attention over it, for the tests: sequence by sequence, on the host."""
import math

import torch

HALF_STEP = 2.0 ** -8  # a rounding to bf16 is off by at most this, relative to the value


def layout(lens, news, page, width=None, seed=0, spare=2):
    """Block table (pages in no order, -1 behind what a sequence needs), lengths, row offsets; int32, on the host."""
    need = [-(-l // page) for l in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), width or max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    start = torch.tensor([0] + list(news)).cumsum(0).to(torch.int32)
    return table, torch.tensor(lens, dtype=torch.int32), start, total


def normal(*shape, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def rotate(x, positions, table):
    """x [T, H, D] turned in 64 bits and rounded once to bf16 (by way of 32 bits)."""
    half = table.shape[1] // 2
    c, s = table[positions].double()[:, None].split(half, -1)
    x = x.double()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1).float().to(torch.bfloat16)


def pairs(x):
    """(step, low) of rows of bf16 values, in 64 bits."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    width = (high - low) / 15.0
    e = torch.clamp(torch.frexp(width)[1] - 8, min=-133)  # bf16 holds eight bits, and nothing below 2^-133
    step = torch.ldexp(torch.ceil(torch.ldexp(width, -e)), e)  # rounded up
    return step, low


def codes(x):
    step, low = pairs(x)
    c = torch.round((x.double() - low) / torch.where(step > 0, step, torch.ones_like(step)))
    return torch.where(step > 0, c.clamp(0, 15), torch.zeros_like(c))


def stored(x, kind):
    """What rows of bf16 values are held as: themselves, or low + code * step, in 64 bits."""
    if kind == "bf16":
        return x.double()
    step, low = pairs(x)
    out = low + codes(x) * step
    wild = ~torch.isfinite(x.double()).all(-1, keepdim=True)
    return torch.where(wild, torch.full_like(out, math.nan), out)


def visible(positions, keys, window, sinks):
    p, j = positions[:, None], torch.arange(keys)[None]
    seen = j <= p
    if window:
        seen = seen & ((p - j < window) | (j < sinks))
    return seen


def attention(q, k, v, first, scale, window=0, sinks=0):
    """One sequence: q [n, H, D] at positions first .. , k and v [L, G, D] (64 bits).  Returns out, lse and, for the bound on
    the error of the kernels, sum of w |v|, and the largest sum of |q k| * scale of a score."""
    n, H, D = q.shape
    G = k.shape[1]
    q = q.double().view(n, G, H // G, D)
    seen = visible(first + torch.arange(n), k.shape[0], window, sinks)
    s = torch.einsum("ngrd,jgd->ngrj", q, k) * scale
    mag = (torch.einsum("ngrd,jgd->ngrj", q.abs(), k.abs()) * scale).masked_fill(~seen[:, None, None], 0.0)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - torch.where(torch.isinf(lse) & (lse < 0), torch.zeros_like(lse), lse)[..., None])
    vv = torch.where(seen.any(0)[:, None, None], v, torch.zeros_like(v))  # (what no row sees need not be a number)
    out = torch.einsum("ngrj,jgd->ngrd", w, vv).reshape(n, H, D)
    mass = torch.einsum("ngrj,jgd->ngrd", w, vv.abs()).reshape(n, H, D)
    worst = float(mag.nan_to_num(0.0).max()) if mag.numel() else 0.0
    return out, lse.reshape(n, H), mass, worst


def attention_bound(out, mass, worst, dim):
    """How far an element may be off.  Weights are rounded to bf16 once (half a step each: HALF_STEP of sum w |v|), the
    output once (HALF_STEP of it).  A score is a 32-bit sum of `dim`
    products, each addition off by 2^-24 of a partial sum of at most `worst`, then scaled and exponentiated (2^-21 of the
    largest power): twice its error, relative, moves a weight and the sum of weights.  4-bit operands carry 128 + code, at
    most 16 times what a code stands for, through the same 32-bit sums."""
    score = dim * 16 * worst * 2.0 ** -24 + 2.0 ** -21 * (worst + 1.0)
    weight = HALF_STEP + 2 * score + dim * 16 * 2.0 ** -24
    return 1.02 * weight * mass + 1.02 * HALF_STEP * out.abs() + 1e-30
