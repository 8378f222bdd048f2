"""The serving operators around the compressed linears, as measurable cases: keys and values appended to a paged cache
(rotated on the way), and attention over that cache -- full or over a sliding window with a few first tokens that
stay visible -- for single tokens and for whole prompts, with the cache in bf16 or in 4 bits.

A batch is described as a server holds it: `query_start` [B + 1] cuts the rows of q, k and v into sequences,
`seq_lens` [B] counts the tokens of each sequence with the new ones, `block_table` [B, P] names its pages.  The new
tokens of a sequence are its last ones.

Formulas (i a query at position p_i, j a key, h a query head, g = h // (heads / kv_heads)):

  rotation   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin), pairs (d, d + D/2), cos and sin from the table's row p
  attention  out[i, h] = sum_j w_j v[j, g],  w = softmax over the visible j of scale * q[i, h] . k[j, g];
             j is visible when j <= p_i and (no window, or p_i - j < window, or j < sinks)
  4 bits     per token and head: low = min, step = (max - min) / 15 rounded up to bf16,
             code = rint((x - low) / step) in 0..15; a stored value stands for low + code * step
"""
import math

import torch

own = False

BLOCK = 32  # tokens whose keys lie together in the cache (one matrix tile)


# ---- the cases ------------------------------------------------------------------------------------------------------

def _case(name, op, kind, seqs, shortest, longest, new, heads=32, kv_heads=8, dim=128, page=64, window=0, sinks=0):
    return dict(name=name, op=op, kind=kind, seqs=seqs, shortest=shortest, longest=longest, new=new, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, window=window, sinks=sinks)


def listed():
    return [
        # one chat, one new token, after a prompt of 128 and half of its 256 answers: latency is everything
        _case("append_one_token", "append", "bf16", 1, 257, 257, 1),
        # a serving step of 64 chats, one token each
        _case("append_decode_64_int4", "append", "int4", 64, 130, 1000, 1),
        # prompts of several users taken in together
        _case("append_prompts_ragged", "append", "bf16", 7, 333, 2100, 2100),
        # the same into the 4-bit cache, heads of 64, another page size
        _case("append_prompts_int4", "append", "int4", 4, 1001, 4097, 4097, heads=16, kv_heads=2, dim=64, page=128),
        # one chat: the shortest context the model benchmark decodes over
        _case("decode_one_chat", "attend", "bf16", 1, 300, 300, 1),
        # many chats of very different length, window and sinks: what a long-running server holds
        _case("decode_window_ragged_64", "attend", "bf16", 64, 17, 32768, 1, window=4096, sinks=4),
        # few long documents, every key visible
        _case("decode_long_documents", "attend", "bf16", 4, 60001, 131072, 1),
        # a prompt read in one pass
        _case("prompt_8192", "attend", "bf16", 1, 8192, 8192, 8192),
        # ragged prompts under a window, heads of 64, no shared key heads
        _case("prompts_window_ragged", "attend", "bf16", 6, 257, 6001, 6001, heads=12, kv_heads=12, dim=64, page=32,
              window=1000, sinks=5),
        # 48 chats over the 4-bit cache
        _case("decode_int4_ragged_48", "attend", "int4", 48, 100, 32768, 1),
        # one long document over the 4-bit cache, one token
        _case("decode_int4_one_document", "attend", "int4", 1, 65531, 65531, 1, page=128),
        # the next part of a prompt behind what the 4-bit cache already holds
        _case("prompt_part_int4", "attend", "int4", 2, 9001, 16384, 1500),
    ]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend"])
    kind = rng.choice(["bf16", "int4"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    page = rng.choice([32, 64, 128, 256])
    window, sinks = (_log_int(rng, 1, 8192), rng.choice([0, 1, 4, 7, 40])) if rng.random() < 0.5 else (0, 0)
    form = rng.choice(["decode", "decode", "prompt", "part"])
    if form == "decode":
        seqs = _log_int(rng, 1, 96)
        longest = _log_int(rng, 1, 400000 // seqs if seqs > 8 else 65536)
        new = 1
    elif form == "prompt":
        seqs = _log_int(rng, 1, 8)
        longest = _log_int(rng, 2, 8192 // seqs)
        new = longest
    else:
        seqs = _log_int(rng, 1, 8)
        longest = _log_int(rng, 300, 16384)
        new = _log_int(rng, 2, min(longest, 2000 // seqs))
    shortest = longest if rng.random() < 0.3 else _log_int(rng, 1, longest)
    if op == "append":  # (the cache comes back whole: keep it no larger than the listed ones)
        shortest, longest = min(shortest, 4096), min(longest, 4096)
        new = min(new, longest)
    return {k: v for k, v in _case("", op, kind, seqs, shortest, longest, new, heads, kv_heads, dim, page, window,
                                   sinks).items() if k != "name"}


def _lens(case):
    """Length of every sequence, and how many of its tokens are new: between the case's bounds, in mixed order."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    lens = [hi if n == 1 else lo + (hi - lo) * ((i * 7 + 3) % n) // (n - 1) for i in range(n)]
    if n % 7 == 0 and n > 1:  # (7 and n share a factor: a plain ramp)
        lens = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return lens, [min(l, case["new"]) for l in lens]


def work(case):
    lens, news = _lens(case)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    stored = 4 * D if case["kind"] == "bf16" else D + 8  # bytes of a token's key and value, per head
    T = sum(news)
    if case["op"] == "append":
        moved = T * (2 * 2 * H * D + 2 * 2 * G * D + 4 * D + G * stored)
        if case["kind"] == "int4":
            moved += T * (G * stored + 2 * 2 * G * D)  # read back as values
        return {"bytes": moved, "flops": 3 * T * (H + G) * D}
    w, s = case["window"], case["sinks"]
    keys = pairs = 0
    for ln, n in zip(lens, news):
        first = ln - n
        if not w:
            keys += ln
            pairs += n * first + n * (n + 1) // 2
            continue
        start = max(0, first - w + 1)
        keys += ln - start + min(s, start)
        for p in range(first, ln):
            b = max(0, p - w + 1)
            pairs += p + 1 - b + min(s, b)
    return {"bytes": keys * G * stored + T * H * D * 4, "flops": 4 * D * H * pairs}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _sequences(case, seed):
    """(q, k, v) of one sequence after the other: queries of its new tokens, keys and values of all of them.  Some
    channels of the keys are far from zero and some are wide, as they are in trained models."""
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    G, D = case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    wide, off = torch.exp(0.4 * normal(G, D)), normal(G, D)
    lens, news = _lens(case)
    for ln, n in zip(lens, news):
        q = (1.5 * normal(n, case["heads"], D)).to(torch.bfloat16)
        k = (normal(ln, G, D) * wide + off).to(torch.bfloat16)
        v = normal(ln, G, D).to(torch.bfloat16)
        yield q, k, v


def _batch(case, seed):
    """Page table and lengths; the pages are handed out in no order, unused entries hold -1."""
    lens, news = _lens(case)
    P = case["page"]
    need = [-(-l // P) for l in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    start = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    return dict(table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32).cuda(), start=start.cuda(),
                host_lens=lens, host_news=news, pages=total)


def _rotary(rows, dim):
    """cos | sin of every position's angles, fp32, from angles in 64 bits."""
    inv = 500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat((ang.cos(), ang.sin()), 1).to(torch.float32).cuda()


def _block_elements(case):
    return 2 * BLOCK * case["dim"]


def prepare(case, seed):
    st = dict(case=case, **_batch(case, seed))
    G, D, P = case["kv_heads"], case["dim"], case["page"]
    if own:
        import comp_inference_amd as ci

        st["ci"] = ci
        st["cache"] = ci.PagedKVCache(st["pages"], P, G, D, kind=case["kind"], device="cuda")
    decode = max(st["host_news"]) == 1
    st["query_start"] = None if decode else st["start"]  # one token each: the form without row offsets
    if case["op"] == "append":
        g = torch.Generator("cuda").manual_seed(seed)
        T = sum(st["host_news"])
        st["qkv"] = torch.randn(T, case["heads"] + 2 * G, D, generator=g, device="cuda").to(torch.bfloat16)
        st["rotary"] = _rotary(max(st["host_lens"]) + 5, D)
        if case["kind"] == "bf16":
            held = torch.randn(st["pages"], G, P // BLOCK, _block_elements(case), generator=g,
                               device="cuda").to(torch.bfloat16)
            if own:
                st["cache"].data.copy_(held.view(st["cache"].data.shape))
            else:
                st["data"] = held
        elif not own:
            st["codes"] = [torch.zeros(st["pages"], P, G, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
            st["grid"] = [torch.zeros(st["pages"], P, G, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        return st
    st["max_seq_len"] = case["longest"]  # (a server knows its longest sequence)
    st["max_query_len"] = max(st["host_news"])
    qs = []
    if not own:
        st["pools"] = [torch.zeros(st["pages"], P, G, D, dtype=torch.bfloat16 if case["kind"] == "bf16" else torch.uint8,
                                   device="cuda") for _ in range(2)]
        if case["kind"] == "int4":
            st["grid"] = [torch.zeros(st["pages"], P, G, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b, (q, k, v) in enumerate(_sequences(case, seed)):
        qs.append(q)
        ln = k.shape[0]
        if own:
            rows = torch.tensor([0, ln], dtype=torch.int32).cuda()
            st["ci"].paged_kv_append(st["cache"], k, v, st["table"][b:b + 1], st["lens"][b:b + 1], query_start=rows)
            continue
        pos = torch.arange(ln, device="cuda")
        page = st["table"][b].long()[pos // P]
        for i, x in enumerate((k, v)):
            if case["kind"] == "int4":
                x, st["grid"][i][page, pos % P] = _quantize(x)
            st["pools"][i][page, pos % P] = x
    st["q"] = torch.cat(qs)
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _positions(st):
    """Sequence and position of every new token."""
    lens, news = st["lens"].long(), torch.diff(st["start"].long())
    seq = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), news, output_size=st["qkv"].shape[0])
    row = torch.arange(seq.numel(), device="cuda")
    return seq, lens[seq] - news[seq] + row - st["start"].long()[seq]


def _rotated(x, cos, sin):
    """In 64 bits: a result next to the border of two bf16 numbers, or of two codes, falls on its own side."""
    a, b = x.double().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).float().to(torch.bfloat16)


def _quantize(x):
    """codes (uint8) and (step, low) in bf16 of every row of x.  In 64 bits: many values of a row lie on, or right
    beside, the border of two codes."""
    x = x.double()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    exact = (high - low) / torch.full_like(low, 15.0)
    step = exact.float()
    step = torch.where(step.double() < exact, torch.nextafter(step, torch.full_like(step, math.inf)), step)
    step = ((step.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32).double()  # up to the next bf16
    code = torch.where(step > 0, torch.round((x - low) / step), torch.zeros_like(x)).clamp(0, 15)
    return code.to(torch.uint8), torch.cat((step, low), -1).to(torch.bfloat16)


def _values(codes, grid):
    grid = grid.float()
    return grid[..., 1:] + codes.float() * grid[..., :1]


def _plain_append(st):
    case = st["case"]
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q, k, v = st["qkv"].split((H, G, G), 1)
    seq, pos = _positions(st)
    cos, sin = st["rotary"][pos].double()[:, None].chunk(2, -1)
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    page, slot = st["table"][seq, pos // P].long(), pos % P
    T = pos.numel()
    if case["kind"] == "int4":
        back = []
        for i, x in enumerate((k, v)):
            codes, grid = _quantize(x)
            st["codes"][i][page, slot] = codes
            st["grid"][i][page, slot] = grid
            back.append(_values(st["codes"][i][page, slot], st["grid"][i][page, slot]).to(torch.bfloat16))
        return q, back[0], back[1]
    # the cache's order: per block of 32 tokens the keys as [D/16][2][32 tokens][8], then the values as
    # [2 halves of 16 tokens][D/32][2][32 channels][2][4], token = 16 half + 8 a + 4 h + b
    kv = st["data"].view(-1, G, P // BLOCK, 2, BLOCK * D)
    blk, t = slot // BLOCK, slot % BLOCK
    kv[:, :, :, 0].view(-1, G, P // BLOCK, D // 16, 2, 32, 8)[page, :, blk, :, :, t] = k.reshape(T, G, D // 16, 2, 8)
    kv[:, :, :, 1].view(-1, G, P // BLOCK, 2, D // 32, 2, 32, 2, 4)[
        page, :, blk, t // 16, :, t // 4 % 2, :, t // 8 % 2, t % 4] = v.reshape(T, G, D // 32, 32)
    return q, st["data"]


def _plain_attend(st):
    case = st["case"]
    H, G, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty_like(st["q"])
    at = 0
    for b, (ln, n) in enumerate(zip(st["host_lens"], st["host_news"])):
        page = st["table"][b, :-(-ln // P)].long()
        k, v = (x[page].reshape(-1, G, D)[:ln] for x in st["pools"])
        if case["kind"] == "int4":
            gk, gv = (x[page].reshape(-1, G, 2)[:ln] for x in st["grid"])
            k, v = _values(k, gk), _values(v, gv)
        k = k.float().permute(1, 2, 0).contiguous()  # [G, D, ln]
        v = v.float().transpose(0, 1).contiguous()   # [G, ln, D]
        step = max(1, (1 << 28) // (H * ln))
        for r in range(0, n, step):
            m = min(step, n - r)
            q = st["q"][at + r:at + r + m].float().view(m, G, H // G, D).permute(1, 0, 2, 3).reshape(G, -1, D)
            s = torch.bmm(q, k).view(G, m, H // G, ln) * D ** -0.5
            p = ln - n + r + torch.arange(m, device="cuda")[:, None]
            j = torch.arange(ln, device="cuda")[None]
            seen = j <= p
            if case["window"]:
                seen = seen & ((p - j < case["window"]) | (j < case["sinks"]))
            s = s.masked_fill(~seen[None, :, None], float("-inf"))
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.bmm(e.view(G, -1, ln), v) / e.sum(-1).view(G, -1, 1)
            out[at + r:at + r + m] = o.view(G, m, H // G, D).permute(1, 0, 2, 3).reshape(m, H, D).to(torch.bfloat16)
        at += n
    return out


# ---- one pass -------------------------------------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if not own:
        return _plain_append(st) if case["op"] == "append" else _plain_attend(st)
    ci = st["ci"]
    if case["op"] == "attend":
        return ci.paged_attention(st["q"], st["cache"], st["table"], st["lens"], query_start=st["query_start"],
                                  window=case["window"], sinks=case["sinks"], max_query_len=st["max_query_len"],
                                  max_seq_len=st["max_seq_len"])
    H, G = case["heads"], case["kv_heads"]
    qkv = st["qkv"]
    q = ci.paged_kv_append(st["cache"], qkv[:, H:H + G], qkv[:, H + G:], st["table"], st["lens"],
                           query_start=st["query_start"], q=qkv[:, :H], rotary=st["rotary"])
    if case["kind"] == "bf16":
        return q, st["cache"].data.view(-1, G, case["page"] // BLOCK, _block_elements(case))
    k, v = ci.paged_kv_read(st["cache"], st["table"], st["lens"], query_start=st["query_start"], tokens=qkv.shape[0])
    return q, k, v


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------

def _exact_stored(x):
    """What a row of 64-bit values is held as in 4 bits."""
    low = x.min(-1, keepdim=True).values
    width = (x.max(-1, keepdim=True).values - low) / 15
    m, e = torch.frexp(width)  # width = m 2^e, m in [0.5, 1): bf16 holds 8 bits of m
    step = torch.ldexp(torch.ceil(m * 256) / 256, e)
    safe = torch.where(step > 0, step, torch.ones_like(step))
    return low + torch.where(step > 0, torch.round((x - low) / safe).clamp(0, 15), torch.zeros_like(x)) * step


def _exact_append(case, seed):
    G, H, D, P = case["kv_heads"], case["heads"], case["dim"], case["page"]
    g = torch.Generator("cuda").manual_seed(seed)
    info = _batch(case, seed)
    T = sum(info["host_news"])
    x = torch.randn(T, H + 2 * G, D, generator=g, device="cuda").to(torch.bfloat16).double()
    table = _rotary(max(info["host_lens"]) + 5, D).double()
    pos = torch.cat([torch.arange(ln - n, ln) for ln, n in zip(info["host_lens"], info["host_news"])]).cuda()
    half = D // 2
    turn = torch.polar(torch.ones_like(table[:, :half]), torch.atan2(table[:, half:], table[:, :half]))
    size = torch.hypot(table[:, half:], table[:, :half])
    z = torch.complex(x[:, :H + G, :half], x[:, :H + G, half:]) * (turn * size)[pos][:, None]
    rot = torch.cat((z.real, z.imag), -1)
    q, k, v = rot[:, :H], rot[:, H:], x[:, H + G:]
    if case["kind"] == "int4":
        return q, None, _exact_stored(v)  # (the keys' codes hang on their rounding to bf16: no value of their own)
    held = torch.randn(info["pages"], G, P // BLOCK, _block_elements(case), generator=g, device="cuda")
    held = held.to(torch.bfloat16).double()
    flat = held.view(-1)
    seq = [b for b, n in enumerate(info["host_news"]) for _ in range(n)]
    page = info["table"][torch.tensor(seq).cuda(), pos // P].long()
    blk, t = pos % P // BLOCK, pos % BLOCK
    d = torch.arange(D, device="cuda")
    for head in range(G):
        base = (((page * G + head) * (P // BLOCK) + blk) * _block_elements(case))[:, None]
        flat[base + d // 16 * 512 + d // 8 % 2 * 256 + t[:, None] * 8 + d % 8] = k[:, head]
        t_ = t[:, None]
        flat[base + BLOCK * D + ((t_ // 16 * (D // 32) + d // 32) * 64 + t_ // 4 % 2 * 32 + d % 32) * 8
             + t_ // 8 % 2 * 4 + t_ % 4] = v[:, head]
    return q, held


def exact(case, seed):
    if case["op"] == "append":
        return _exact_append(case, seed)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    outs = []
    for q, k, v in _sequences(case, seed):
        q, k, v = q.double(), k.double(), v.double()
        if case["kind"] == "int4":
            k, v = _exact_stored(k), _exact_stored(v)
        n, ln = q.shape[0], k.shape[0]
        out = torch.empty_like(q)
        j = torch.arange(ln, device="cuda")
        for h in range(H):
            kh, vh = k[:, h // (H // G)], v[:, h // (H // G)]
            for r in range(0, n, 2048):
                p = torch.arange(ln - n + r, min(ln - n + r + 2048, ln), device="cuda")
                score = q[r:r + 2048, h] @ kh.T / math.sqrt(D)
                ahead = p[:, None] - j
                hidden = ahead < 0
                if case["window"]:
                    hidden |= (ahead >= case["window"]) & (j >= case["sinks"])
                score[hidden] = -math.inf
                out[r:r + 2048, h] = torch.softmax(score, -1) @ vh
        outs.append(out)
    return torch.cat(outs)
