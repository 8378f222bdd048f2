"""The benchmark's decoder on the 4-bit cache: every layer's attention, for the prompt and for single tokens, against plain
attention in 64 bits over the values that 4 bits stand for (tests/paged_ref.py), on the queries, keys and values the decoder
itself computed.  (Two decoders side by side do not stay together: a last bit of a linear's output that differs moves a code
in a hundred across its border, by a step of a third of the values' width.)"""
import pytest
import torch

import paged_ref as R
from test_gpu_model_paged import dense  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["int4", "bf16"])
def test_attention_inside_the_decoder(dense, kind):  # noqa: F811
    bm, dev, ops, prompt = dense
    s = bm.Shape
    worst_of, calls = [], []

    class Checked(bm.Decoder):
        def __init__(self):
            super().__init__(ops, 2, 90, dev, "paged-int4" if kind == "int4" else "paged")
            self.rows = [None, None]

        def _paged_context(self, l, qkv, lens, start, T):
            got = super()._paged_context(l, qkv, lens, start, T)
            q, k, v = qkv.split((s.heads, s.kv_heads, s.kv_heads), 1)
            first = int(lens[0]) - T
            pos = torch.arange(first, first + T, device=dev)
            new = [R.rotate(k, pos, self.rotary), v]
            self.rows[l] = new if first == 0 else [torch.cat(x) for x in zip(self.rows[l], new)]
            k, v = (R.stored(x.cpu(), kind).to(dev) for x in self.rows[l])  # (powers of two are not exact on every device)
            size = v.abs() + (7.5 * R.pairs(self.rows[l][1].cpu())[0].to(dev) if kind == "int4" else 0.0)  # what a weight's rounding meets, at most
            heads = lambda x: x.repeat_interleave(s.heads // s.kv_heads, 1).transpose(0, 1).contiguous()  # noqa: E731
            q = R.rotate(q, pos, self.rotary).double().transpose(0, 1).contiguous()
            score = lambda q, k: torch.bmm(q, heads(k).transpose(1, 2).contiguous()) * s.head_dim ** -0.5  # noqa: E731
            hidden = torch.arange(k.shape[0], device=dev)[None] > pos[:, None]
            w = torch.softmax(score(q, k).masked_fill(hidden[None], float("-inf")), -1)
            want, mass = (torch.bmm(w, heads(x)).transpose(0, 1) for x in (v, size))
            bound = R.attention_bound(want, mass, float(score(q.abs(), k.abs()).max()), s.head_dim)
            worst_of.append(float(((got.double() - want).abs() - bound).max()))
            calls.append((l, T))
            return got

    with torch.no_grad():
        bm.teacher_forced(Checked(), prompt, prompt[:16].tolist())
    assert {(l, T) for l in (0, 1) for T in (1, len(prompt))} <= set(calls)
    assert max(worst_of) <= 0, max(worst_of)
