"""The benchmark's decoder (two layers, full widths, dense random weights) on the paged cache: append with rotation and
attention in every layer, prompt and single tokens, eager and as one graph replay per token."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dense():
    import bench_model as bm

    s, dev = bm.Shape, torch.device("cuda", 0)
    g = torch.Generator("cuda").manual_seed(5)
    draw = lambda k, n: bm.Dense((torch.randn(k, n, generator=g, device=dev) * 0.02).to(torch.bfloat16))  # noqa: E731
    width = (s.heads + 2 * s.kv_heads) * s.head_dim
    ops = {"qkv": [draw(s.hidden, width) for _ in range(2)], "o": [draw(s.heads * s.head_dim, s.hidden) for _ in range(2)],
           "gate_up": [draw(s.hidden, 2 * s.ffn) for _ in range(2)], "down": [draw(s.ffn, s.hidden) for _ in range(2)]}
    table = draw(1000, s.hidden).w
    ops["embed"] = lambda ids: table.index_select(0, ids)
    ops["head"] = lambda x: torch.matmul(x, table.t())
    prompt = torch.randint(0, 1000, (70,), generator=torch.Generator().manual_seed(6)).to(dev)
    return bm, dev, ops, prompt


@pytest.mark.parametrize("kv", ["paged", "paged-int4"])
def test_graph_replays_give_the_eager_tokens(dense, kv):
    bm, dev, ops, prompt = dense
    with torch.no_grad():
        eager, _ = bm.generate(bm.Decoder(ops, 2, 70 + 24 + 1, dev, kv), prompt, 24, False)
        graph, _ = bm.generate(bm.Decoder(ops, 2, 70 + 24 + 1, dev, kv), prompt, 24, True)
    assert graph == eager and len(set(eager)) > 1


def test_logits_on_the_paged_cache_are_those_on_the_static_one(dense):
    """Two bf16 pipelines that round at different places: the bar of the whole-model test on decompressed weights (1e-2 of
    the logit matrix in the Frobenius norm), for the prompt and sixteen fed tokens."""
    bm, dev, ops, prompt = dense
    ids = prompt[:16].tolist()
    with torch.no_grad():
        want = bm.teacher_forced(bm.Decoder(ops, 2, 90, dev), prompt, ids)
        got = bm.teacher_forced(bm.Decoder(ops, 2, 90, dev, "paged"), prompt, ids)
    assert float((got - want).norm() / want.norm()) <= 1e-2
    import comp_inference_amd as ci

    assert ci.device_status() == 0
