"""The decode loop of examples/decode_loop.py: its logits against the same model
computed in 64 bits, its CUDA graph against its eager steps."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("decode_loop", os.path.join(ROOT, "examples", "decode_loop.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def exact_linear(layer, x):
    """An Int8Linear of 64-bit x, which the layer sees rounded to bf16."""
    x = x.bfloat16().double()
    scale = (x.abs().amax(1, keepdim=True) / 127.0).float().double()
    q = (x / scale).float().double().round().clamp(-127, 127)
    return (q @ layer.weight.double().T) * scale * layer.scale.double()


def exact_logits(model, prompt, rows):
    """Logits after the last token of each row (the tokens past the prompt)."""
    out = []
    for row in rows:
        tokens = torch.tensor(prompt + row, device="cuda")
        hidden = model.embedding[tokens].double()
        qkv = exact_linear(model.qkv, hidden).bfloat16().double().view(len(tokens), -1, model.dim)
        table = model.rope[:len(tokens)].double()
        turned = qkv.clone()
        half, n = model.dim // 2, model.heads + model.kv_heads
        a, b = qkv[:, :n, :half], qkv[:, :n, half:]
        c, s = table[:, None, 0], table[:, None, 1]
        turned[:, :n] = torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().double()
        q = turned[-1, :model.heads]
        k = turned[:, model.heads:n].repeat_interleave(model.heads // model.kv_heads, 1)
        v = turned[:, n:].repeat_interleave(model.heads // model.kv_heads, 1)
        p = torch.softmax(torch.einsum("hd,khd->hk", q, k) * model.dim ** -0.5, -1)
        mixed = torch.einsum("hk,khd->hd", p, v).bfloat16().reshape(1, -1)
        last = (hidden[-1:] + exact_linear(model.out, mixed).bfloat16().double()).bfloat16()
        out.append(exact_linear(model.head, last))
    return torch.cat(out)


@gpu
def test_logits_match_the_model_in_64_bits():
    """Rounding to bf16 and to 8 bits is made at the same places, so most
    entries agree; where a value lies next to a rounding boundary the
    projections' 8-bit integers differ by one step (1/127 of a row's largest),
    and the attention's own error is bf16's.  In norm the logits are within 4
    such roundings of the 8-bit steps: 4 / 127 / sqrt(12)."""
    ex = example()
    model = ex.ToyModel(vocab=1001, hidden=256, heads=6, kv_heads=2, dim=64, seed=3)
    gen = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, 1001, (150,), generator=gen).tolist()
    loop = ex.DecodeLoop(model, prompt, rows=5, steps=20)
    rows = [[prompt[-1]] for _ in range(5)]
    for _ in range(17):
        logits = loop.logits()
        fed = torch.randint(0, 1001, (5,), generator=gen)
        loop.tokens.copy_(fed)
        want = exact_logits(model, prompt, rows)
        err = (logits.double() - want).norm() / want.norm()
        assert float(err) <= 4 / 127 / 12 ** 0.5, float(err)
        for b in range(5):
            rows[b].append(int(fed[b]))


@gpu
def test_graph_equals_eager_steps():
    from miniserve_b200 import Sampler
    ex = example()
    model = ex.ToyModel(vocab=2003, hidden=128, heads=4, kv_heads=2, dim=64, seed=4)
    prompt = list(range(100))
    params = dict(temperature=torch.full((9,), 0.9, dtype=torch.float64, device="cuda"),
                  top_k=torch.full((9,), 40, dtype=torch.int32, device="cuda"),
                  top_p=torch.full((9,), 0.9, dtype=torch.float64, device="cuda"))
    uniforms = torch.rand((24, 9), generator=torch.Generator().manual_seed(6), dtype=torch.float64).cuda()
    sampler = Sampler()
    eager, graphed = (ex.DecodeLoop(model, prompt, rows=9, steps=25) for _ in range(2))
    graph = graphed.capture(sampler, **params)
    for u in uniforms:
        for loop in (eager, graphed):
            loop.uniforms.copy_(u)
        eager.step(sampler, **params)
        graph.replay()
        assert torch.equal(eager.tokens, graphed.tokens)
    assert len(set(eager.tokens.tolist())) > 1
