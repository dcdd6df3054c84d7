"""The operators of a drafting decode step together, as examples/drafted_loop.py
runs them: the logits against the model in 64 bits over what the 4-bit cache
stands for, the tokens against the logits, the CUDA graph against eager steps."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import read_kv4  # noqa: E402

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("drafted_loop", os.path.join(ROOT, "examples", "drafted_loop.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def exact_linear(layer, x):
    """An Int8Linear of 64-bit x, which the layer sees rounded to bf16."""
    x = x.bfloat16().double()
    scale = (x.abs().amax(1, keepdim=True) / 127.0).float().double()
    q = (x / scale).float().double().round().clamp(-127, 127)
    return (q @ layer.weight.double().T) * scale * layer.scale.double()


def rotated(model, x, place):
    """x [T, heads, dim] in 64 bits, turned by the table's rows."""
    half = model.dim // 2
    c, s = model.rope[place].double()[:, None, 0], model.rope[place].double()[:, None, 1]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def exact_logits(loop, b, first, tokens):
    """Logits after each of ``tokens``, fed at positions first.., over row b's cache."""
    m = loop.model
    place = torch.arange(first + len(tokens), device="cuda")
    k, v, status = read_kv4(loop.cache, loop.slots(place[None], loop.rows[b:b + 1])[0])
    assert not status.any()
    k, v = (t.double().repeat_interleave(m.heads // m.kv_heads, 1) for t in (k, v))
    hidden = m.embedding[tokens].double()
    qkv = exact_linear(m.qkv, hidden).bfloat16().double().view(len(tokens), -1, m.dim)
    q = rotated(m, qkv[:, :m.heads], place[first:]).bfloat16().double()
    score = torch.einsum("thd,khd->htk", q, k) * m.dim ** -0.5
    score.masked_fill_(place[None, None, :] > place[None, first:, None], -float("inf"))
    mixed = torch.einsum("htk,khd->thd", torch.softmax(score, -1), v).bfloat16().flatten(1)
    last = (hidden + exact_linear(m.out, mixed).bfloat16().double()).bfloat16()
    return exact_linear(m.head, last)


def start(ex, rows=5, steps=8, drafts=3, seed=7, heads=6, kv_heads=2, dim=64):
    model = ex.ToyModel(vocab=1003, hidden=256, heads=heads, kv_heads=kv_heads, dim=dim, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, 40, (1 + 23 * b,), generator=gen).tolist() for b in range(rows)]  # tokens that recur
    torch.manual_seed(seed)
    return ex.DraftedLoop(model, prompts, steps, drafts)


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (16, 2, 32), (4, 4, 80)])
def test_logits_match_the_model_in_64_bits(heads, kv_heads, dim):
    """Rounding to bf16 and to 8 bits is made at the same places; where a value
    lies next to a boundary the projections' integers differ by one step, and
    keys and values that were read back are rounded to bf16 (2^-9 of an entry,
    less than such a step).  In norm the logits are within 4 roundings of the
    8-bit steps: 4 / 127 / sqrt(12)."""
    loop = start(example(), heads=heads, kv_heads=kv_heads, dim=dim)
    gen = torch.Generator().manual_seed(3)
    for step in range(4):
        drafts = torch.randint(0, 40, (5, 3), generator=gen).cuda()
        drafts[1, 1:] = -1
        drafts[3] = -1
        first, newest = loop.lengths.tolist(), loop.newest.tolist()
        logits = loop.logits(drafts)
        for b in range(5):
            fed = [newest[b]] + [t for t in drafts[b].tolist() if t >= 0]
            want = exact_logits(loop, b, first[b], torch.tensor(fed, device="cuda"))
            err = (logits[b, :len(fed)].double() - want).norm() / want.norm()
            assert float(err) <= 4 / 127 / 12 ** 0.5, (step, b, float(err))
        loop.lengths += torch.tensor([4, 1, 2, 1, 3], device="cuda")  # some drafts are dropped: their slots are written again
        loop.newest.copy_(torch.randint(0, 40, (5,), generator=gen))


@gpu
def test_greedy_tokens_are_the_logits_largest():
    """At temperature 0 a step keeps drafts as long as each is the largest logit
    and adds the largest one more; the text then holds what was kept."""
    loop = start(example(), steps=20)
    for _ in range(20):
        drafts = loop.propose()
        state = [t.clone() for t in (loop.lengths, loop.newest)]
        best = loop.logits(drafts).argmax(-1)
        tokens, counts = loop.step()
        for b in range(5):
            n = 0
            while n < 3 and int(drafts[b, n]) == int(best[b, n]):
                n += 1
            assert tokens[b].tolist() == best[b, :n + 1].tolist() + [-1] * (3 - n) and int(counts[b]) == n + 1
        assert torch.equal(loop.lengths, state[0] + counts) and torch.equal(loop.newest, tokens[loop.rows, counts.long() - 1])


@gpu
def test_drafts_that_the_model_agrees_with_are_kept():
    """Drafts made of the model's own largest logits, one of them replaced by
    another token: what is before it is kept.  The logits of one, two, ... and
    all tokens at once are the same bits here as far as their order goes: the
    model's projections take each token alone, and a token's attention is over
    the same keys; where the two largest logits are closer than attention's
    error of 2^-8 of them, the row is left out."""
    loop = start(example(), steps=12)
    checked = 0
    for step in range(12):
        drafts = torch.full((5, 3), -1, device="cuda")
        clear = torch.ones(5, dtype=torch.bool, device="cuda")
        for i in range(4):
            top = loop.logits(drafts)[:, i].topk(2, dim=-1)
            clear &= top.values[:, 0] - top.values[:, 1] > 2.0 ** -8 * top.values.abs().amax(-1)
            if i < 3:
                drafts[:, i] = top.indices[:, 0]
        last = top.indices[:, 0]
        where = [(step + b) % 4 for b in range(5)]  # 3: none is replaced
        fed = drafts.clone()
        for b, i in enumerate(where):
            if i < 3:
                fed[b, i] = (int(drafts[b, i]) + 1 + b) % 1003
        loop.propose = lambda: fed
        tokens, counts = loop.step()
        for b, i in enumerate(where):
            if not clear[b]:
                continue
            checked += 1
            want = drafts[b, :i + 1].tolist() if i < 3 else drafts[b].tolist() + [int(last[b])]
            assert tokens[b, :i + 1].tolist() == want and int(counts[b]) == i + 1, (step, b)
    assert checked >= 30


@gpu
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_graph_equals_eager_steps(temperature):
    ex = example()
    eager, captured = start(ex, steps=12), start(ex, steps=12)
    assert torch.equal(eager.pages, captured.pages)
    heat = torch.full((5,), temperature, dtype=torch.float64, device="cuda")
    graph, (tokens, counts) = captured.capture(heat)
    uniforms = torch.rand((12, 5, 4), generator=torch.Generator().manual_seed(2), dtype=torch.float64).cuda()
    for u in uniforms:
        eager.uniforms.copy_(u)
        captured.uniforms.copy_(u)
        want = eager.step(heat)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(counts, want[1])
        assert torch.equal(captured.lengths, eager.lengths) and torch.equal(captured.follows, eager.follows)


@gpu
def test_example_runs(capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["drafted_loop.py", "--rows", "3", "--steps", "4", "--prompt", "40", "--drafts", "2"])
    example().main()
    out = capsys.readouterr().out
    assert "3 rows, 4 steps" in out and out.count("row ") >= 3
