"""verify_drafts against its definition, step by step in 64 bits.

Tokens and counts are equal unless an acceptance's u q(d) lies within 2^-17 of
p(d) (no seed here does); draws compare in 64 bits.  Probabilities: the sum of
an accepted position's weights is in fp32, each weight's exponent t (units of
log2) off by |t| 2^-23 (the factor's rounding and the product's), the
exponential by 2^-22, sums of 32 weights by 32 * 2^-24, one over the other the
same in p; then p is rounded to fp32: p (sum p |t| 2^-23 + 2^-22 + 2^-19 +
2^-24).  The drawn token's is in 64 bits, rounded once: 2^-24.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import _lib, verify_drafts  # noqa: E402

gpu = pytest.mark.gpu


def expect(logits, drafts, uniforms, draft_probs, heat):
    """One row: (tokens, probs, relative bounds, flags or None, smallest margin)."""
    n = logits.shape[0] - 1
    tokens, probs, bounds, flags, margin = [], [], [], 0, math.inf

    def target(i):
        nonlocal flags
        x = logits[i].double()
        if bool(x.isnan().any()) or bool((x == math.inf).any()):
            flags |= _lib.MS_ROW_NONFINITE
        x = torch.where(x.isnan(), -math.inf, x)
        top = x.max()
        if heat == 0:
            p = torch.zeros_like(x)
            p[int((x == top).nonzero()[0])] = 1.0
            return p, 0.0
        if top == -math.inf:
            return None, 0.0
        t = torch.where(x == top, 0.0, (x - top) / heat)
        w = t.exp()
        p = w / w.sum()
        spread = float((p * torch.where(p > 0, t, 0.0).abs()).sum()) * 1.4427
        return p, spread * 2.0 ** -23 + 2.0 ** -22 + 2.0 ** -19 + 2.0 ** -24

    i = 0
    while True:
        p, slip = target(i)
        if p is None:
            return [-1] * (n + 1), [0.0] * (n + 1), [0.0] * (n + 1), _lib.MS_ROW_ALL_MASKED | flags, margin
        weight = p
        d = int(drafts[i]) if i < n else -1
        if d >= 0:
            q = draft_probs[i].double() if draft_probs is not None and heat != 0 else None
            need = float(uniforms[i]) * (float(q[d]) if q is not None else 1.0)
            if heat != 0:
                margin = min(margin, abs(need - float(p[d])) / max(float(p[d]), 1e-300))
            if need < float(p[d]):
                tokens.append(d), probs.append(float(p[d])), bounds.append(slip)
                i += 1
                continue
            if heat != 0:
                if q is not None:
                    if not bool(((q >= 0) & (q < math.inf)).all()):
                        flags |= _lib.MS_ROW_NONFINITE
                    rest = (p - torch.where(q.isnan(), 0.0, q.clamp(min=0))).clamp(min=0)
                else:
                    rest = p.clone()
                    rest[d] = 0
                weight = rest if float(rest.sum()) > 0 else p
        mass = weight.cumsum(0)
        past = (mass > float(uniforms[n]) * float(mass[-1])).nonzero()
        token = int(past[0]) if len(past) else int((weight > 0).nonzero()[-1])
        tokens.append(token), probs.append(float(p[token])), bounds.append(2.0 ** -23)
        rest = n + 1 - len(tokens)
        return tokens + [-1] * rest, probs + [0.0] * rest, bounds + [0.0] * rest, flags, margin


def check(logits, drafts, uniforms, draft_probs=None, temperature=1.0):
    """Run and compare every row; returns (tokens, counts, status)."""
    tokens, probs, counts, status = verify_drafts(logits, drafts, uniforms, draft_probs=draft_probs, temperature=temperature)
    B, n = logits.shape[0], logits.shape[1] - 1
    assert tokens.dtype == torch.int64 and tokens.shape == (B, n + 1) and probs.shape == (B, n + 1)
    heat = temperature.tolist() if isinstance(temperature, torch.Tensor) else [temperature] * B
    for b in range(B):
        want, p, slack, flags, margin = expect(logits[b], drafts[b], uniforms[b],
                                               draft_probs[b] if draft_probs is not None else None, heat[b])
        assert margin > 2.0 ** -17, (b, margin)
        assert tokens[b].tolist() == want, b
        assert int(counts[b]) == sum(t >= 0 for t in want)
        assert int(status[b]) == flags, b
        for got, exact, room in zip(probs[b].tolist(), p, slack):
            assert abs(got - exact) <= exact * room + 1e-45, (b, got, exact)
    return tokens, counts, status


def problem(B, n, V, dtype=torch.float32, seed=1, sharp=2.5, probs=True, near=0.7, fewer=True, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    store = torch.randn((B, n + 1, V + pad), generator=gen, device="cuda") * sharp
    logits = store.to(dtype)[..., pad // 2:pad // 2 + V]
    q = torch.softmax(logits[:, :n].float() + near * torch.randn((B, n, V), generator=gen, device="cuda"), -1)
    drafts = (q / torch.empty_like(q).exponential_(generator=gen)).argmax(-1) if n else q.new_zeros((B, 0)).long()
    if fewer and n:
        count = torch.randint(0, n + 1, (B, 1), generator=gen, device="cuda")
        count[0] = n
        drafts = torch.where(torch.arange(n, device="cuda") < count, drafts, -1 - drafts)
    uniforms = torch.rand((B, n + 1), generator=gen, device="cuda", dtype=torch.float64)
    return logits, drafts, uniforms, q if probs else None


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("B,n,V,sharp,pad", [
    (1, 0, 1, 2.5, 0), (3, 1, 2, 2.5, 0), (7, 3, 5, 1.0, 0), (20, 4, 33, 2.5, 3), (9, 8, 1000, 3.0, 0), (5, 2, 2049, 4.0, 2),
    (4, 4, 32003, 4.0, 0), (2, 3, 151936, 2.5, 0), (2, 1, 262147, 4.0, 1), (40, 33, 130, 1.0, 0)])
def test_against_definition(B, n, V, sharp, pad, probs, dtype):
    logits, drafts, uniforms, q = problem(B, n, V, dtype, seed=B + n + V, sharp=sharp, probs=probs, pad=pad)
    heat = 0.5 + torch.rand(B, generator=torch.Generator().manual_seed(V), dtype=torch.float64).cuda()
    heat[1::3] = 0.0
    check(logits, drafts, uniforms, q, heat)


@gpu
@pytest.mark.parametrize("probs", [True, False])
def test_refusals_and_acceptances_all_occur(probs):
    """Small vocabularies: every number of accepted drafts, over many rows."""
    logits, drafts, uniforms, q = problem(300, 4, 6, seed=11, sharp=2.0, probs=probs, fewer=False)
    _, counts, _ = check(logits, drafts, uniforms, q)
    assert sorted(set(counts.tolist())) == [1, 2, 3, 4, 5]


@gpu
@pytest.mark.parametrize("probs", [True, False])
def test_tokens_are_distributed_as_the_target(probs):
    """200000 rows of the same two positions: the first token's frequencies are p's, and the second's the next
    position's where one draft was accepted.  Five standard deviations of a binomial each."""
    B, V = 200000, 5
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.tensor([[0.0, 1.0, -1.0, 0.5, -math.inf], [1.0, 0.0, 0.3, -2.0, 0.1]], device="cuda")
    logits = base.expand(B, 2, V)
    q = torch.tensor([0.4, 0.1, 0.2, 0.25, 0.05], device="cuda")
    drafts = torch.multinomial(q, B, replacement=True, generator=gen).view(B, 1)
    if not probs:  # a lookup: always token 3
        drafts.fill_(3)
    uniforms = torch.rand((B, 2), generator=gen, device="cuda", dtype=torch.float64)
    tokens, _, counts, status = verify_drafts(logits, drafts, uniforms, draft_probs=q.expand(B, 1, V) if probs else None,
                                              temperature=0.7)
    assert not status.any()
    for pos, rows in ((0, torch.ones(B, dtype=torch.bool, device="cuda")), (1, counts == 2)):
        p = torch.softmax(base[pos].double() / 0.7, 0)
        m = int(rows.sum())
        seen = torch.bincount(tokens[rows, pos], minlength=V).double()
        assert bool(((seen - m * p).abs() <= 5 * (m * p * (1 - p)).sqrt() + 1e-9).all()), (pos, seen / m, p)


@gpu
def test_ends_of_the_draw():
    """u = 0 draws the first token with any mass, the largest u below 1 the last one."""
    V = 5000
    logits = torch.zeros((4, 2, V), device="cuda")
    logits[:, :, :100] = -math.inf
    logits[:, :, -77:] = -math.inf
    drafts = torch.tensor([[-1], [150], [-5], [150]], device="cuda")
    high = 1.0 - 2.0 ** -53
    uniforms = torch.tensor([[0.5, 0.0], [0.9, 0.0], [0.5, high], [0.9, high]], device="cuda", dtype=torch.float64)
    tokens, counts, _ = check(logits, drafts, uniforms)
    assert tokens[:, 0].tolist() == [100, 100, V - 78, V - 78]
    # the refused draft is the first, or the last, token with mass
    drafts = torch.tensor([[100], [V - 78]], device="cuda")
    tokens, _, _ = check(logits[:2], drafts, uniforms[[1, 3]])
    assert tokens[:, 0].tolist() == [101, V - 79]
    # nothing is left of p: the draw is from p as it is
    q = torch.ones((4, 1, V), device="cuda")
    refused = torch.tensor([[0.9, 0.0], [0.9, high], [0.9, 0.25], [0.9, 0.75]], device="cuda", dtype=torch.float64)
    check(logits, torch.full((4, 1), 200, device="cuda"), refused, q)
    one = torch.full((1, 2, 3), -math.inf, device="cuda")
    one[..., 1] = 4.0  # all mass on the refused draft's neighbour, then on the draft itself
    check(one, torch.tensor([[0]], device="cuda"), refused[:1])
    q = torch.tensor([[[0.0, 2.0, 0.0]]], device="cuda")
    check(one, torch.tensor([[1]], device="cuda"), refused[:1], q)


@gpu
def test_greedy():
    logits, drafts, uniforms, q = problem(6, 3, 20011, torch.bfloat16, seed=5, fewer=False)
    best = logits.float().argmax(-1)
    logits[2, 1, 77] = logits[2, 1, 19000] = 100.0  # a tie: the first
    logits[3, 2] = -math.inf                         # nothing allowed: token 0, as Sampler has it
    drafts[:, :] = best[:, :3]
    drafts[0, 1] = (drafts[0, 1] + 1) % 20011
    drafts[2, 1] = 19000
    tokens, counts, status = check(logits, drafts, uniforms, q, 0.0)
    assert counts.tolist() == [2, 4, 2, 3, 4, 4] and int(tokens[2, 1]) == 77 and int(tokens[3, 2]) == 0
    assert tokens[1].tolist() == best[1].tolist()


@gpu
@pytest.mark.parametrize("heat", [1e-300, 5e-324, 1e-30, 1e-3, 50.0, 1e30, 1e300])
def test_temperatures_of_any_size(heat):
    logits, drafts, uniforms, q = problem(4, 2, 3001, seed=6, sharp=3.0)
    logits[:, :, ::7] = -math.inf
    check(logits, drafts, uniforms, None, heat)
    check(logits, drafts, uniforms, q, heat)


@gpu
def test_bad_rows():
    logits, drafts, uniforms, q = problem(8, 2, 500, seed=7, fewer=False)
    heat = torch.ones(8, dtype=torch.float64, device="cuda")
    heat[0], heat[1], heat[2] = -1.0, math.nan, math.inf
    drafts[3, 1] = 500
    drafts[4, 0], drafts[4, 1] = -1, 10 ** 12  # behind the end: not looked at
    logits[5, 0] = -math.inf
    heat[6], drafts[6, 0] = math.nan, 2 ** 40
    tokens, probs, counts, status = verify_drafts(logits, drafts, uniforms, draft_probs=q, temperature=heat)
    T, D, M = _lib.MS_ROW_BAD_TEMPERATURE, _lib.MS_ROW_BAD_DRAFT, _lib.MS_ROW_ALL_MASKED
    assert status.tolist() == [T, T, T, D, 0, M, T | D, 0]
    for b in (0, 1, 2, 3, 5, 6):
        assert tokens[b].tolist() == [-1, -1, -1] and int(counts[b]) == 0 and not probs[b].any()
    good = [4, 7]
    check(logits[good], drafts[good], uniforms[good], q[good])
    # a masked position behind the refusal is not met
    logits[7, 1:] = -math.inf
    drafts[7, 0] = int(logits[7, 0].argmin())
    uniforms[7, 0] = 0.999
    q[7, 0] = 1.0 / 500
    check(logits[7:], drafts[7:], uniforms[7:], q[7:])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_and_infinite_entries(dtype):
    logits, drafts, uniforms, q = problem(8, 2, 4099, dtype, seed=8, fewer=False)
    logits[0, 0, 4098] = math.nan
    logits[1, 0, 17] = math.inf
    logits[2, 0, 5], logits[2, 0, 4000] = math.inf, math.inf
    drafts[2, 0] = 4000
    logits[3, 2, 9] = math.nan       # met only where both drafts are accepted
    uniforms[3, 0] = 0.9999999
    drafts[3, 0] = int(logits[3, 0].float().argmin())
    logits[4, 0, :] = math.nan
    drafts[4, 0] = -1
    q[5, 0, 11], q[5, 0, 12], q[5, 0, 13] = math.nan, math.inf, -0.5
    drafts[5, 0] = int(logits[5, 0].float().argmin())
    uniforms[5, 0] = 0.9999999
    q[6, 0, int(drafts[6, 0])] = math.nan  # the draft's own: refused
    check(logits, drafts, uniforms, q)
    check(logits, drafts, uniforms, q, 0.0)
    rows = [0, 1, 2, 3, 4, 7]
    check(logits[rows], drafts[rows], uniforms[rows], None, 0.8)


@gpu
def test_strides_and_repeats():
    logits, drafts, uniforms, q = problem(5, 3, 1234, seed=9)
    want = verify_drafts(logits, drafts, uniforms, draft_probs=q)
    swapped = logits.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((5, 5), dtype=torch.int64, device="cuda")
    wide[:, :3] = drafts
    u = torch.zeros((5, 9), dtype=torch.float64, device="cuda")
    u[:, 2:6] = uniforms
    p = torch.empty((3, 5, 1237), device="cuda").transpose(0, 1)[..., 1:1235]
    p.copy_(q)
    for got in (verify_drafts(swapped, wide[:, :3], u[:, 2:6], draft_probs=p), verify_drafts(logits, drafts, uniforms, draft_probs=q),
                verify_drafts(logits, drafts, uniforms, draft_probs=q, temperature=[1.0] * 5)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = verify_drafts(logits[:0], drafts[:0], uniforms[:0])
    assert [t.shape[0] for t in empty] == [0, 0, 0, 0]


@gpu
def test_graph_and_stream():
    a, b = problem(6, 4, 40000, seed=12), problem(1, 2, 151936, torch.bfloat16, seed=13, probs=False)
    heat = torch.full((6,), 0.8, dtype=torch.float64, device="cuda")
    one = torch.ones(1, dtype=torch.float64, device="cuda")
    want = verify_drafts(*a[:3], draft_probs=a[3], temperature=heat), verify_drafts(*b[:3], temperature=one)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = verify_drafts(*a[:3], draft_probs=a[3], temperature=heat)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(other, want[0]))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        first = verify_drafts(*a[:3], draft_probs=a[3], temperature=heat)
    with torch.cuda.graph(graphs[1]):
        second = verify_drafts(*b[:3], temperature=one)
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = verify_drafts(*a[:3], draft_probs=a[3], temperature=heat)
        torch.cuda.synchronize()
        for got, exact in ((first, want[0]), (second, want[1]), (eager, want[0])):
            assert all(torch.equal(x, y) for x, y in zip(got, exact))
    a[2].uniform_(generator=torch.Generator(device="cuda").manual_seed(1))
    graphs[0].replay()
    torch.cuda.synchronize()
    now = verify_drafts(*a[:3], draft_probs=a[3], temperature=heat)
    assert all(torch.equal(x, y) for x, y in zip(first, now))


@gpu
def test_logits_past_32_bits():
    """Rows whose logits lie more than 2^32 entries into their tensor."""
    V, n = 151936, 1
    B = 2 ** 32 // (2 * V) + 2
    logits = torch.zeros((B, 2, V), dtype=torch.bfloat16, device="cuda")
    logits[-1, 0, 7], logits[-1, 1, 151000] = 20.0, 20.0
    logits[0, 0, 5] = 20.0
    drafts = torch.full((B, 1), -1, device="cuda")
    drafts[-1] = 7
    tokens, _, counts, status = verify_drafts(logits, drafts, torch.full((B, 2), 0.5, dtype=torch.float64, device="cuda"))
    assert not status.any()
    # equal weights: the running mass, j + 1 of 151936 at token j, passes the half, 75968, at token 75968
    assert tokens[-1].tolist() == [7, 151000] and tokens[0].tolist() == [5, -1] and tokens[1].tolist() == [75968, -1]


@gpu
def test_call_refusals():
    logits, drafts, uniforms, q = problem(3, 2, 50)
    for args, kw in (((logits.double(), drafts, uniforms), {}), ((logits, drafts.int(), uniforms), {}),
                     ((logits, drafts, uniforms.float()), {}), ((logits, drafts, uniforms), dict(draft_probs=q.double())),
                     ((logits.cpu(), drafts, uniforms), {}), ((logits, None, uniforms), {})):
        with pytest.raises(TypeError):
            verify_drafts(*args, **kw)
    for args, kw in (((logits[0], drafts, uniforms), {}), ((logits, drafts[:, :1], uniforms), {}),
                     ((logits, drafts, uniforms[:, :2]), {}), ((logits, drafts[:2], uniforms), {}),
                     ((logits, drafts, uniforms), dict(draft_probs=q[:, :1])), ((logits, drafts, uniforms), dict(draft_probs=q[..., :49])),
                     ((logits, drafts, uniforms), dict(temperature=[1.0, 2.0])), ((logits[..., ::2], drafts, uniforms), {}),
                     ((logits[:, :0], drafts, uniforms), {}), ((logits[..., :0], drafts, uniforms), {}),
                     ((logits, drafts.cpu(), uniforms), {}),
                     ((torch.zeros((1, 257, 2), device="cuda"), torch.zeros((1, 256), dtype=torch.int64, device="cuda"),
                       torch.zeros((1, 257), dtype=torch.float64, device="cuda")), {})):
        with pytest.raises(ValueError):
            verify_drafts(*args, **kw)


def test_cpu_tensors_are_refused():
    with pytest.raises(TypeError, match="CUDA"):
        verify_drafts(torch.zeros((1, 2, 5)), torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 2), dtype=torch.float64))


def test_entry_point_refusals():
    """The C entry point refuses on the host, before any launch."""
    import ctypes
    L = _lib.lib()
    some = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(some) + 255) // 256 * 256

    def call(**other):
        return L.ms_verify_drafts(_lib.VerifyArgs(**{**dict(
            dtype=0, drafts=1, rows=1, vocab=10, logits=p, draft_tokens=p, uniforms=p, temperature=p, tokens=p, probs=p,
            counts=p, status=p, workspace=p, workspace_bytes=16), **other}), None)

    assert call(rows=0) == 0
    assert call(dtype=3) == -2
    for bad in (dict(rows=-1), dict(drafts=-1), dict(drafts=256), dict(vocab=0), dict(vocab=1 << 31), dict(logits=None),
                dict(draft_tokens=None), dict(uniforms=None), dict(temperature=None), dict(tokens=None), dict(probs=None),
                dict(counts=None), dict(status=None), dict(workspace=None), dict(workspace=p + 8), dict(),
                dict(rows=1 << 29)):
        assert call(**bad) == -1, bad
    assert L.ms_verify_drafts(None, None) == -1
    assert L.ms_verify_workspace(0, 1, 10) == 0 and L.ms_verify_workspace(1, 256, 10) == 0


@gpu
@pytest.mark.parametrize("top", [20.0, 50.0, 100.0])
@pytest.mark.parametrize("heat", [1e-10, 1e-9, 2e-9, 1e-8, 5e-8, 1e-6])
def test_near_ties_at_small_temperatures(heat, top):
    """The second largest logit a few units in the last place below the largest,
    hundreds or thousands of octaves apart in weight: neighbours, and at the
    row's two ends."""
    V, cases = 3001, [(ulps, at) for ulps in (1, 2, 5, 20) for at in ((1500, 1501), (7, 2990), (2990, 7))]
    logits, _, uniforms, q = problem(len(cases), 2, V, seed=14, sharp=0.5, fewer=False)
    step = float(torch.tensor(top) - torch.nextafter(torch.tensor(top), torch.tensor(0.0)))
    first, second = (torch.tensor([at[i] for _, at in cases], device="cuda") for i in range(2))
    rows = torch.arange(len(cases), device="cuda")
    logits[rows, :, first] = top
    logits[rows, :, second] = top - step * torch.tensor([float(u) for u, _ in cases], device="cuda")[:, None]
    none = torch.full_like(first, -1)
    for drafts in ((none, none), (first, second), (second, first), (first, first)):
        drafts = torch.stack(drafts, 1)
        check(logits, drafts, uniforms, None, heat)
        given = q * 0.3
        for at, much in ((first, 0.3), (second, 0.4)):
            given[rows, :, at] = much
        check(logits, drafts, uniforms, given, heat)


@gpu
@pytest.mark.parametrize("heat", [1.0, 1e26, 1e30, 1e300])
def test_lowest_logits_alone(heat):
    """Rows whose only values are the type's lowest, which a mask may write: they share the probability."""
    V, low = 2500, torch.finfo(torch.float32).min
    logits = torch.full((3, 2, V), low, device="cuda")
    logits[1, :, ::3] = -math.inf
    logits[2, :, 40:] = -math.inf
    drafts = torch.tensor([[-1], [4], [39]], device="cuda")
    uniforms = torch.tensor([[0.5, 0.30013], [0.9, 0.7], [0.9, 0.999]], dtype=torch.float64, device="cuda")
    check(logits, drafts, uniforms, None, heat)
    check(logits, drafts, uniforms, torch.full((3, 1, V), 1e-3, device="cuda"), heat)


@gpu
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("heat", [1e32, 1e36, 1e37, 1e38, 3e38, 1e39, 1e42])
def test_logits_as_large_as_the_temperature(heat, probs):
    """Logits over all of fp32's range, at temperatures where they weigh alike."""
    logits, drafts, uniforms, q = problem(20, 3, 1200, seed=15, probs=probs)
    big = torch.finfo(torch.float32).max
    logits.clamp_(-3, 3)
    logits *= min(big / 3, heat / 2)
    logits[::2, :, ::5] = -big
    logits[1::4, :, 3::7] = big
    check(logits, drafts, uniforms, q, heat)


@gpu
def test_greedy_over_positions_without_a_value():
    """The first largest of a position that holds nothing but -inf is token 0: a draft of it is accepted."""
    logits, drafts, uniforms, q = problem(4, 3, 700, seed=16, fewer=False)
    best = logits.argmax(-1)
    drafts.copy_(best[:, :3])
    logits[:3, 1] = -math.inf
    logits[2, 1] = math.nan
    drafts[0, 1], drafts[1, 1], drafts[2, 1] = 0, 5, 0
    tokens, counts, status = check(logits, drafts, uniforms, q, 0.0)
    assert counts.tolist() == [4, 2, 4, 4] and tokens[0].tolist() == [int(best[0, 0]), 0, int(best[0, 2]), int(best[0, 3])]
    assert status.tolist() == [0, 0, _lib.MS_ROW_NONFINITE, 0]


@gpu
def test_draws_beside_borders_of_long_rows():
    """2^24 tokens, a CTA a row: u lies 2^-37 (twice what a weight may be off by)
    beside a border of what the draft leaves.  One token holds a fifteenth of p,
    the others are 20 octaves below it, so that an error of the weights' unit
    moves their sum; the draft's share of them lies in the second half alone, so
    that an error of it moves the first half's borders."""
    V, B = 1 << 24, 600
    # a temperature whose factor log2(e) / T is rounded by almost half a unit in the last place of fp32
    heat = max((1.0 + i * 1e-4 for i in range(400)),
               key=lambda t: abs(float(torch.tensor(1.4426950408889634 / t)) * t / 1.4426950408889634 - 1.0))
    gen = torch.Generator(device="cuda").manual_seed(17)
    base = torch.rand((2, V), generator=gen, device="cuda") * 0.01
    base[:, V // 2 + 3] = 14.0 * heat
    p = torch.softmax(base[0].double() / heat, 0)
    q = torch.zeros(V, device="cuda")
    q[V // 2:] = 0.47 * float(p[0])
    q[V - 1] = 1e-3
    mass = (p - q.double()).clamp(min=0).cumsum(0)
    at = torch.randint(V // 8, V // 2, (B,), generator=gen, device="cuda")
    above = torch.arange(B, device="cuda") % 2
    uniforms = torch.full((B, 2), 0.9, dtype=torch.float64, device="cuda")
    uniforms[:, 1] = mass[at] / mass[-1] + (above * 2 - 1) * 2.0 ** -37
    tokens, probs, counts, status = verify_drafts(base.expand(B, 2, V), torch.full((B, 1), V - 1, device="cuda"), uniforms,
                                                  draft_probs=q.expand(B, 1, V), temperature=heat)
    assert not status.any() and bool((counts == 1).all())
    assert torch.equal(tokens[:, 0], at + above)
    assert bool(((probs[:, 0].double() - p[tokens[:, 0]]).abs() <= p[tokens[:, 0]] * 2.0 ** -23).all())
