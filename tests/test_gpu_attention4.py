"""attention_kv4 against its definition in 64 bits, over what the cache's codes
and parameters stand for: entry = z + s (c - 8).

Tolerance, with U the half unit of q's type (2^-8 bf16, 2^-11 fp16), u = 2^-11
fp16's, n a token's keys and p the exact weights:

* a score is summed in fp32 from products of magnitudes |q| s (c + 8) and
  |q| |z|, A their sum times the scale: a product instruction adds 17 or 18
  terms, each truncated at worst to 2^-23 of the largest, so that all of a
  score's sums are within e = 2^-18 A;
* weights are then off by a factor within 2 e + 2^-20 (the exponential's
  argument and result) and rounded to fp16, with the value's scale (for c - 8)
  or without (for z): u sum p (s |c - 8| + |z|).  Weights are scaled so that the
  largest is at least 2^6 (2^7 less a half for the power of two that is at most
  twice the largest s), so that fp16's steps of 2^-24 below its normal range
  are within 2^-30 of the largest: 2^-30 sum (16 S + Z), S and Z the largest
  scale and middle;
* sums over the keys hold terms of magnitude p s (c + 8) and p |z|:
  (n + 64) 2^-22 of their sum R, and the weights' factor acts on R as well;
* the output is rounded once.

So |out - exact| <= u sum p (s |c - 8| + |z|) + (4 e + 2^-19 + (n + 64) 2^-22) R
+ 2^-30 n (16 S + Z) + U |exact| + 2^-25, and lse is within 2 e + 2^-20 + (n +
64) 2^-23 + 2^-22 |lse|.
"""
import copy
import math

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import KvCache4, _lib, append_kv4, attention_kv4, read_kv4  # noqa: E402

gpu = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
HALF_ULP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11}


def split(codes, params, dim):
    """(c, s, z) of codes [..., bytes] and params [..., groups, 2], in 64 bits."""
    i = torch.arange(dim, device=codes.device)
    c = ((codes[..., i // 2].int() >> (4 * (i % 2))) & 15).double()
    return c, params[..., i // 32, 0].double(), params[..., i // 32, 1].double()


class Problem:
    """Random codes and parameters; what no token sees holds NaN."""

    def __init__(self, B, T, H, Hkv, D, lens, page, dtype=BF16, seed=1, spread=1.5, scales=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        lens = torch.tensor(lens, dtype=torch.int32).view(B, -1)
        if lens.shape[1] == 1 and T > 1:  # drafted tokens: each sees one key more
            lens = (lens - torch.arange(T - 1, -1, -1)).clamp(min=0).int()
        most = lens.amax(1).tolist()
        used = [-(-n // page) for n in most]
        total = sum(used) + 1
        self.cache = cache = KvCache4.empty(total, page, Hkv, D, dtype=dtype)
        self.used_groups = -(-D // 32)
        for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
            codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device="cuda", dtype=torch.uint8))
            params[..., 0] = torch.rand(params.shape[:-1], generator=gen, device="cuda") * 0.3 + 0.05
            params[..., 1] = torch.randn(params.shape[:-1], generator=gen, device="cuda") * 0.5
        perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32).cpu()
        table = torch.full((B, max(used + [1]) + 1), -5, dtype=torch.int32)  # entries past the row's keys are not read
        keep = torch.zeros((total, page), dtype=torch.bool)
        at = 0
        for b, n in enumerate(most):
            table[b, :used[b]] = perm[at:at + used[b]]
            for i in range(used[b]):
                keep[int(perm[at + i]), :min(page, n - i * page)] = True
            at += used[b]
        hidden = ~keep.cuda()
        for params in (cache.k_params, cache.v_params):
            params.transpose(1, 2)[hidden] = math.nan
            params[:, :, :, self.used_groups:] = math.nan  # not a head's parameters
        self.table = table.cuda()
        self.pages = self.table[:, :-1]
        self.lengths = lens.cuda()
        if scales:
            scales(self)
        self.q = (torch.randn((B, T, H, D), generator=gen, device="cuda") * spread).to(dtype)
        self.lens, self.page = lens.tolist(), page

    def run(self, **kw):
        if self.q.shape[1] == 1:  # the form for one token a row
            out, lse, status = attention_kv4(self.q[:, 0], self.cache, self.pages, self.lengths[:, 0].contiguous(), **kw)
            return out[:, None], lse[:, None], status
        return attention_kv4(self.q, self.cache, self.pages, self.lengths, **kw)

    def keys(self, b, n, codes, params):
        """[Hkv, n, D] each: c, s, z of the row's first n keys."""
        pages = self.pages[b, :-(-n // self.page)].long()
        flat = [t[pages].transpose(1, 2).flatten(0, 1)[:n].transpose(0, 1) for t in (codes, params)]
        return split(*flat, self.q.shape[-1])

    def check(self, out, lse, status, scale=None, tokens=None):
        B, T, H, D = self.q.shape
        Hkv = self.cache.kv_heads
        scale = D ** -0.5 if scale is None else scale
        assert not status.any()
        for b in range(B):
            for t in range(T) if tokens is None else tokens:
                n = self.lens[b][t]
                if n == 0:
                    assert not out[b, t].any() and bool((lse[b, t] == -math.inf).all())
                    continue
                c, s, z = self.keys(b, n, self.cache.k_codes, self.cache.k_params)
                q = self.q[b, t].double().view(Hkv, H // Hkv, D)
                score = q @ (z + s * (c - 8)).transpose(1, 2) * scale      # [Hkv, G, n]
                mag = (q.abs() @ (s * (c + 8) + z.abs()).transpose(1, 2) * scale).amax(-1, keepdim=True)
                want_lse = torch.logsumexp(score, -1, keepdim=True)
                p = (score - want_lse).exp()
                c, s, z = self.keys(b, n, self.cache.v_codes, self.cache.v_params)
                want = p @ (z + s * (c - 8))
                near, room = p @ (s * (c - 8).abs() + z.abs()), p @ (s * (c + 8) + z.abs())
                e = 2.0 ** -18 * mag
                bound = 2.0 ** -11 * near + (4 * e + 2.0 ** -19 + (n + 64) * 2.0 ** -22) * room
                bound = bound + 2.0 ** -30 * n * (16 * s.max() + z.abs().max()) + HALF_ULP[self.q.dtype] * want.abs() + 2.0 ** -25
                err = (out[b, t].double().view(Hkv, H // Hkv, D) - want).abs()
                assert bool((err <= bound).all()), (b, t, float((err - bound).max()))
                tol = 2 * e + 2.0 ** -20 + (n + 64) * 2.0 ** -23 + 2.0 ** -22 * want_lse.abs()
                assert bool(((lse[b, t].double().view(Hkv, -1, 1) - want_lse).abs() <= tol).all()), (b, t)


CASES = [
    # B, T, heads, kv_heads, D, keys of each row (of its last token), page
    (1, 1, 1, 1, 16, [1], 1),
    (1, 1, 14, 2, 64, [300], 16),
    (2, 1, 4, 4, 64, [0, 1], 16),
    (3, 1, 14, 2, 64, [15, 16, 17], 16),
    (5, 1, 7, 1, 80, [1, 0, 33, 0, 128], 8),
    (4, 1, 8, 8, 128, [5, 250, 64, 0], 24),
    (3, 1, 16, 1, 96, [70, 3, 129], 64),     # sixteen query rows
    (2, 1, 40, 1, 128, [90, 200], 16),       # more than an item takes
    (2, 1, 40, 1, 64, [90, 200], 5),
    (2, 1, 24, 1, 32, [65, 31], 16),
    (3, 1, 6, 3, 48, [40, 41, 7], 3),
    (2, 1, 5, 5, 112, [1000, 999], 64),
    (2, 4, 4, 1, 64, [100, 2], 16),          # the first tokens of a row see nothing
    (3, 5, 14, 2, 64, [333, 48, 5], 16),     # 35 query rows of a key head
    (2, 8, 8, 2, 128, [77, 400], 64),
    (2, 3, 3, 3, 80, [60, 61], 24),
    (1, 6, 8, 2, 96, [500], 1),
    (2, 17, 2, 1, 64, [64, 19], 16),
    (300, 2, 2, 1, 64, [(7 * i) % 50 for i in range(300)], 16),
    (1, 1, 8, 2, 128, [20000], 64),          # a long row over all warps
]


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_against_definition(case, dtype):
    p = Problem(*case, dtype=dtype, seed=len(str(case)))
    p.check(*p.run())


@gpu
def test_any_lengths_of_tokens():
    """Each token has a length of its own, in any order."""
    lens = [[5, 100, 0, 37], [0, 0, 0, 0], [64, 64, 1, 16], [17, 16, 15, 200]]
    p = Problem(4, 4, 6, 2, 64, lens, 16)
    p.check(*p.run())
    p = Problem(4, 4, 12, 2, 128, lens, 24, dtype=FP16)
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (80, 6)])
def test_nan_past_a_tokens_keys(dim, page):
    """Keys that some of a row's tokens see and others do not hold NaN: it
    reaches the tokens that see them, in the key's and the groups' places, and
    no others."""
    lens = [[20, 21, 22, 50], [50, 49, 3, 0]]
    p = Problem(2, 4, 6, 2, dim, lens, page)
    cache = p.cache
    place = [(int(p.pages[b, j // page]), j % page) for b, j in ((0, 21), (1, 48))]
    for (pg, off), t, g in zip(place, (cache.v_params, cache.v_params), (0, 1)):
        t[pg, 0, off, g, 1] = math.nan   # values of key head 0, one group
        t[pg, 0, off, g, 0] = math.inf
    out, lse, status = p.run()
    assert not status.any()
    seen = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    seen[0, 2:, :3, 0:32] = True
    seen[1, :2, :3, 32:64] = True
    assert torch.equal(out.isnan(), seen)
    assert not bool(lse.isnan().any())
    for b, t in ((0, 0), (0, 1), (1, 2), (1, 3)):  # tokens that see none of it
        alone = attention_kv4(p.q[b:b + 1, t], cache, p.pages[b:b + 1], p.lengths[b:b + 1, t].contiguous())
        assert bool(((out[b, t].double() - alone[0][0].double()).abs() <= 2.0 ** -7 * alone[0][0].double().abs() + 1e-3).all())
    # keys that are no numbers: all of the heads that see them
    cache.v_params[place[0][0], 0, place[0][1], 0] = 0
    cache.v_params[place[1][0], 0, place[1][1], 1] = 0
    cache.k_params[place[0][0], 1, place[0][1], 0, 1] = math.nan
    out, lse, status = p.run()
    seen = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    seen[0, 2:, 3:] = True
    assert torch.equal(out.isnan(), seen) and torch.equal(lse.isnan(), seen[..., 0])


@gpu
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_value_scales_of_any_size(dim):
    """Scales that grow and shrink along the keys over fp16's range, and groups of no scale."""
    def scales(p):
        for pos in range(p.cache.pages):
            p.cache.v_params[pos, :, :, :p.used_groups, 0] *= 2.0 ** (-14 + (pos * 7) % 26)
            p.cache.v_params[pos, :, :, 0, 0] = 0
    p = Problem(2, 2, 4, 2, dim, [300, 90], 16, scales=scales)
    p.check(*p.run())

    def tiny(p):
        p.cache.v_params[..., :p.used_groups, 0] = 2.0 ** -24 * 5
        p.cache.v_params[..., :p.used_groups, 1] = 0
        p.cache.v_params[..., 1, 0] = 2.0 ** -24 * 900
    # a group whose scales are far below another's keeps the bits that 2^-30 of the largest leaves
    p = Problem(1, 1, 4, 2, dim, [130], 16, scales=tiny, dtype=FP16)
    out, _, status = p.run()
    assert not status.any() and bool((out.abs() <= 2.0 ** -24 * 900 * 9).all())
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("spread,scale", [(0.0, None), (1e-30, None), (60.0, None), (1.5, 1e-3), (1.5, 4.0), (1e4, 30.0)])
def test_scores_of_any_size(spread, scale):
    p = Problem(2, 1, 14, 2, 64, [100, 513], 16, spread=spread, dtype=BF16)
    out, lse, status = p.run(scale=scale)
    if spread == 1e4:  # one key has all the weight: compared by the maximum's value
        assert not status.any() and bool(out.isfinite().all())
        for b in range(2):
            c, s, z = p.keys(b, p.lens[b][0], p.cache.k_codes, p.cache.k_params)
            score = p.q[b, 0].double().view(2, 7, 64) @ (z + s * (c - 8)).transpose(1, 2) * scale
            top = score.amax(-1)
            assert bool(((lse[b, 0].double().view(2, 7) - top).abs() <= 2.0 ** -18 * score.abs().amax(-1) + 5).all())
    else:
        p.check(out, lse, status, scale=scale)


@gpu
def test_queries_far_apart_in_size():
    """Rows of one item have magnitudes of their own."""
    p = Problem(2, 2, 8, 2, 64, [100, 40], 16, dtype=BF16)
    p.q *= torch.tensor([1.0, 1e-6, 20.0, 1e-20, 0.0, 3.0, 1e-3, 10.0], device="cuda").bfloat16()[:, None]
    p.check(*p.run())


@gpu
def test_bad_rows_are_flagged_alone():
    p = Problem(5, 2, 4, 2, 64, [40, 40, 40, 40, 40], 16)
    want = p.run()
    p.lengths[1, 0] = -1
    p.lengths[2, 1] = p.pages.shape[1] * 16 + 1
    p.pages[3, 1] = p.cache.pages
    p.pages[4, 2] = -1
    out, lse, status = p.run()
    L, G = _lib.MS_ROW_BAD_LENGTH, _lib.MS_ROW_BAD_PAGE
    assert status.tolist() == [0, L, L, G, G]
    assert torch.equal(out[0], want[0][0]) and torch.equal(lse[0], want[1][0])
    assert not bool(out[1:].any()) and bool((lse[1:] == -math.inf).all())


@gpu
@pytest.mark.parametrize("dim", [64, 80])
def test_strides(dim):
    p = Problem(3, 3, 6, 2, dim, [100, 5, 64], 16)
    want = p.run()
    B, T, H, D = p.q.shape
    odd = torch.empty((B, T, H, D + 1), dtype=BF16, device="cuda")[..., 1:]
    heads_first = torch.empty((H, B, T, D), dtype=BF16, device="cuda").permute(1, 2, 0, 3)
    wide = torch.empty((B, T, H + 2, D), dtype=BF16, device="cuda")[:, :, 1:-1]
    for q in (odd, heads_first, wide):
        q.copy_(p.q)
        for like in (odd, heads_first, wide):
            target = torch.full_like(like, 7.0).as_strided(like.shape, like.stride()) if like is heads_first else torch.empty_like(like)
            out, lse, status = attention_kv4(q, p.cache, p.pages, p.lengths, out=target)
            assert out is target and torch.equal(out, want[0]) and torch.equal(lse, want[1])
    lengths = torch.empty((B, T + 2), dtype=torch.int32, device="cuda")[:, :T]
    lengths.copy_(p.lengths)
    assert torch.equal(attention_kv4(p.q, p.cache, p.pages, lengths)[0], want[0])
    # all rows the same lengths: one row repeated
    same = p.lengths[:1].expand(B, T)
    again = attention_kv4(p.q, p.cache, p.pages[:1].expand(B, -1), same)
    copied = attention_kv4(p.q, p.cache, p.pages[:1].expand(B, -1).contiguous(), same.contiguous())
    assert torch.equal(again[0], copied[0])


@gpu
def test_repeats_are_equal_and_graphs_replay():
    """Equal calls give equal bits; two captured calls of other sizes replay in turn beside eager ones."""
    p = Problem(9, 2, 14, 2, 64, [(91 * i) % 700 for i in range(9)], 16)
    r = Problem(2, 1, 8, 2, 128, [3000, 10], 64, seed=3)
    want, wanted = p.run(), r.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = p.run()
    torch.cuda.synchronize()
    assert torch.equal(again[0], want[0])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        first = p.run()
    with torch.cuda.graph(graphs[1]):
        second = r.run()
    for _ in range(3):
        for g in graphs:
            g.replay()
        eager = p.run()
        torch.cuda.synchronize()
        for got, exact in ((first, want), (second, wanted), (eager, want)):
            assert all(torch.equal(x, y) for x, y in zip(got, exact))
    # replays read the tensors' new contents
    p.lengths.clamp_(max=50)
    graphs[0].replay()
    torch.cuda.synchronize()
    p.lens = p.lengths.tolist()
    p.check(*first)


@gpu
@pytest.mark.parametrize("T,H,Hkv,D", [(1, 1, 1, 16), (1, 8, 2, 64), (1, 8, 1, 128), (5, 14, 2, 64), (3, 12, 1, 48), (4, 64, 1, 96)])
def test_fp16_is_rounded_once(T, H, Hkv, D):
    """Of one key the weight is 1, whatever its score: only the answer's rounding
    (2^-11) and what two halves of a weight leave (2^-22 each of two parts,
    and fp16's steps below its normal range) are left of the error."""
    p = Problem(2, T, H, Hkv, D, [[1] * T, [1] * T], 16, dtype=FP16, seed=T + H + D)
    out, lse, status = p.run()
    assert not status.any()
    for b in range(2):
        c, s, z = p.keys(b, 1, p.cache.v_codes, p.cache.v_params)
        want = (z + s * (c - 8)).expand(Hkv, H // Hkv, D)
        room = (s * (c - 8).abs() + z.abs()).expand(Hkv, H // Hkv, D)
        for t in range(T):
            err = (out[b, t].double().view(Hkv, H // Hkv, D) - want).abs()
            assert bool((err <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * room + 2.0 ** -25).all()), (b, t)


@gpu
@pytest.mark.parametrize("T,H,D", [(1, 4, 64), (1, 8, 64), (2, 8, 64), (3, 8, 128)])
def test_long_items_keep_their_precision(T, H, D):
    """Items of thousands of keys a warp, whose answers are sums of terms of both
    signs far smaller than the sum of their magnitudes: over an answer the
    error's mean square is at most that of its own rounding, a third of the
    square of 2^-11 of the entries, and a tenth of the root for what else there
    is (weights to 2^-20 or so, in terms whose signs differ)."""
    B, n = (320, 32768) if D == 64 else (200, 16384)
    p = Problem(1, T, H, 1, D, [[n - t for t in range(T)]], 16, dtype=FP16, seed=T + H)
    p.q = p.q.expand(B, T, H, D).contiguous()
    p.q *= torch.rand((B, 1, 1, 1), generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").half()
    p.pages, p.lengths = p.pages.expand(B, -1).contiguous(), p.lengths.expand(B, -1).contiguous()
    out, lse, status = p.run()
    assert not status.any()
    for b in (0, B // 3, B - 1):
        for t in range(T):
            c, s, z = p.keys(b, n - t, p.cache.k_codes, p.cache.k_params)
            w = torch.softmax(p.q[b, t].double() @ (z + s * (c - 8))[0].T * D ** -0.5, -1)
            c, s, z = p.keys(b, n - t, p.cache.v_codes, p.cache.v_params)
            want = w @ (z + s * (c - 8))[0]
            err = (out[b, t].double() - want).norm() / want.norm()
            assert float(err) <= 1.1 * 2.0 ** -11 / 3 ** 0.5, (b, t, float(err))


@gpu
@pytest.mark.parametrize("H,Hkv,T", [(6, 2, 4), (2, 1, 2), (28, 2, 3)])
def test_nan_and_infinite_parameters_fp16(H, Hkv, T):
    """As for bf16: a value's group that is no number reaches the tokens that see it, and its group alone."""
    p = Problem(1, T, H, Hkv, 64, [[20] * (T - 1) + [40]], 16, dtype=FP16)
    clean = p.run()
    pg, off = int(p.pages[0, 1]), 14  # key 30
    p.cache.v_params[pg, 0, off, 0, 1] = math.nan
    p.cache.v_params[pg, 0, off, 1, 0] = math.inf
    out, lse, status = p.run()
    assert not status.any() and torch.equal(lse, clean[1])
    seen = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    seen[0, T - 1, :H // Hkv] = True
    assert torch.equal(out.isnan(), seen)
    assert torch.equal(out[~seen], clean[0][~seen])
    p.cache.v_params[pg, 0, off, 1, 0] = 0.25
    out = p.run()[0]
    assert torch.equal(out.isnan(), seen & (torch.arange(64, device="cuda") < 32))


@gpu
@pytest.mark.parametrize("H,Hkv,T", [(8, 2, 1), (8, 1, 1), (14, 2, 5)])
@pytest.mark.parametrize("spread,scale", [(0.0, None), (1e-5, None), (60.0, None), (1.5, 4.0)])
def test_scores_of_any_size_fp16(H, Hkv, T, spread, scale):
    p = Problem(2, T, H, Hkv, 64, [100, 513], 16, spread=spread, dtype=FP16)
    p.check(*p.run(scale=scale), scale=scale)


def rows_of(p, rows):
    """The problem of some rows alone, for check."""
    part = copy.copy(p)
    part.q, part.pages, part.lens = p.q[rows], p.pages[rows], [p.lens[b] for b in rows]
    return part


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,H,Hkv", [(1, 4, 1), (1, 8, 1), (3, 14, 2)])
def test_queries_that_are_no_numbers(T, H, Hkv, dtype):
    """A query that holds a NaN or an infinity gives NaN, and nothing else does."""
    p = Problem(3, T, H, Hkv, 64, [50, 300, 7], 16, dtype=dtype)
    p.q[1, T - 1, 1, 40] = math.nan
    p.q[2, 0, H - 1, 3] = math.inf
    out, lse, status = p.run()
    bad = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    bad[1, T - 1, 1] = bad[2, 0, H - 1] = True
    assert not status.any() and torch.equal(lse.isnan(), bad) and torch.equal(out.isnan(), bad[..., None].expand_as(out))
    clean = copy.copy(p)
    clean.q = torch.where(bad[..., None], 0.0, p.q)
    want = clean.run()
    clean.check(torch.where(bad[..., None], want[0], out), torch.where(bad, want[1], lse), status)


@gpu
@pytest.mark.parametrize("T,H", [(1, 4), (1, 8), (2, 14)])
def test_scores_past_whole_numbers(T, H):
    """Scores so large that one key has all the weight: the answer is its value."""
    p = Problem(2, T, H, 1 if H < 14 else 2, 64, [100, 513], 16, spread=1e30)
    out, lse, status = p.run()
    assert not status.any()
    for b in range(2):
        for t in range(T):
            c, s, z = p.keys(b, p.lens[b][t], p.cache.k_codes, p.cache.k_params)
            score = p.q[b, t].double().view(s.shape[0], -1, 64) @ (z + s * (c - 8)).transpose(1, 2) / 8
            top, place = score.max(-1)
            assert bool(((lse[b, t].double().view_as(top) - top).abs() <= 2.0 ** -18 * score.abs().amax(-1)).all())
            c, s, z = p.keys(b, p.lens[b][t], p.cache.v_codes, p.cache.v_params)
            want = torch.gather(z + s * (c - 8), 1, place[..., None].expand(-1, -1, 64))
            err = (out[b, t].double().view_as(want) - want).abs()
            assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * (s.max() * 8 + z.abs().max())).all())


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_many_tokens_heads_and_rows(dtype):
    p = Problem(1, 1024, 4, 1, 64, [1500], 16, dtype=dtype)
    out, lse, status = p.run()
    p.check(out, lse, status, tokens=[0, 1, 511, 700, 1023])
    p = Problem(2, 1, 250, 2, 128, [333, 40], 64, dtype=dtype)
    p.check(*p.run())
    p = Problem(20011, 2, 3, 1, 48, [(b * 7) % 6 for b in range(20011)], 4, dtype=dtype)
    out, lse, status = p.run()
    assert not status.any()
    rows = [0, 1, 2, 5, 9999, 20009, 20010]
    rows_of(p, rows).check(out[rows], lse[rows], status[rows])


@gpu
def test_out_may_be_q():
    p = Problem(5, 3, 14, 2, 64, [5, 100, 0, 37, 600], 16)
    want = p.run()
    out, lse, status = p.run(out=p.q)
    assert out is p.q and torch.equal(out, want[0]) and torch.equal(lse, want[1])


@gpu
def test_calls_on_two_streams():
    """Two calls under way at once have workspaces of their own."""
    p = Problem(64, 1, 14, 2, 64, [(91 * i) % 700 for i in range(64)], 16)
    r = Problem(16, 4, 14, 2, 64, [(301 * i) % 3000 for i in range(16)], 16, seed=5)
    want = p.run(), r.run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (problem, stream) in enumerate(zip((p, r), streams)):
            with torch.cuda.stream(stream):
                got[i].append(problem.run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for one in got[i] for x, y in zip(one, want[i]))


@gpu
def test_over_appended_tokens():
    """What append_kv4 wrote, against attention over what read_kv4 gives back."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    B, n, H, Hkv, D, page = 3, 70, 8, 2, 80, 16
    cache = KvCache4.empty(B * 5, page, Hkv, D, dtype=FP16)
    pages = torch.randperm(B * 5, generator=gen, device="cuda").int().view(B, 5)
    k, v = (torch.randn((B * n, Hkv, D), generator=gen, device="cuda").half() for _ in range(2))
    j = torch.arange(n, device="cuda")
    slots = (pages[:, j // page].long() * page + j % page).flatten()
    _, status = append_kv4(cache, k, v, slots)
    assert not status.any()
    q = torch.randn((B, H, D), generator=gen, device="cuda").half()
    out, lse, _ = attention_kv4(q, cache, pages, torch.full((B,), n, dtype=torch.int32, device="cuda"))
    kk, vv, _ = read_kv4(cache, slots)
    kk, vv = (t.double().view(B, n, Hkv, D).repeat_interleave(H // Hkv, 2).transpose(1, 2) for t in (kk, vv))
    score = (q.double()[:, :, None] * kk).sum(-1) * D ** -0.5
    p = torch.softmax(score, -1)[..., None]
    want = (p * vv).sum(2)
    # read_kv4 rounds to fp16: 2^-11 of each entry, the scores' part of it weighs sum p |v|
    slip = ((q.abs().double()[:, :, None] * kk.abs()).sum(-1) * D ** -0.5 * 2.0 ** -11).amax(-1)[..., None]
    bound = (p * vv.abs()).sum(2) * (2 * slip + 2.0 ** -9) + 2.0 ** -10 * want.abs() + 2.0 ** -10
    assert bool(((out.double() - want).abs() <= bound).all())
    assert bool(((lse.double() - torch.logsumexp(score, -1)).abs() <= slip[..., 0] + 2.0 ** -16).all())


@gpu
def test_offsets_past_32_bits():
    """Pages at the end of a cache whose codes are over 4 GB."""
    page, heads, dim = 64, 8, 64
    pages = 2 ** 32 // (page * heads * 32) + 2
    cache = KvCache4.empty(pages, page, heads, dim)
    gen = torch.Generator(device="cuda").manual_seed(6)
    k = torch.randn((100, heads, dim), generator=gen, device="cuda").bfloat16()
    where = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    j = torch.arange(100, device="cuda")
    append_kv4(cache, k, -k, where[0, j // page].long() * page + j % page)
    small = KvCache4(*(t[[pages - 1, pages - 2]].contiguous() for t in cache._args[:4]), head_dim=dim, dtype=BF16)
    q = torch.randn((1, 16, dim), generator=gen, device="cuda").bfloat16()
    n = torch.tensor([100], dtype=torch.int32, device="cuda")
    got = attention_kv4(q, cache, where, n)
    want = attention_kv4(q, small, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), n)
    assert bool(got[0].any()) and all(torch.equal(x, y) for x, y in zip(got, want))


@gpu
def test_empty_batch():
    cache = KvCache4.empty(1, 16, 2, 64)
    out, lse, status = attention_kv4(torch.empty((0, 4, 64), dtype=BF16, device="cuda"), cache,
                                     torch.empty((0, 1), dtype=torch.int32, device="cuda"),
                                     torch.empty(0, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4) and status.shape == (0,)
    # rows without any pages
    out, lse, status = attention_kv4(torch.ones((3, 4, 64), dtype=BF16, device="cuda"), cache,
                                     torch.empty((3, 0), dtype=torch.int32, device="cuda"),
                                     torch.tensor([0, 1, 0], dtype=torch.int32, device="cuda"))
    assert not out.any() and bool((lse == -math.inf).all()) and status.tolist() == [0, _lib.MS_ROW_BAD_LENGTH, 0]


@gpu
def test_call_refusals():
    cache = KvCache4.empty(4, 16, 2, 64)
    q = torch.zeros((3, 2, 4, 64), dtype=BF16, device="cuda")
    pages = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    lengths = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    attention_kv4(q, cache, pages, lengths)
    for args, kw in (((q.half(), cache, pages, lengths), {}), ((q, cache, pages.long(), lengths), {}),
                     ((q, cache, pages, lengths.long()), {}), ((q, (cache,), pages, lengths), {}),
                     ((q, cache, pages, lengths), dict(out=q.half()))):
        with pytest.raises(TypeError):
            attention_kv4(*args, **kw)
    for args, kw in (((q[..., :48], cache, pages, lengths), {}), ((q[:, :, :3], cache, pages, lengths), {}),
                     ((q[:, :, :0], cache, pages, lengths), {}), ((q[:, :0], cache, pages, lengths[:, :0]), {}),
                     ((q, cache, pages[:2], lengths), {}), ((q, cache, pages, lengths[:, :1]), {}),
                     ((q, cache, pages, lengths[:, 0]), {}), ((q[:, 0], cache, pages, lengths), {}),
                     ((q[:, 0], cache, pages, lengths[:, 0]), {}),  # strided: rows of a wider tensor
                     ((q, cache, pages.cpu(), lengths), {}), ((q, cache, pages, lengths), dict(scale=0.0)),
                     ((q, cache, pages, lengths), dict(scale=math.nan)), ((q, cache, pages, lengths), dict(scale=1e39)),
                     ((q, cache, pages, lengths), dict(out=q[:2])),
                     ((q, cache, pages, lengths), dict(out=q[:, :, :1].expand(3, 2, 4, 64))),
                     ((q.expand(3, 2, 4, 64)[:, :, :, ::2], cache, pages, lengths), {})):
        with pytest.raises(ValueError):
            attention_kv4(*args, **kw)
    with pytest.raises(ValueError):
        attention_kv4(torch.zeros((1, 1025, 2, 64), dtype=BF16, device="cuda"), cache, pages[:1],
                      torch.zeros((1, 1025), dtype=torch.int32, device="cuda"))


def test_entry_point_refusals():
    """The C entry point refuses on the host, before any launch."""
    import ctypes
    L = _lib.lib()
    some = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(some) + 255) // 256 * 256

    def call(cache=None, **other):
        c = _lib.Kv4Cache(**{**dict(kv_heads=2, head_dim=64, pages=3, page_size=4, k_codes=p, k_params=p, v_codes=p,
                                    v_params=p), **(cache or {})})
        return L.ms_kv4_attention(_lib.Kv4AttentionArgs(**{**dict(
            dtype=1, tokens=1, heads=4, rows=1, q=p, cache=c, table=p, table_width=1, table_row=1, lengths=p, length_row=1,
            scale=1.0, out=p, lse=p, status=p, workspace=p, workspace_bytes=16), **other}), None)

    assert call(rows=0) == 0
    assert call(dtype=0) == -2
    for bad in (dict(rows=-1), dict(rows=(1 << 20) + 1), dict(tokens=0), dict(tokens=1025), dict(heads=0), dict(heads=3),
                dict(heads=65538), dict(rows=1 << 20, tokens=1024, heads=4), dict(table_width=-1), dict(table_row=-1),
                dict(length_row=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=3e38), dict(q=None),
                dict(table=None), dict(lengths=None), dict(out=None), dict(lse=None), dict(status=None),
                dict(workspace=None), dict(workspace=p + 128)):
        assert call(**bad) == -1, bad
    assert call(cache=dict(pages=0)) == -1 and call(cache=dict(head_dim=72)) == -4
    assert L.ms_kv4_attention(None, None) == -1
    assert L.ms_kv4_attention_workspace(1, 0, 4, 2, 64) == 0


def test_cpu_tensors_are_refused():
    cache = KvCache4.empty(1, 16, 2, 64, device="cpu")
    with pytest.raises(TypeError, match="CUDA"):
        attention_kv4(torch.zeros((1, 4, 64), dtype=BF16), cache, torch.zeros((1, 1), dtype=torch.int32),
                      torch.zeros(1, dtype=torch.int32))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("share", [0.5, 1.0])
@pytest.mark.parametrize("T,H,Hkv,D", [(1, 8, 2, 64), (1, 4, 1, 128), (5, 14, 2, 64), (3, 8, 1, 96)])
def test_scales_of_either_sign(T, H, Hkv, D, dtype, share):
    """m + s (c - 8) is m + (-s) ((16 - c) - 8): a cache of some scales' other
    sign stands for the same entries, whatever their size."""
    def scales(p):
        for codes in (p.cache.k_codes, p.cache.v_codes):  # no code of 0: 16 is none
            codes.copy_(codes | (((codes & 15) == 0) + 16 * ((codes >> 4) == 0)).to(torch.uint8))
        p.cache.v_params[..., :p.used_groups, 0] *= 2.0 ** 13
    p = Problem(3, T, H, Hkv, D, [300, 17, 90], 16, dtype=dtype, scales=scales)
    p.check(*p.run())
    gen = torch.Generator(device="cuda").manual_seed(18)
    mirrored = copy.copy(p)
    tensors = [t.clone() for t in p.cache._args[:4]]
    for codes, params in (tensors[:2], tensors[2:]):
        for g in range(params.shape[-2]):
            turn = torch.rand(params.shape[:3], generator=gen, device="cuda") < share
            part = codes[..., 16 * g:16 * g + 16]
            part.copy_(torch.where(turn[..., None], (16 - (part & 15)) | ((16 - (part >> 4)) << 4), part))
            params[..., g, 0] = torch.where(turn, -params[..., g, 0], params[..., g, 0])
    mirrored.cache = KvCache4(*tensors, head_dim=D, dtype=dtype)
    p.check(*mirrored.run())


@gpu
@pytest.mark.parametrize("spread,scale", [(1e35, None), (1.5, 1e35), (1e4, 1e31)])
@pytest.mark.parametrize("T,H,dtype", [(1, 4, BF16), (1, 8, BF16), (2, 14, BF16), (1, 4, FP16), (3, 8, FP16)])
def test_scores_near_the_end_of_fp32(T, H, dtype, spread, scale):
    """Scores of 1e35 and more: lse is the largest one, within what scores may be
    off by, and nothing is infinite or NaN."""
    if dtype == FP16:
        spread = min(spread, 1e4)
    p = Problem(2, T, H, 1 if H < 14 else 2, 64, [100, 3000], 16, dtype=dtype, spread=spread)
    by = 0.125 if scale is None else scale
    out, lse, status = p.run(scale=scale)
    assert not status.any() and bool(out.isfinite().all())
    for b in range(2):
        for t in range(T):
            c, s, z = p.keys(b, p.lens[b][t], p.cache.k_codes, p.cache.k_params)
            q = p.q[b, t].double().view(s.shape[0], -1, 64)
            want = (q @ (z + s * (c - 8)).transpose(1, 2)).amax(-1) * by
            mag = (q.abs() @ (s * (c + 8) + z.abs()).transpose(1, 2)).amax(-1) * by
            assert bool((mag < 2e38).all())
            assert bool(((lse[b, t].double().view_as(want) - want).abs() <= 2.0 ** -18 * mag).all())
