"""prefix_attention against its definition in 64 bits.

Tolerance, with u the unit roundoff of the type (2^-8 bf16, 2^-11 fp16), n the
row's keys, p the exact weights and A = scale max_j sum |q||k_j|:
a score's error is at most e = (D + 8) 2^-23 A (D products and sums in fp32,
the scaling); the weights are then off by a factor within 2 e + 2^-20 (the
exponential's argument and result), their rounding to the type by u more, or
2^-25 of the largest weight where fp16 is below its normal range; sums over n
keys by (n + 64) 2^-23.  So an output is within
(u + 4 e + 2^-19 + 2 (n + 64) 2^-23) sum p |v| + 2^-25 sum |v| plus its own
rounding, u |out|, and lse within 2 e + 2^-20 + (n + 64) 2^-23 + 2^-22 |lse|.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import _lib  # noqa: E402

gpu = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Problem:
    def __init__(self, B, H, Hkv, D, prefix, lens, page, order="nhd", dtype=torch.bfloat16, seed=1, spread=1.5,
                 hole=math.nan):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        used = [-(-n // page) for n in lens]
        n_prefix = -(-prefix // page)
        total = n_prefix + sum(used) + 1
        shape = (total, page, Hkv, D) if order == "nhd" else (total, Hkv, page, D)
        caches = []
        for _ in range(2):
            t = torch.randn(shape, generator=gen, device="cuda").to(dtype)
            caches.append(t if order == "nhd" else t.transpose(1, 2))
        self.ck, self.cv = caches
        perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32).cpu()
        self.prefix_pages = perm[:n_prefix].cuda()
        width = max(used + [1])
        table = torch.full((B, width + 1), -5, dtype=torch.int32)  # entries past the row's keys are not read
        at = n_prefix
        keep = torch.zeros((total, page), dtype=torch.bool)
        for i, p in enumerate(perm[:n_prefix].tolist()):
            keep[p, :min(page, prefix - i * page)] = True
        for b, n in enumerate(lens):
            table[b, :used[b]] = perm[at:at + used[b]]
            for i in range(used[b]):
                keep[int(perm[at + i]), :min(page, n - i * page)] = True
            at += used[b]
        # what no row sees may hold anything
        self.ck[~keep.cuda()] = hole
        self.cv[~keep.cuda()] = hole
        self.pages = table.cuda()[:, :width]
        self.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.q = (torch.randn((B, H, D), generator=gen, device="cuda") * spread).to(dtype)
        self.prefix, self.lens, self.page = prefix, lens, page

    def run(self, **kw):
        from miniserve_b200.attention import prefix_attention
        return prefix_attention(self.q, self.ck, self.cv, self.pages, self.lengths, prefix_pages=self.prefix_pages,
                                prefix_length=self.prefix, **kw)

    def keys(self, b, cache):
        parts = []
        if self.prefix:
            parts.append(cache[self.prefix_pages.long()].flatten(0, 1)[:self.prefix])
        if self.lens[b]:
            n = -(-self.lens[b] // self.page)
            parts.append(cache[self.pages[b, :n].long()].flatten(0, 1)[:self.lens[b]])
        return torch.cat(parts).double() if parts else None  # [n, Hkv, D]

    def check(self, out, lse, status, scale=None, rows=None):
        B, H, D = self.q.shape
        G = H // self.ck.shape[2]
        u = UNIT[self.q.dtype]
        scale = D ** -0.5 if scale is None else scale
        assert not status.any()
        for b in rows if rows is not None else range(B):
            k = self.keys(b, self.ck)
            if k is None:
                assert not out[b].any() and bool((lse[b] == -math.inf).all())
                continue
            n = k.shape[0]
            k = k.repeat_interleave(G, 1).transpose(0, 1)              # [H, n, D]
            v = self.keys(b, self.cv).repeat_interleave(G, 1).transpose(0, 1)
            q = self.q[b].double()[:, None]
            s = (q * k).sum(-1) * scale
            mag = ((q.abs() * k.abs()).sum(-1) * scale).amax(-1)
            want_lse = torch.logsumexp(s, -1)
            p = (s - want_lse[:, None]).exp()[..., None]
            want, room = (p * v).sum(1), (p * v.abs()).sum(1)
            e = ((D + 8) * 2.0 ** -23 * mag)[:, None]
            sums = (n + 64) * 2.0 ** -23
            bound = (u + 4 * e + 2.0 ** -19 + 2 * sums) * room + 2.0 ** -25 * v.abs().sum(1) + u * want.abs() + 2.0 ** -25
            err = (out[b].double() - want).abs()
            assert bool((err <= bound).all()), (b, float((err - bound).max()))
            tol = 2 * e[:, 0] + 2.0 ** -20 + sums + 2.0 ** -22 * want_lse.abs()
            assert bool(((lse[b].double() - want_lse).abs() <= tol).all()), b


CASES = [
    # B, heads, kv_heads, D, prefix, lens, page, order
    (1, 1, 1, 8, 0, [1], 1, "nhd"),
    (1, 14, 2, 64, 0, [300], 16, "nhd"),
    (1, 8, 1, 128, 3000, [17], 64, "hnd"),
    (2, 4, 4, 64, 1, [0, 1], 16, "nhd"),
    (3, 14, 2, 64, 15, [0, 16, 17], 16, "nhd"),
    (5, 7, 1, 64, 16, [1, 0, 33, 0, 128], 8, "hnd"),
    (4, 8, 8, 128, 129, [5, 250, 64, 0], 24, "nhd"),
    (3, 40, 2, 80, 257, [100, 3, 0], 24, "hnd"),        # groups of 20: two chunks of heads
    (9, 32, 1, 16, 40, list(range(9)), 7, "nhd"),
    (2, 66, 1, 128, 130, [31, 0], 16, "nhd"),
    (40, 4, 2, 96, 500, [(7 * i) % 41 for i in range(40)], 16, "nhd"),
    (130, 14, 2, 64, 1000, [(13 * i) % 150 for i in range(130)], 16, "hnd"),
    (37, 8, 1, 128, 128, [1] * 37, 64, "nhd"),
    (16, 16, 1, 64, 256, [0] * 16, 128, "nhd"),
    (300, 3, 1, 40, 127, [i % 3 for i in range(300)], 3, "nhd"),
    (6, 12, 4, 128, 2049, [2048, 1, 0, 999, 16, 15], 1, "hnd"),
    (3, 4, 2, 64, 0, [0, 0, 0], 16, "nhd"),
    (3, 6, 2, 56, 0, [0, 5000, 1], 16, "nhd"),
    (8, 8, 2, 64, 20000, [3] * 8, 16, "nhd"),
    (40, 4, 2, 48, 300, [i % 19 for i in range(40)], 16, "nhd"),   # boxes wider than a head
    (40, 4, 1, 24, 200, [i % 7 for i in range(40)], 32, "hnd"),
    (40, 4, 1, 72, 333, [i % 33 for i in range(40)], 128, "nhd"),
    (21, 5, 5, 88, 640, [40] * 21, 8, "hnd"),
    (2, 2, 1, 128, 9000, [6000, 7], 48, "nhd"),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_matches_definition(case, dtype):
    B, H, Hkv, D, prefix, lens, page, order = case
    p = Problem(B, H, Hkv, D, prefix, lens, page, order, dtype, seed=B * 1000 + D)
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix", [0, 700])
def test_sharp_and_growing_scores(dtype, prefix):
    """Scores that grow along the keys (every tile a new maximum, by large
    steps), and queries that settle on single keys."""
    p = Problem(20, 8, 2, 64, prefix, [(29 * i) % 200 for i in range(20)], 16, "nhd", dtype, seed=8, spread=6.0)
    ramp = torch.linspace(0.05, 4.0, p.ck.shape[0], device="cuda")[:, None, None, None].to(dtype)
    p.ck.mul_(ramp)
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("B,H,Hkv,D,prefix", [(512, 14, 2, 64, 4097), (512, 14, 2, 64, 700), (300, 32, 4, 128, 1500),
                                              (1000, 8, 1, 64, 257), (64, 64, 8, 128, 3000), (5000, 4, 2, 64, 100),
                                              (5000, 4, 2, 64, 0)])
def test_grids_of_every_sm(B, H, Hkv, D, prefix):
    """Two CTAs on every SM, and more than one wave of them."""
    p = Problem(B, H, Hkv, D, prefix, [(7 * i) % 40 for i in range(B)], 16, "nhd", torch.bfloat16, seed=B)
    p.check(*p.run(), rows=[0, 1, B // 3, B // 2, B - 2, B - 1])
    first, second = p.run(), p.run()
    assert torch.equal(first[0], second[0]) and bool(first[0].isfinite().all())


@gpu
@pytest.mark.parametrize("scale", [1e-3, 0.5, 1.0])
def test_scale_and_strided_tensors(scale):
    p = Problem(33, 6, 2, 64, 200, [(5 * i) % 77 for i in range(33)], 16, "nhd", torch.bfloat16, seed=4)
    wide = torch.zeros((33, 10, 64), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:8] = p.q
    p.q = wide[:, 2:8]
    room = torch.full((33, 7, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    out, lse, status = p.run(scale=scale, out=room[:, :6, :64])
    p.check(out, lse, status, scale=scale)
    assert bool((room[:, 6] == 9.0).all()) and bool((room[..., 64:] == 9.0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Hkv,D,prefix", [(33, 6, 2, 64, 200), (130, 8, 1, 128, 130), (3, 6, 2, 72, 50),
                                              (5, 40, 2, 80, 0)])
@pytest.mark.parametrize("offset,gap", [(1, 0), (0, 3), (4, 4)])
def test_queries_off_the_16_byte_grid(B, H, Hkv, D, prefix, offset, gap, dtype):
    """A base, or strides, that 16-byte reads of the queries do not fit: the
    prefix kernel (first two), a prefix of few rows and plain rows."""
    p = Problem(B, H, Hkv, D, prefix, [(5 * i) % 77 for i in range(B)], 16, "nhd", dtype, seed=B + D)
    flat = torch.full((offset + B * H * (D + gap),), math.nan, dtype=dtype, device="cuda")
    view = flat[offset:].view(B, H, D + gap)[..., :D]
    view.copy_(p.q)
    p.q = view
    assert view.data_ptr() % 16 or view.stride(1) % 8
    p.check(*p.run())


@gpu
def test_keys_and_values_in_one_allocation_of_wide_slots():
    """K and V interleaved in one tensor (different bases, equal odd strides)."""
    p = Problem(17, 8, 4, 64, 90, [(11 * i) % 60 for i in range(17)], 16, "nhd", torch.float16, seed=6)
    both = torch.full((*p.ck.shape[:2], 3, p.ck.shape[2], 64), math.nan, dtype=torch.float16, device="cuda")
    both[:, :, 0], both[:, :, 2] = p.ck, p.cv
    p.ck, p.cv = both[:, :, 0], both[:, :, 2]
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("hole", [math.inf, -math.inf, 65504.0])
def test_unseen_entries_do_not_matter(hole):
    p = Problem(20, 8, 2, 128, 333, [(17 * i) % 90 for i in range(20)], 16, "nhd", torch.float16, seed=7, hole=hole)
    p.check(*p.run())


@gpu
def test_values_that_are_not_finite_stay_in_their_rows():
    p = Problem(20, 4, 2, 64, 300, [20] * 20, 16, "nhd", torch.bfloat16, seed=12)
    p.cv[p.pages[3, 0].long(), 2, 0, 5] = math.nan
    p.ck[p.pages[4, 1].long(), 1, 1, 0] = math.nan
    out, lse, status = p.run()
    assert bool(out[3, :2, 5].isnan().all()) and int(out[3].isnan().sum()) == 2
    assert bool(out[4, 2:].isnan().all()) and bool(lse[4, 2:].isnan().all()) and not bool(out[4, :2].isnan().any())
    p.check(out, lse, status, rows=[b for b in range(20) if b not in (3, 4)])


@gpu
def test_equal_calls_give_equal_bits_on_any_stream():
    p = Problem(100, 14, 2, 64, 1500, [(37 * i) % 300 for i in range(100)], 16, "nhd", torch.bfloat16, seed=3)
    first = p.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = p.run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("prefix", [0, 200])
def test_bad_rows_are_flagged(prefix):
    p = Problem(8, 4, 2, 64, prefix, [30] * 8, 16, "nhd", torch.bfloat16, seed=2)
    p.lengths[1] = -1
    p.lengths[2] = 33         # two pages of 16
    p.lengths[3] = 2 ** 31 - 1
    p.pages[4, 1] = p.ck.shape[0]
    p.pages[5, 0] = -1
    out, lse, status = p.run()
    L, P = _lib.MS_ROW_BAD_LENGTH, _lib.MS_ROW_BAD_PAGE
    assert status.tolist() == [0, L, L, L, P, P, 0, 0]
    assert not out[1:6].any() and bool((lse[1:6] == -math.inf).all())
    status.zero_()
    p.check(out, lse, status, rows=[0, 6, 7])
    if prefix:
        p.prefix_pages[-1] = 1 << 30
        out, lse, status = p.run()
        assert bool((status & P != 0).all()) and not out.any()


@gpu
def test_cache_offsets_past_32_bits():
    """A page whose first entry lies past 2^32 entries of the cache."""
    free, _ = torch.cuda.mem_get_info()
    if free < 22 << 30:
        pytest.skip("needs 20 GB of device memory")
    pages = (1 << 32) // (64 * 128) + 4
    ck = torch.empty((pages, 64, 1, 128), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    ck[-3:] = torch.randn((3, 64, 1, 128), generator=gen, device="cuda").bfloat16()
    ck[:3] = 0
    p = Problem(20, 2, 1, 128, 50, [40] * 20, 64, seed=5)
    p.ck = p.cv = ck
    p.prefix_pages = torch.tensor([pages - 1], dtype=torch.int32, device="cuda")
    p.pages = torch.full((20, 1), pages - 2, dtype=torch.int32, device="cuda")
    p.check(*p.run())


@gpu
@pytest.mark.parametrize("dtype,top", [(torch.bfloat16, 1e6), (torch.float16, 6e4)])
@pytest.mark.parametrize("prefix,own", [(200, 20), (0, 200)])
def test_scores_past_the_integers_of_fp32(dtype, top, prefix, own):
    """Finite scores of 1e9 and more, where neighbouring fp32 numbers are
    hundreds apart: a key ahead of the others by half of that has weight 1 and
    they have none, so that out is its value (two fp32 roundings and the
    type's) and lse its score (the product's, the scale's and lse's own
    roundings: 2^-22 of it)."""
    p = Problem(40, 8, 2, 64, prefix, [own] * 40, 16, "nhd", dtype, seed=31)
    gen = torch.Generator(device="cuda").manual_seed(32)
    factor = (0.5 + torch.rand((40, 8), generator=gen, device="cuda")) * 0.6 * top
    p.q.zero_()
    p.q[..., 0] = factor.to(dtype)
    near = torch.rand(p.ck.shape[:3], generator=gen, device="cuda") * 0.5 * top
    p.ck[..., 0] = torch.where(p.ck[..., 0].isnan(), math.nan, near).to(dtype)
    pages = p.prefix_pages[None].expand(40, -1) if prefix else p.pages
    at = (pages[:, 77 // 16].long(), 77 % 16)  # key 77 of the prefix, or of every row
    p.ck[(*at, slice(None), 0)] = top
    out, lse, status = p.run(scale=1.0)
    assert not status.any()
    want = p.cv[at].double().repeat_interleave(4, 1)
    bound = want.abs() * (UNIT[dtype] + 2.0 ** -22)
    assert bool(((out.double() - want).abs() <= bound).all())
    score = p.q[..., 0].double() * torch.tensor(top, device="cuda").to(dtype).double()
    assert bool(((lse.double() - score).abs() <= score * 2.0 ** -22).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prefix,own", [(500, 3), (3, 500), (0, 700)])
@pytest.mark.parametrize("drop", [9.7, 13.9, 16.264])
def test_keys_far_below_the_largest_keep_their_share(dtype, prefix, own, drop):
    """A first key takes nearly all the weight and has a value of zero, as
    trained heads' first tokens do; what is left comes from keys exp(-drop)
    below it.  Their weights are rounded to the type relative to themselves
    down to 2^-21 of the largest (fp16's normal range, the weights scaled up
    by at least 2^7), by 2^-32 of the largest below that."""
    p = Problem(40, 8, 2, 64, prefix, [own] * 40, 16, "nhd", dtype, seed=33)
    gen = torch.Generator(device="cuda").manual_seed(34)
    p.q.zero_()
    p.q[..., 0] = 8.0  # a score is k[0], as the scale is 1 / 8
    p.ck[..., 0] = torch.where(p.ck[..., 0].isnan(), math.nan, -drop).to(dtype)
    p.cv[:] = torch.where(p.cv.isnan(), math.nan, 500 + 1000 * torch.rand(p.cv.shape, generator=gen, device="cuda"))
    first = p.prefix_pages[:1] if prefix else p.pages[:, 0]
    p.ck[first.long(), 0, :, 0] = 0
    p.cv[first.long(), 0] = 0
    out, lse, status = p.run()
    assert not status.any()
    u = UNIT[dtype]
    for b in (0, 17, 39):
        k, v = (p.keys(b, c).repeat_interleave(4, 1).transpose(0, 1) for c in (p.ck, p.cv))
        s = (p.q[b].double()[:, None] * k).sum(-1) / 8
        want = (torch.softmax(s, -1)[..., None] * v).sum(1)
        e, sums = 72 * 2.0 ** -23 * drop, (k.shape[1] + 64) * 2.0 ** -23
        bound = (2 * u + 4 * e + 2.0 ** -19 + 2 * sums) * want + 2.0 ** -32 * v.sum(1) + 2.0 ** -25
        err = (out[b].double() - want).abs()
        assert bool((err <= bound).all()), (b, float((err / want).max()))


@gpu
def test_reads_what_append_wrote():
    from miniserve_b200.kvcache import append_kv, rope_table
    p = Problem(6, 8, 2, 64, 40, [3, 16, 0, 20, 31, 8], 16, "nhd", torch.bfloat16, seed=21, hole=0.0)
    gen = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn((6, 12, 64), generator=gen, device="cuda").bfloat16()
    table = torch.full((6, 3), -1, dtype=torch.int32, device="cuda")
    table[:, :p.pages.shape[1]] = p.pages
    spare = int(p.prefix_pages.max()) * 0 + p.ck.shape[0]
    more = torch.zeros((6, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
    p.ck, p.cv = torch.cat([p.ck, more]), torch.cat([p.cv, more])
    lens = p.lengths.clone()
    for b, n in enumerate(p.lens):
        if n % 16 == 0:
            table[b, n // 16] = spare + b
    rows = torch.arange(6, device="cuda")
    slots = table[rows, (lens // 16).long()].long() * 16 + lens.long() % 16
    p.q, status = append_kv(p.ck, p.cv, qkv[:, 8:10], qkv[:, 10:], slots, q=qkv[:, :8], positions=lens.long() + 40,
                            rope=rope_table(128, 64))
    assert not status.any()
    p.pages, p.lengths, p.lens = table, lens + 1, [n + 1 for n in p.lens]
    p.check(*p.run())


@gpu
def test_refusals():
    from miniserve_b200.attention import prefix_attention
    c = torch.zeros((4, 8, 2, 16), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((3, 4, 16), dtype=torch.bfloat16, device="cuda")
    t = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    ok = dict(q=q, cache_k=c, cache_v=c, pages=t, lengths=n)
    prefix_attention(**ok)
    odd = torch.zeros((4, 8, 2, 20), dtype=torch.bfloat16, device="cuda")
    big = torch.zeros((1, 8, 1, 136), dtype=torch.bfloat16, device="cuda")
    for err, change in [
        (TypeError, dict(q=q.half())), (ValueError, dict(q=q[:, :3])), (ValueError, dict(q=q[..., :8])),
        (TypeError, dict(pages=t.long())), (TypeError, dict(lengths=n.long())), (ValueError, dict(lengths=n[:2])),
        (ValueError, dict(pages=t[:2])), (ValueError, dict(cache_v=c[:2])), (TypeError, dict(cache_k=c.cpu())),
        (ValueError, dict(prefix_length=1)), (ValueError, dict(prefix_pages=t[0], prefix_length=17)),
        (ValueError, dict(prefix_length=-1)), (TypeError, dict(prefix_pages=t[0].long(), prefix_length=1)),
        (ValueError, dict(scale=0.0)), (ValueError, dict(scale=-1.0)), (ValueError, dict(scale=math.nan)),
        (ValueError, dict(scale=math.inf)), (ValueError, dict(out=q[:2])), (TypeError, dict(out=q.float())),
        (ValueError, dict(out=q[:1].expand(3, 4, 16))),
        (ValueError, dict(cache_k=odd[..., :16], cache_v=odd[..., 4:])),
        (ValueError, dict(cache_k=odd, cache_v=odd, q=torch.zeros((3, 4, 20), dtype=torch.bfloat16, device="cuda"))),
        (ValueError, dict(cache_k=big, cache_v=big, q=torch.zeros((3, 1, 136), dtype=torch.bfloat16, device="cuda"))),
    ]:
        with pytest.raises(err):
            prefix_attention(**{**ok, **change})


def test_c_entry_refuses_bad_arguments():
    import ctypes
    L = _lib.lib()
    assert L.ms_prefix_attention(None, None) == -1
    a = _lib.PrefixAttentionArgs()
    assert L.ms_prefix_attention(ctypes.byref(a), None) == -2
    a.dtype, a.heads, a.kv_heads, a.head_dim, a.pages, a.page_size, a.scale = _lib.MS_DTYPE_F16, 4, 2, 64, 1, 16, 1.0
    assert L.ms_prefix_attention(ctypes.byref(a), None) == 0    # no rows
    for field, bad, code in [("heads", 3, -1), ("head_dim", 36, -4), ("head_dim", 136, -4), ("ck_page", 4, -4),
                             ("cache_v", 8, -4), ("scale", 0.0, -1), ("scale", math.nan, -1), ("page_size", 0, -1),
                             ("prefix_length", -1, -1), ("rows", -1, -1), ("rows", 1, -1)]:
        keep = getattr(a, field)
        setattr(a, field, bad)
        assert L.ms_prefix_attention(ctypes.byref(a), None) == code, field
        setattr(a, field, keep)
    assert L.ms_prefix_attention_workspace(1, 3, 2, 64, 0) == 0
