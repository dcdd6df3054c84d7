"""append_kv4 and read_kv4 against the format's definition in 64 bits.

Tolerance of a stored entry y (a rotated key or a value) in a group of minimum
lo and maximum hi, t = (hi - lo) / 15:

* scale s is t rounded to fp16: within 2^-11 t, or 2^-25 below fp16's normal
  range; middle m is lo + 8 s rounded to fp16: within 2^-11 |m| + 2^-25;
* a code inside its range is within s / 2 of y; at the range's ends lo is
  m - 8 s and hi is m + 7 s up to those two roundings, so that clamping adds at
  most 2^-11 |m| + 15 (2^-11 t + 2^-25);
* fp32's roundings of differences and products, 2^-24 of each, are below
  2^-20 (|lo| + |hi|) together, and the rotation's below 3 * 2^-24 (|a c| + |b s|);
* reading back rounds once: half a unit in the last place, 2^-8 of bf16's value
  and 2^-11 of fp16's (2^-25 below its normal range).
"""
import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import KvCache4, _lib, append_kv4, read_kv4, rope_table  # noqa: E402

gpu = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, FP16 = torch.bfloat16, torch.float16


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def turned(x, table, interleaved):
    """(rotated, bound of fp32's error) of x [T, H, D] by table rows [T, rotary]."""
    x = x.double()
    half = table.shape[1] // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = table[:, None, :half].double(), table[:, None, half:].double()
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    mag[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    mag[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, mag * 3 * 2.0 ** -24


def held_within(got, y, slack, dtype):
    """got [T, H, D] (what read_kv4 gives) stands for y up to the format's tolerance."""
    for g in range(0, y.shape[-1], 32):
        z, d = y[..., g:g + 32], slack[..., g:g + 32].amax(-1, keepdim=True)
        lo, hi = z.amin(-1, keepdim=True) - d, z.amax(-1, keepdim=True) + d
        t = (hi - lo) / 15
        s = t * (1 + 2.0 ** -11) + 2.0 ** -25
        m = (lo + 8 * s).abs() + (hi - lo) * 2.0 ** -8
        bound = s / 2 + 2.0 ** -11 * m + 2.0 ** -25 + 15 * (2.0 ** -11 * t + 2.0 ** -25)
        bound = bound + 2.0 ** -20 * (lo.abs() + hi.abs()) + d
        bound = bound + (z.abs() + bound) * HALF_ULP[dtype] + 2.0 ** -25
        err = (got[..., g:g + 32].double() - z).abs()
        assert bool((err <= bound).all()), float((err - bound).max())


def decoded(codes, params, dim):
    """What codes [..., bytes] and params [..., groups, 2] stand for, in 64 bits."""
    i = torch.arange(dim, device=codes.device)
    code = (codes[..., i // 2].int() >> (4 * (i % 2))) & 15
    return params[..., i // 32, 1].double() + params[..., i // 32, 0].double() * (code - 8).double()


def filled(pages, page, heads, dim, dtype, seed):
    """A cache of random codes and parameters."""
    gen = generator(seed)
    cache = KvCache4.empty(pages, page, heads, dim, dtype=dtype)
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device="cuda", dtype=torch.uint8))
        params[..., 0] = torch.rand(params.shape[:-1], generator=gen, device="cuda") * 0.3
        params[..., 1] = torch.randn(params.shape[:-1], generator=gen, device="cuda") * 0.5
    return cache


def at_slots(t, slots, page):
    """[T, heads, ...] of a cache's tensor at slots."""
    return t[slots // page, :, slots % page]


SHAPES = [
    # dtype, T, heads, kv_heads, dim, rotary, interleaved, page, slices of one tensor
    (BF16, 1, 14, 2, 64, 64, False, 16, True),
    (FP16, 77, 8, 8, 128, 128, False, 64, True),
    (BF16, 130, 6, 3, 80, 40, True, 24, False),
    (FP16, 33, 4, 2, 48, 24, False, 8, True),   # 12 pairs: pieces of four
    (BF16, 19, 5, 5, 112, 56, False, 5, False),  # 28 pairs
    (BF16, 9, 3, 1, 96, 12, False, 16, True),   # 6 pairs: single entries
    (FP16, 21, 2, 1, 16, 16, True, 1, True),
    (BF16, 40, 4, 4, 32, 2, True, 7, False),
    (FP16, 3, 2, 2, 128, 0, False, 16, True),
    (BF16, 300, 0, 2, 64, 64, False, 16, True),  # no queries
    (FP16, 2500, 32, 8, 128, 64, True, 64, True),  # several blocks' items a thread
]


@gpu
@pytest.mark.parametrize("dtype,T,heads,kv,dim,rotary,interleaved,page,fused", SHAPES)
def test_append_and_read(dtype, T, heads, kv, dim, rotary, interleaved, page, fused):
    gen = generator(1)
    qkv = torch.randn((T, heads + 2 * kv, dim), generator=gen, device="cuda").to(dtype)
    qkv[:, :, ::13] *= 5
    q, k, v = qkv.split([heads, kv, kv], 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pages = T // page + 4
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T]
    if T > 4:
        slots[3] = -1
        slots[4] = pages * page
    positions = torch.randint(0, 50, (T,), generator=gen, device="cuda")
    if T > 6 and rotary:
        positions[5], positions[6] = -1, 50
    rope = rope_table(50, rotary) if rotary else None
    cache = filled(pages, page, kv, dim, dtype, 2)
    before = [t.clone() for t in cache._args[:4]]
    q_out, status = append_kv4(cache, k, v, slots, q=q if heads else None, positions=positions, rope=rope,
                               interleaved=interleaved)
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    want = torch.zeros(T, dtype=torch.int32, device="cuda")
    if T > 4:
        good[3] = good[4] = False
        want[4] = _lib.MS_ROW_BAD_SLOT
    if T > 6 and rotary:
        good[5] = good[6] = False
        want[5] = want[6] = _lib.MS_ROW_BAD_POSITION
    assert torch.equal(status, want)
    table = (rope.reshape(50, -1)[positions.clamp(0, 49)] if rotary else qkv.new_zeros((T, 0)).float())
    kk, slack = turned(k, table, interleaved)
    got_k, got_v, read = read_kv4(cache, slots)
    assert torch.equal(read, torch.where(want == _lib.MS_ROW_BAD_SLOT, want, 0))
    held_within(got_k[good], kk[good], slack[good], dtype)
    held_within(got_v[good], v.double()[good], torch.zeros_like(slack)[good], dtype)
    if T > 4:
        assert not bool(got_k[3:5].any()) and not bool(got_v[3:5].any())
    # no other slot's bytes have changed
    touched = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    touched[slots[good]] = True
    rest = torch.arange(pages * page, device="cuda")[~touched]
    for t, old in zip(cache._args[:4], before):
        assert torch.equal(at_slots(t, rest, page), at_slots(old, rest, page))
    if heads:
        qq, qs = turned(q, table, interleaved)
        if T > 6 and rotary:
            qq[5:7] = qs[5:7] = 0
        bound = qq.abs() * HALF_ULP[dtype] + qs * (1 + HALF_ULP[dtype]) + 2.0 ** -25
        assert bool(((q_out.double() - qq).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_read_of_any_codes(dim, dtype):
    page, heads = 12, 3
    cache = filled(30, page, heads, dim, dtype, dim)
    slots = torch.randint(0, 360, (501,), generator=generator(3), device="cuda")  # repeated ones too
    out = torch.empty((2, 501, heads, dim + 3), dtype=dtype, device="cuda")  # rows off the 16-byte grid
    for ks, vs in ((None, None), (out[0, ..., :dim], out[1, ..., :dim])):
        k, v, status = read_kv4(cache, slots, k_out=ks, v_out=vs)
        assert not bool(status.any())
        for got, codes, params in ((k, cache.k_codes, cache.k_params), (v, cache.v_codes, cache.v_params)):
            want = decoded(at_slots(codes, slots, page), at_slots(params, slots, page), dim)
            err = (got.double() - want).abs()  # the fp32 sum of an exact product and m: 2^-24, then the type's rounding
            assert bool((err <= want.abs() * (HALF_ULP[dtype] + 2.0 ** -23) + 2.0 ** -25).all())


@gpu
def test_read_within_fp16():
    """An fp16 cache's finite entries read back finite, whatever a step past the largest one says."""
    v = torch.linspace(-65504, 65504, 64, device="cuda").half().view(1, 1, 64)
    cache = KvCache4.empty(1, 1, 1, 64, dtype=FP16)
    slot = torch.zeros(1, dtype=torch.int64, device="cuda")
    _, status = append_kv4(cache, v, -v, slot)
    assert int(status[0]) == 0
    k, w, _ = read_kv4(cache, slot)
    assert bool(k.isfinite().all()) and bool(w.isfinite().all())
    held_within(k, v.double(), torch.zeros_like(v).double(), FP16)
    held_within(w, -v.double(), torch.zeros_like(v).double(), FP16)


@gpu
@pytest.mark.parametrize("dtype,bad", [(BF16, float("nan")), (BF16, float("inf")), (BF16, -float("inf")), (BF16, 3e38),
                                       (BF16, -1e6), (FP16, float("nan")), (FP16, float("inf"))])
def test_what_is_not_held_reads_as_nan(dtype, bad):
    gen = generator(5)
    k = torch.randn((4, 2, 80), generator=gen, device="cuda").to(dtype)
    v = torch.randn((4, 2, 80), generator=gen, device="cuda").to(dtype)
    k[1, 1, 40] = bad
    v[2, 0, 79] = bad
    slots = torch.tensor([5, 9, 0, -1], device="cuda")
    k[3, 0, 0] = float("nan")  # padding: not looked at
    cache = KvCache4.empty(3, 4, 2, 80, dtype=dtype)
    _, status = append_kv4(cache, k, v, slots)
    assert status.tolist() == [0, _lib.MS_ROW_NONFINITE, _lib.MS_ROW_NONFINITE, 0]
    got_k, got_v, _ = read_kv4(cache, slots)
    nan_k, nan_v = torch.zeros_like(k, dtype=torch.bool), torch.zeros_like(v, dtype=torch.bool)
    nan_k[1, 1, 32:64] = True
    nan_v[2, 0, 64:80] = True
    assert torch.equal(got_k.isnan(), nan_k) and torch.equal(got_v.isnan(), nan_v)
    zero = torch.zeros(3, 2, 80, device="cuda", dtype=torch.float64)
    held_within(torch.where(nan_k, 0, got_k)[:3], torch.where(nan_k, 0, k)[:3].double(), zero, dtype)
    held_within(torch.where(nan_v, 0, got_v)[:3], torch.where(nan_v, 0, v)[:3].double(), zero, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_flat_and_tiny_groups(dtype):
    """Constant groups are exact; ranges below fp16's smallest steps, and offsets far beyond a range, stay within the bound."""
    rows = torch.stack([torch.full((64,), 1.5), torch.zeros(64), torch.full((64,), -3.0e-5), torch.linspace(0, 1e-7, 64),
                        torch.linspace(0, 3e-6, 64), 1000 + torch.linspace(0, 4, 64), torch.linspace(-1e-4, 1e-4, 64)])
    k = rows.to(dtype).cuda()[:, None]
    cache = KvCache4.empty(7, 1, 1, 64, dtype=dtype)
    slots = torch.arange(7, device="cuda")
    _, status = append_kv4(cache, k, k, slots)
    assert not bool(status.any())
    got, again, _ = read_kv4(cache, slots)
    assert torch.equal(got, again)
    held_within(got, k.double(), torch.zeros_like(k).double(), dtype)
    assert torch.equal(got[:2], k[:2])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(80, 80), (128, 64), (64, 24), (48, 12)])
def test_queries_in_place(dim, rotary, interleaved):
    gen = generator(7)
    qkv = torch.randn((500, 9, dim), generator=gen, device="cuda").bfloat16()
    q, k, v = qkv.split([5, 2, 2], 1)
    rope, positions = rope_table(64, rotary), torch.randint(0, 64, (500,), generator=gen, device="cuda")
    caches = [KvCache4.empty(40, 16, 2, dim) for _ in range(2)]
    slots = torch.randperm(640, generator=gen, device="cuda")[:500]
    want, _ = append_kv4(caches[0], k, v, slots, q=q, positions=positions, rope=rope, interleaved=interleaved)
    got, _ = append_kv4(caches[1], k, v, slots, q=q, positions=positions, rope=rope, interleaved=interleaved, q_out=q)
    assert got is q and torch.equal(got, want)
    for a, b in zip(caches[0]._args[:4], caches[1]._args[:4]):
        assert torch.equal(a, b)


@gpu
def test_same_bytes_from_any_strides():
    """Rows off the 16-byte grid, another order of heads and tokens, a range of pages: the cache's bytes are the same."""
    gen = generator(8)
    k = torch.randn((100, 4, 64), generator=gen, device="cuda").half()
    v = torch.randn((100, 4, 64), generator=gen, device="cuda").half()
    rope, positions = rope_table(100, 64), torch.arange(100, device="cuda")
    slots = torch.randperm(128, generator=gen, device="cuda")[:100]
    want = KvCache4.empty(8, 16, 4, 64, dtype=FP16)
    append_kv4(want, k, v, slots, positions=positions, rope=rope)
    odd = torch.empty((100, 4, 67), dtype=FP16, device="cuda")[..., 1:65]
    four = torch.empty((100, 4, 68), dtype=FP16, device="cuda")[..., 4:68]
    heads_first = torch.empty((4, 100, 64), dtype=FP16, device="cuda").transpose(0, 1)
    for other in (odd, four, heads_first):
        whole = KvCache4.empty(12, 16, 4, 64, dtype=FP16)
        part = whole[3:11]
        other.copy_(k)
        append_kv4(part, other, v, slots, positions=positions, rope=rope)
        for a, b in zip(want._args[:4], part._args[:4]):
            assert torch.equal(a, b)
        assert not bool(whole[:3].k_codes.any()) and not bool(whole[11:].v_codes.any())


@gpu
def test_empty_call_and_streams():
    cache = KvCache4.empty(4, 16, 2, 64)
    none = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    q_out, status = append_kv4(cache, none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert q_out is None and status.shape == (0,)
    assert read_kv4(cache, torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)
    gen = generator(9)
    k = torch.randn((30, 2, 64), generator=gen, device="cuda").bfloat16()
    slots = torch.arange(30, device="cuda")
    append_kv4(cache, k, -k, slots)
    want = read_kv4(cache, slots)
    torch.cuda.synchronize()
    # on another stream, and captured: what is replayed reads the buffers' new contents
    side = torch.cuda.Stream()
    other = KvCache4.empty(4, 16, 2, 64)
    buffer = torch.zeros_like(k)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        append_kv4(other, buffer, buffer, slots)
        read_kv4(other, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_kv4(other, buffer, buffer, slots)
        got = read_kv4(other, slots)
    buffer.copy_(k)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], got[0])


@gpu
def test_offsets_past_32_bits():
    """A cache whose codes are over 4 GB: its last slots are its own."""
    page, heads = 64, 8
    pages = 2 ** 32 // (page * heads * 32) + 2
    cache = KvCache4.empty(pages, page, heads, 64)
    gen = generator(10)
    k = torch.randn((5, heads, 64), generator=gen, device="cuda").bfloat16()
    last = pages * page - 1
    slots = torch.tensor([last, last - 64, 0, 2 ** 32 // (heads * 32) - 2, 1], device="cuda")
    _, status = append_kv4(cache, k, -k, slots)
    assert not bool(status.any())
    got_k, got_v, _ = read_kv4(cache, slots)
    held_within(got_k, k.double(), torch.zeros_like(k).double(), BF16)
    held_within(got_v, -k.double(), torch.zeros_like(k).double(), BF16)
    want = decoded(cache.k_codes[-1, :, -1], cache.k_params[-1, :, -1], 64)
    assert bool(((got_k[0].double() - want).abs() <= want.abs() * 2.0 ** -7).all())
    assert int(cache.k_codes[:, :, 2:62].count_nonzero()) == 0


def test_cache_refusals():
    codes = torch.zeros((3, 2, 4, 48), dtype=torch.uint8)
    params = torch.zeros((3, 2, 4, 4, 2), dtype=torch.float16)
    good = dict(head_dim=80, dtype=BF16)
    cache = KvCache4(codes, params, codes.clone(), params.clone(), **good)
    assert (cache.pages, cache.kv_heads, cache.page_size, cache.nbytes) == (3, 2, 4, 2 * (24 * 48 + 24 * 16))
    assert cache[1:].pages == 2
    with pytest.raises(TypeError):
        cache[1]
    for kinds in ((codes.int(), params, codes, params), (codes, params.float(), codes, params), (codes, params, None, params)):
        with pytest.raises(TypeError):
            KvCache4(*kinds, **good)
    for shapes in ((codes[..., :32], params, codes[..., :32], params), (codes, params[..., :2, :], codes, params),
                   (codes, params, codes[:2], params[:2]), (codes, params, codes[:, :1], params),
                   (codes[:0], params[:0], codes[:0], params[:0]),
                   (codes.transpose(1, 2), params.transpose(1, 2), codes.transpose(1, 2), params.transpose(1, 2))):
        with pytest.raises(ValueError):
            KvCache4(*shapes, **good)
    for dim in (0, 8, 72, 144, -16, 64.0):
        with pytest.raises(ValueError):
            KvCache4(codes, params, codes, params, head_dim=dim, dtype=BF16)
        with pytest.raises(ValueError):
            KvCache4.empty(1, 1, 1, dim, device="cpu")
    with pytest.raises(TypeError):
        KvCache4(codes, params, codes, params, head_dim=80, dtype=torch.float32)
    k = torch.zeros((1, 2, 80), dtype=BF16)
    slots = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(TypeError, match="CUDA"):
        append_kv4(cache, k, k, slots)
    with pytest.raises(TypeError, match="CUDA"):
        read_kv4(cache, slots)
    with pytest.raises(TypeError, match="KvCache4"):
        append_kv4((codes, params), k, k, slots)


def test_entry_point_refusals():
    """The C entry points refuse on the host, before any launch."""
    import ctypes
    L = _lib.lib()
    some = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(some) + 255) // 256 * 256

    def cache(**other):
        return _lib.Kv4Cache(**{**dict(kv_heads=2, head_dim=64, pages=3, page_size=4, k_codes=p, k_params=p, v_codes=p,
                                       v_params=p), **other})

    def append(c=None, **other):
        return L.ms_kv4_append(_lib.Kv4AppendArgs(**{**dict(dtype=1, tokens=1, k=p, v=p, slots=p, cache=c or cache()),
                                                     **other}), None)

    def read(c=None, **other):
        return L.ms_kv4_read(_lib.Kv4ReadArgs(**{**dict(dtype=1, tokens=1, slots=p, k_out=p, v_out=p,
                                                        cache=c or cache()), **other}), None)

    assert append(tokens=0) == 0 and read(tokens=0) == 0
    assert append(dtype=0) == read(dtype=0) == -2
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(heads=-1), dict(heads=1), dict(rotary=1), dict(rotary=66),
                dict(rotary=64), dict(k=None), dict(v=None), dict(slots=None)):
        assert append(**bad) == -1, bad
    for bad in (dict(tokens=-1), dict(tokens=1 << 31), dict(slots=None), dict(k_out=None), dict(v_out=None)):
        assert read(**bad) == -1, bad
    for bad in (dict(kv_heads=0), dict(pages=0), dict(page_size=0), dict(pages=1 << 31), dict(head_dim=0),
                dict(k_codes=None), dict(v_params=None), dict(pages=0x7FFFFFFF, page_size=0x7FFFFFFF)):
        assert append(cache(**bad)) == read(cache(**bad)) == -1, bad
    for bad in (dict(head_dim=72), dict(head_dim=144), dict(k_codes=p + 8), dict(v_params=p + 4)):
        assert append(cache(**bad)) == read(cache(**bad)) == -4, bad
    assert L.ms_kv4_append(None, None) == L.ms_kv4_read(None, None) == -1


@gpu
def test_call_refusals():
    cache = KvCache4.empty(3, 4, 2, 80)
    k = torch.zeros((5, 2, 80), dtype=BF16, device="cuda")
    q = torch.zeros((5, 6, 80), dtype=BF16, device="cuda")
    slots = torch.zeros(5, dtype=torch.int64, device="cuda")
    rope = rope_table(9, 80)
    for args, kw in (((k.half(), k, slots), {}), ((k, k, slots.int()), {}), ((k, k.float(), slots), {}),
                     ((k, k, slots), dict(q=q.half())), ((k, k, slots), dict(positions=slots, rope=rope.half()))):
        with pytest.raises(TypeError):
            append_kv4(cache, *args, **kw)
    for args, kw in (((k[:, :1], k, slots), {}), ((k, k[..., :64], slots), {}), ((k, k[:4], slots), {}),
                     ((k, k, slots[:4]), {}), ((k, k, slots), dict(rope=rope)),
                     ((k, k, slots), dict(rope=rope, positions=slots[:2])), ((k, k, slots), dict(q_out=q)),
                     ((k, k, slots), dict(q=q, q_out=q[:, :5])), ((k, k, slots), dict(q=q, q_out=q[:, :1].expand(5, 6, 80))),
                     ((k, k, slots.cpu()), {}), ((k, k, slots), dict(rope=rope_table(9, 96), positions=slots)),
                     ((k.transpose(1, 2).contiguous().transpose(1, 2), k, slots), {})):
        with pytest.raises(ValueError):
            append_kv4(cache, *args, **kw)
    for args, kw in (((slots.view(1, 5),), {}), ((slots,), dict(k_out=k[:4])), ((slots,), dict(k_out=k, v_out=k)),
                     ((slots,), dict(v_out=k[:1].expand(5, 2, 80)))):
        with pytest.raises(ValueError):
            read_kv4(cache, *args, **kw)
    with pytest.raises(TypeError):
        read_kv4(cache, slots, k_out=k.half())


@gpu
@pytest.mark.parametrize("dim,kv,page", [(64, 1, 5), (48, 3, 1), (16, 1, 7), (80, 1, 3), (128, 1, 1)])
def test_any_range_of_pages(dim, kv, page):
    """Ranges that start at an odd page of odd size, where a page's parameters
    are 8 bytes off the 16-byte grid: the bytes, what is read back and the
    attention are those of a cache of its own."""
    from miniserve_b200 import attention_kv4
    gen = generator(11)
    T = 6 * page
    k, v = (torch.randn((T, kv, dim), generator=gen, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((2, 3, 2 * kv, dim), generator=gen, device="cuda").bfloat16()
    rope, positions = rope_table(T, 16), torch.arange(T, device="cuda")
    slots = torch.randperm(T, generator=gen, device="cuda")
    pages = torch.tensor([[0, 3, 5], [4, 1, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([[3 * page - 2, 3 * page - 1, 3 * page], [1, 0, 2 * page]], dtype=torch.int32, device="cuda").clamp(min=0)
    want = KvCache4.empty(6, page, kv, dim)
    append_kv4(want, k, v, slots, positions=positions, rope=rope)
    read = read_kv4(want, slots)
    many = q.repeat(1, 6, 1, 1), lengths.repeat(1, 6)  # eighteen tokens a row: the other kernel
    seen = attention_kv4(q, want, pages, lengths), attention_kv4(many[0], want, pages, many[1])
    for first in (1, 2, 3):
        whole = KvCache4.empty(11, page, kv, dim)
        part = whole[first:first + 6]
        append_kv4(part, k, v, slots, positions=positions, rope=rope)
        for a, b in zip(want._args[:4], part._args[:4]):
            assert torch.equal(a, b)
        assert not bool(whole[:first].k_params.any()) and not bool(whole[first + 6:].v_params.any())
        for a, b in zip(read, read_kv4(part, slots)):
            assert torch.equal(a, b)
        for a, b in zip(seen[0], attention_kv4(q, part, pages, lengths)):
            assert torch.equal(a, b)
        for a, b in zip(seen[1], attention_kv4(many[0], part, pages, many[1])):
            assert torch.equal(a, b)


def test_bases_off_their_grid():
    """Codes lie on 16 bytes and parameters on a slot's 8 or 16: what does not is refused as the cache is made, and by
    the entry points."""
    import ctypes
    for dim, row, groups in ((64, 32, 2), (96, 48, 4)):
        codes, params = torch.zeros((3, 1, 5, row), dtype=torch.uint8), torch.zeros((3, 1, 5, groups, 2), dtype=torch.float16)
        cache = KvCache4(codes, params, codes.clone(), params.clone(), head_dim=dim, dtype=BF16)
        assert cache[1:].pages == 2 and cache[1:2].pages == 1
        for name in ("k_codes", "k_params", "v_codes", "v_params"):
            like = getattr(cache, name)
            step = 8 if like.dtype == torch.uint8 else 2
            moved = torch.zeros(like.numel() + step, dtype=like.dtype)[step:].view(like.shape)
            with pytest.raises(ValueError, match=name):
                KvCache4(**{**{n: getattr(cache, n) for n in ("k_codes", "k_params", "v_codes", "v_params")}, name: moved},
                         head_dim=dim, dtype=BF16)
    L = _lib.lib()
    some = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(some) + 255) // 256 * 256

    def call(dim, **other):
        c = _lib.Kv4Cache(**{**dict(kv_heads=1, head_dim=dim, pages=3, page_size=5, k_codes=p, k_params=p, v_codes=p, v_params=p),
                             **other})
        return {L.ms_kv4_append(_lib.Kv4AppendArgs(dtype=1, tokens=0, cache=c), None),
                L.ms_kv4_read(_lib.Kv4ReadArgs(dtype=1, tokens=0, cache=c), None),
                L.ms_kv4_attention(_lib.Kv4AttentionArgs(dtype=1, tokens=1, heads=1, rows=0, scale=1.0, cache=c), None)}

    for name in ("k_params", "v_params"):
        assert call(64, **{name: p + 8}) == {0} and call(96, **{name: p + 8}) == {-4}
        assert call(64, **{name: p + 4}) == {-4}
    for name in ("k_codes", "v_codes"):
        assert call(64, **{name: p + 8}) == {-4}
