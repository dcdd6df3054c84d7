"""append_kv against the rotation's definition in 64 bits.

Tolerance: the kernel computes a c - b s in fp32 (two products and a sum, each
within 2^-24 of its magnitude) and rounds once to the cache's type, so an
entry is within half a unit in the last place (2^-8 of it for bf16's 8
significant bits, 2^-11 for fp16's 11, 2^-25 below fp16's normal range) plus
3 * 2^-24 (|a c| + |b s|).
"""
import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import _lib  # noqa: E402

gpu = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_cache(gen, pages, page, heads, dim, dtype, order):
    shape = (pages, page, heads, dim) if order == "nhd" else (pages, heads, page, dim)
    t = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    return t if order == "nhd" else t.transpose(1, 2)


def turned(x, table, interleaved):
    """(expected, bound) of x [T, H, D] turned by table rows [T, rotary]."""
    x = x.double()
    rotary = table.shape[1]
    half = rotary // 2
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = table[:, None, :half].double(), table[:, None, half:].double()
    y, mag = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    mag[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    mag[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, mag * 3 * 2.0 ** -24


def close(got, want, slack, dtype):
    bound = want.abs() * HALF_ULP[dtype] + slack * (1 + HALF_ULP[dtype]) + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


def expect(cache_k, cache_v, q, k, v, slots, positions, rope, interleaved):
    page = cache_k.shape[1]
    T = k.shape[0]
    table = rope.reshape(rope.shape[0], -1)[positions] if rope is not None else k.new_zeros((T, 0)).float()
    ck, cv = cache_k.double(), cache_v.double()
    slack = torch.zeros_like(ck)
    kk, ks = turned(k, table, interleaved)
    for t in range(T):
        s = int(slots[t])
        if s >= 0:
            ck[s // page, s % page], slack[s // page, s % page] = kk[t], ks[t]
            cv[s // page, s % page] = v[t].double()
    qq = turned(q, table, interleaved) if q is not None else None
    return qq, (ck, slack), cv


CASES = [
    # tokens, heads, kv_heads, dim, rotary, page, interleaved, order
    (1, 14, 2, 64, 64, 16, False, "nhd"),
    (1, 1, 1, 16, 16, 1, True, "hnd"),
    (7, 4, 4, 128, 64, 24, True, "nhd"),
    (33, 6, 2, 80, 40, 16, False, "hnd"),   # rotary not a multiple of 16
    (33, 3, 1, 80, 80, 16, True, "nhd"),
    (50, 5, 5, 33, 10, 7, False, "nhd"),    # odd head size: single entries
    (50, 5, 5, 33, 32, 7, True, "hnd"),
    (129, 8, 8, 256, 256, 64, False, "nhd"),
    (5000, 14, 2, 64, 64, 16, False, "nhd"),  # one head a thread still (LARGE has two)
    (2500, 9, 3, 96, 48, 16, True, "hnd"),
    (64, 0, 2, 64, 64, 16, False, "nhd"),   # keys and values only
    (64, 2, 2, 64, 0, 16, False, "nhd"),    # no rotation
    (0, 2, 2, 64, 64, 16, False, "nhd"),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_append_matches_definition(case, dtype):
    from miniserve_b200.kvcache import append_kv, rope_table
    T, H, Hkv, D, rotary, page, interleaved, order = case
    gen = torch.Generator(device="cuda").manual_seed(T * 131 + D)
    pages = T // page + 3
    ck, cv = (make_cache(gen, pages, page, Hkv, D, dtype, order) for _ in range(2))
    qkv = torch.randn((T, H + 2 * Hkv, D), generator=gen, device="cuda").to(dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T].clone()
    slots[::5] = -1
    rope = rope_table(301, rotary) if rotary else None
    positions = torch.randint(0, 301, (T,), generator=gen, device="cuda") if rotary else None
    qq, (kk, kslack), vv = expect(ck, cv, q if H else None, k, v, slots, positions, rope, interleaved)
    q_out, status = append_kv(ck, cv, k, v, slots, q=q if H else None, positions=positions, rope=rope,
                              interleaved=interleaved)
    assert not status.any()
    if H:
        close(q_out, *qq, dtype)
    else:
        assert q_out is None
    close(ck, kk, kslack, dtype)
    assert torch.equal(cv.double(), vv)


# Above this many entries a thread takes two heads.
TWO_HEADS = 16 * 4 * 148 * 2048
LARGE = [
    # tokens, heads, kv_heads, dim, rotary, page, interleaved, order, a base's offset in entries: 16-byte pieces ...
    (30011, 14, 2, 64, 64, 16, False, "nhd", 0),
    (25000, 13, 3, 64, 64, 16, False, "hnd", 0),   # odd head counts: a thread without a second head
    (25000, 13, 3, 64, 32, 24, True, "nhd", 0),
    (24000, 11, 1, 64, 64, 16, False, "nhd", 0),   # one key head
    (24000, 0, 7, 64, 64, 16, True, "nhd", 0),     # no queries
    (11000, 9, 5, 96, 96, 64, True, "hnd", 0),
    (20000, 13, 3, 80, 40, 16, False, "nhd", 0),   # 8-byte pieces
    (20000, 13, 3, 80, 40, 7, True, "hnd", 0),
    (25000, 13, 3, 64, 64, 16, False, "nhd", 4),
    (30000, 13, 3, 35, 10, 16, False, "nhd", 0),   # single entries
    (30000, 13, 3, 35, 34, 16, True, "hnd", 0),
    (25000, 13, 3, 64, 64, 16, False, "nhd", 1),
]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", LARGE, ids=str)
def test_append_of_prompts_matches_definition(case, dtype):
    """Calls large enough for two heads a thread, in pieces of every size."""
    from miniserve_b200.kvcache import append_kv, rope_table
    T, H, Hkv, D, rotary, page, interleaved, order, offset = case
    assert T * (H + 2 * Hkv) * D > TWO_HEADS
    gen = torch.Generator(device="cuda").manual_seed(T + D)
    pages = T // page + 3
    ck, cv = (make_cache(gen, pages, page, Hkv, D, dtype, order) for _ in range(2))
    flat = torch.randn(offset + T * (H + 2 * Hkv) * D, generator=gen, device="cuda").to(dtype)
    qkv = flat[offset:].view(T, H + 2 * Hkv, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T].clone()
    slots[::5] = -1
    rope = rope_table(301, rotary)
    positions = torch.randint(0, 301, (T,), generator=gen, device="cuda")
    table = rope.reshape(301, -1)[positions]
    kept = torch.nonzero(slots >= 0)[:, 0]
    at = (torch.div(slots[kept], page, rounding_mode="floor"), slots[kept] % page)
    kk, ks = turned(k, table, interleaved)
    want_k, slack = ck.double(), torch.zeros(ck.shape, dtype=torch.float64, device="cuda")
    want_k[at], slack[at] = kk[kept], ks[kept]
    want_v = cv.clone()
    want_v[at] = v[kept]
    q_out, status = append_kv(ck, cv, k, v, slots, q=q if H else None, positions=positions, rope=rope,
                              interleaved=interleaved)
    assert not status.any()
    if H:
        close(q_out, *turned(q, table, interleaved), dtype)
    close(ck, want_k, slack, dtype)
    assert torch.equal(cv, want_v)


@gpu
def test_table_is_the_definition():
    from miniserve_b200.kvcache import rope_table
    t = rope_table(1000, 64, base=1e6, device="cuda")
    p = torch.arange(1000, dtype=torch.float64)[:, None]
    angle = p * 1e6 ** (-2 * torch.arange(32, dtype=torch.float64) / 64)
    # the rounding to fp32 and the argument's own rounding (2^-52 of up to 1000)
    assert (t[:, 0].cpu().double() - angle.cos()).abs().max() <= 2.0 ** -25 + 1e-12
    assert (t[:, 1].cpu().double() - angle.sin()).abs().max() <= 2.0 ** -25 + 1e-12


@gpu
@pytest.mark.parametrize("dim,offset", [(64, 0), (64, 4), (64, 1), (40, 0)])
def test_in_place_and_unaligned(dim, offset):
    """q rotated in place; bases off the 16-byte grid take the 8-byte or the single-entry path."""
    from miniserve_b200.kvcache import append_kv, rope_table
    dtype, T, H = torch.bfloat16, 19, 4
    gen = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(T * 3 * H * dim + offset, generator=gen, device="cuda").to(dtype)
    qkv = flat[offset:].view(T, 3 * H, dim)
    q, k, v = qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:]
    ck, cv = (make_cache(gen, 4, 8, H, dim, dtype, "nhd") for _ in range(2))
    slots = torch.randperm(32, generator=gen, device="cuda")[:T].clone()
    positions = torch.arange(T, device="cuda")
    rope = rope_table(T, dim)
    qq, (kk, kslack), vv = expect(ck, cv, q, k, v, slots, positions, rope, False)
    out, status = append_kv(ck, cv, k, v, slots, q=q, positions=positions, rope=rope, q_out=q)
    assert out is q and not status.any()
    close(q, *qq, dtype)
    close(ck, kk, kslack, dtype)
    assert torch.equal(cv.double(), vv)


@gpu
@pytest.mark.parametrize("T,H", [(1, 4), (3, 1), (1, 1)])
def test_in_place_through_another_view(T, H):
    """q's memory as q_out through a view that differs in the stride of a
    dimension of one entry; views that lie otherwise are refused."""
    from miniserve_b200.kvcache import append_kv, rope_table
    gen = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn((T, H + 2, 64), generator=gen, device="cuda").bfloat16()
    q, k, v = qkv[:, :H], qkv[:, H:H + 1], qkv[:, H + 1:]
    ck, cv = (make_cache(gen, 4, 8, 1, 64, torch.bfloat16, "nhd") for _ in range(2))
    slots = torch.arange(T, device="cuda")
    rope = rope_table(T + 3, 64)
    qq, (kk, kslack), vv = expect(ck, cv, q, k, v, slots, slots + 2, rope, False)
    view = q.as_strided((T, H, 64), (q.stride(0) if T > 1 else 7, q.stride(1) if H > 1 else 9, 1))
    out, status = append_kv(ck, cv, k, v, slots, q=q, positions=slots + 2, rope=rope, q_out=view)
    assert out is view and not status.any()
    close(q, *qq, torch.bfloat16)
    close(ck, kk, kslack, torch.bfloat16)
    if T * H > 1:
        other = q.as_strided((T, H, 64), (64 * H, 64, 1) if T > 1 else (0, 32, 1))
        with pytest.raises(ValueError):
            append_kv(ck, cv, k, v, slots, q=q, positions=slots + 2, rope=rope, q_out=other)


@gpu
@pytest.mark.parametrize("dim", [64, 40])
def test_bad_rows_are_flagged_and_write_nothing(dim):
    from miniserve_b200.kvcache import append_kv, rope_table
    gen = torch.Generator(device="cuda").manual_seed(5)
    ck, cv = (make_cache(gen, 4, 8, 2, dim, torch.float16, "nhd") for _ in range(2))
    k, v, q = (torch.randn((5, 2, dim), generator=gen, device="cuda").half() for _ in range(3))
    before = ck.clone(), cv.clone()
    slots = torch.tensor([32, 1 << 40, 3, -7, 5], device="cuda")
    positions = torch.tensor([0, 1, 10, 2, -1], device="cuda")
    q_out, status = append_kv(ck, cv, k, v, slots, q=q, positions=positions, rope=rope_table(10, dim))
    S, P = _lib.MS_ROW_BAD_SLOT, _lib.MS_ROW_BAD_POSITION
    assert status.tolist() == [S, S, P, 0, P]
    assert torch.equal(ck, before[0]) and torch.equal(cv, before[1])
    assert not q_out[2].any() and not q_out[4].any() and bool(q_out[[0, 1, 3]].any())


@gpu
def test_slots_past_32_bits():
    """A cache view of repeated page strides is refused, so a slot past 2^32
    needs a cache of that many tokens: one head of one entry is 8 GB a half."""
    from miniserve_b200.kvcache import append_kv
    n = (1 << 32) + 64
    free, _ = torch.cuda.mem_get_info()
    if free < 6 * n:
        pytest.skip("needs 25 GB of device memory")
    ck = torch.zeros((n // 64, 64, 1, 1), dtype=torch.bfloat16, device="cuda")
    cv = torch.zeros((n // 64, 64, 1, 1), dtype=torch.bfloat16, device="cuda")
    k = torch.full((2, 1, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    slots = torch.tensor([(1 << 32) + 5, 7], device="cuda")
    _, status = append_kv(ck, cv, k, k, slots)
    assert not status.any()
    flat = ck.view(-1)
    assert float(flat[(1 << 32) + 5]) == 2.0 and float(flat[7]) == 2.0 and float(flat[5]) == 0.0


@gpu
def test_refusals():
    from miniserve_b200.kvcache import append_kv, rope_table
    c = torch.zeros((2, 4, 2, 16), dtype=torch.float16, device="cuda")
    k = torch.zeros((3, 2, 16), dtype=torch.float16, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    rope = rope_table(4, 16)
    ok = dict(cache_k=c, cache_v=c.clone(), k=k, v=k, slots=s)
    append_kv(**ok)
    for err, change in [
        (TypeError, dict(cache_k=c.float())), (TypeError, dict(k=k.bfloat16())), (TypeError, dict(slots=s.int())),
        (TypeError, dict(cache_k=c.cpu())), (ValueError, dict(k=k.cpu())), (ValueError, dict(k=k[:, :1])),
        (ValueError, dict(cache_v=c[:1])), (ValueError, dict(slots=s[:2])), (ValueError, dict(v=k[..., ::2])),
        (ValueError, dict(cache_k=c[:1].expand(2, 4, 2, 16))), (ValueError, dict(rope=rope)),
        (ValueError, dict(rope=rope_table(4, 32), positions=s)), (ValueError, dict(rope=rope, positions=s[:1])),
        (ValueError, dict(q=k[:2])), (ValueError, dict(q_out=k)),
        (ValueError, dict(q=k, q_out=k.view(-1)[:48].view(3, 1, 16).expand(3, 2, 16))),
    ]:
        with pytest.raises(err):
            append_kv(**{**ok, **change})


def test_host_refusals_without_a_gpu():
    from miniserve_b200.kvcache import append_kv, rope_table
    c = torch.zeros((2, 4, 2, 16), dtype=torch.float16)
    with pytest.raises(TypeError):
        append_kv(c, c, c[0], c[0], torch.zeros(4, dtype=torch.int64))
    for bad in ((0, 16), (4, 0), (4, 7)):
        with pytest.raises(ValueError):
            rope_table(*bad, device="cpu")


def test_c_entry_refuses_bad_arguments():
    import ctypes
    L = _lib.lib()
    assert L.ms_kv_append(None, None) == -1
    a = _lib.KvAppendArgs()
    assert L.ms_kv_append(ctypes.byref(a), None) == -2  # fp32
    a.dtype, a.kv_heads, a.head_dim, a.pages, a.page_size = _lib.MS_DTYPE_BF16, 1, 16, 1, 16
    assert L.ms_kv_append(ctypes.byref(a), None) == 0   # no tokens
    a.tokens = 1
    assert L.ms_kv_append(ctypes.byref(a), None) == -1  # null pointers
    a.rotary = 3
    assert L.ms_kv_append(ctypes.byref(a), None) == -1
    a.rotary = 0
    a.pages = 1 << 62
    assert L.ms_kv_append(ctypes.byref(a), None) == -1
