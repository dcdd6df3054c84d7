"""The 8-bit integer product against its definition.

The integers and scales are compared exactly.  Tolerance of the product: the
integer sum is exact, then one rounding each of the sum to fp32, the scales'
product, the scaled sum and the bias' sum: within 3 * 2^-24 of the scaled sum
plus 2^-24 of the result (2^-23 in all where there is a bias), and half a unit
in the last place of a 16-bit output (2^-8 of it for bf16, 2^-11 for fp16,
2^-25 below fp16's normal range).
"""
import math

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import _lib  # noqa: E402

gpu = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def quantized(x):
    """(integers, scales) of the definition; a 32-bit quotient is the 64-bit
    quotient rounded once."""
    x = x.double()
    scale = (x.abs().amax(1) / 127.0).float()
    s = scale.double()[:, None]
    q = torch.where(s > 0, (x / torch.where(s > 0, s, 1.0)).float().double().round().clamp(-127, 127), 0.0)
    return q.to(torch.int8), scale


def check_product(out, xq, xs, wq, ws, bias):
    y = (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()
    bound = y.abs() * 4 * 2.0 ** -24
    if bias is not None:
        y = y + bias.double()
    if out.dtype != torch.float32:
        bound = bound + y.abs() * HALF_ULP[out.dtype] + 2.0 ** -25
    bound = bound + y.abs() * 2.0 ** -24
    err = (out.double() - y).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 896), (2, 1001), (33, 4096), (1, 20000), (0, 16)])
def test_quantize_matches_definition(M, K, dtype):
    from miniserve_b200.int8 import quantize_rows
    gen = torch.Generator(device="cuda").manual_seed(M * 31 + K)
    x = (torch.randn((M, K), generator=gen, device="cuda") * 3).to(dtype)
    if M > 2:
        x[1] = 0
        x[2] *= 2.0 ** -12
    q, scale = quantize_rows(x)
    wq, ws = quantized(x)
    assert torch.equal(q, wq) and torch.equal(scale, ws)
    assert q.stride(0) % 16 == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_ties_views_and_extremes(dtype):
    """Ties go to the even integer; a row stride off the 16-byte grid and an
    odd base take the single-entry loads; the smallest and largest magnitudes."""
    from miniserve_b200.int8 import quantize_rows
    info = torch.finfo(dtype)
    row = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 3.0], device="cuda").to(dtype)
    flat = torch.zeros(4 * 11 + 1, dtype=dtype, device="cuda")
    x = flat[1:].view(4, 11)[:, :8]
    x[0], x[1], x[2] = row, info.max, info.tiny
    x[3, 0] = info.smallest_normal * 2.0 ** -6  # below the normal range of every type but bf16 and fp32's inputs
    q, scale = quantize_rows(x)
    wq, ws = quantized(x)
    assert torch.equal(q, wq) and torch.equal(scale, ws)


PRODUCTS = [  # M, N, K
    (1, 1, 1), (1, 128, 128), (2, 129, 127), (15, 100, 129), (16, 256, 896), (17, 1000, 1001), (77, 3203, 1001),
    (128, 640, 2048), (129, 300, 333), (256, 20000, 64), (257, 515, 160), (300, 38000, 96), (700, 129, 4097),
    (5, 151936, 32), (0, 16, 16),
]


@gpu
@pytest.mark.parametrize("M,N,K", PRODUCTS)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_product_matches_definition(M, N, K, out_dtype):
    from miniserve_b200.int8 import Int8Linear
    gen = torch.Generator(device="cuda").manual_seed(M * 7 + N * 3 + K)
    x = torch.randn((M, K), generator=gen, device="cuda").bfloat16()
    wq = torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8)
    ws = torch.rand(N, generator=gen, device="cuda") * 1e-3
    bias = torch.randn(N, generator=gen, device="cuda") if N % 2 else None
    layer = Int8Linear(wq, ws, bias)
    out = layer(x, out_dtype=out_dtype)
    assert out.dtype == out_dtype and out.shape == (M, N)
    check_product(out, *quantized(x), wq, ws, bias)


# M, N, K, out type, and what they are to run on 148 SMs: tokens and channels of a tile, two SMs a tile, stages of the
# ring, rounds of tiles.  All have several steps of K and several rounds of tiles (a ring and an accumulator carried from
# tile to tile), each in another form.
TILINGS = [
    (1, 151936, 896, torch.float32, (16, 115, False, 6, 9)),      # one row of an LM head
    (5, 60000, 1001, torch.float32, (16, 102, False, 6, 4)),
    (37, 21595, 1277, torch.float16, (48, 73, False, 9, 2)),      # a last round one tile short
    (16, 30001, 8192, torch.bfloat16, (16, 102, False, 10, 2)),    # long rows: the whole ring for a few tokens
    (40, 70001, 1300, torch.float32, (32, 128, True, 10, 8)),
    (77, 40003, 1001, torch.float32, (80, 91, False, 8, 3)),
    (100, 64001, 1100, torch.bfloat16, (64, 128, True, 10, 7)),   # the longest ring
    (129, 60001, 640, torch.float32, (144, 128, False, 6, 4)),
    (155, 33765, 2650, torch.float16, (160, 115, False, 5, 2)),
    (231, 48437, 1030, torch.bfloat16, (256, 128, True, 6, 3)),   # a token tile that is part full
    (512, 40000, 896, torch.bfloat16, (256, 128, True, 6, 5)),
    (513, 38001, 897, torch.float32, (192, 128, True, 7, 7)),     # a last token tile of 129, channels and K off the grid
    (785, 8597, 262, torch.float16, (208, 128, False, 4, 2)),     # the shortest ring
    (1401, 2337, 279, torch.float32, (176, 64, False, 5, 2)),
    (2048, 8192, 1000, torch.bfloat16, (256, 128, True, 6, 4)),   # a prompt's projection
]


def test_the_tilings_that_the_shapes_are_to_run(tmp_path):
    """The launch's own rule, compiled for the host."""
    import ctypes
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    source, made = tmp_path / "tiling.cpp", tmp_path / "tiling.so"
    source.write_text('''#include "ms_int8_tiling.h"
        extern "C" void tiling(int64_t M, int64_t N, int64_t K, int size, int *out) {
          const ms::I8Tiling t = ms::i8_tiling(M, N, K, size, 148);
          out[0] = t.bn, out[1] = t.rows, out[2] = t.pair, out[3] = ms::i8_stages(M, K, t.bn, t.pair);
        }''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", csrc, "-o", made, source], check=True)
    rule = ctypes.CDLL(str(made)).tiling
    rule.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.c_void_p]
    forms = set()
    for M, N, K, out_dtype, (bn, rows, pair, stages, rounds) in TILINGS:
        got = (ctypes.c_int * 4)()
        rule(M, N, K, out_dtype.itemsize, got)
        assert tuple(got) == (bn, rows, pair, stages), (M, N, K)
        each = 2 if pair else 1
        tiles = -(-M // bn) * -(-N // (rows * each))
        assert -(-tiles // (148 // each)) == rounds >= 2 and K > 256, (M, N, K)
        forms.add((pair, stages))
    assert {(False, 4), (False, 9), (True, 6), (True, 10)} <= forms


@gpu
@pytest.mark.parametrize("M,N,K,out_dtype", [t[:4] for t in TILINGS], ids=str)
def test_products_of_several_rounds_and_steps(M, N, K, out_dtype):
    from miniserve_b200.int8 import Int8Linear
    gen = torch.Generator(device="cuda").manual_seed(M + N + K)
    x = torch.randn((M, K), generator=gen, device="cuda").bfloat16()
    wq = torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8)
    ws = torch.rand(N, generator=gen, device="cuda") * 1e-3
    bias = torch.randn(N, generator=gen, device="cuda") if N % 2 else None
    room = torch.full((M + 1, N), 7.0, dtype=out_dtype, device="cuda")
    out = Int8Linear(wq, ws, bias)(x, out=room[:M])
    check_product(out, *quantized(x), wq, ws, bias)
    assert bool((room[M] == 7.0).all())


@gpu
def test_extreme_integers_are_exact():
    """Every product 127 * 127 or -127 * 127, or int8's lowest value, up to the
    longest rows: the int32 sum neither saturates nor wraps."""
    from miniserve_b200.int8 import int8_matmul
    K = 131072
    xq = torch.full((3, K), 127, dtype=torch.int8, device="cuda")
    xq[1] = -127
    xq[2, 1::2] = -127
    wq = torch.full((130, K), 127, dtype=torch.int8, device="cuda")
    wq[7] = -128
    one = torch.ones(130, device="cuda")
    out = int8_matmul(xq, one[:3].contiguous(), wq, one)
    want = (xq.double() @ wq.double().T).float()
    assert torch.equal(out, want)


@gpu
def test_scales_zero_nan_and_written_region():
    """Zero rows give the bias, rows with a NaN or an infinity NaN; rows of an
    output view wider than N keep what lies past N."""
    from miniserve_b200.int8 import Int8Linear
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((6, 200), generator=gen, device="cuda")
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 199] = math.inf
    x[4, 0] = -math.inf
    wq = torch.randint(-127, 128, (333, 200), generator=gen, device="cuda").to(torch.int8)
    ws = torch.rand(333, generator=gen, device="cuda")
    bias = torch.randn(333, generator=gen, device="cuda")
    room = torch.full((6, 400), 7.0, device="cuda")
    out = Int8Linear(wq, ws, bias)(x, out=room[:, :333])
    assert out.data_ptr() == room.data_ptr() and bool((room[:, 333:] == 7.0).all())
    assert torch.equal(out[1], bias)
    assert bool(out[2:5].isnan().all())
    keep = [0, 5]
    check_product(out[keep], *quantized(x[keep]), wq, ws, bias)


@gpu
def test_views_streams_and_repeats():
    """Strided inputs, a side stream, and equal results from equal calls."""
    from miniserve_b200.int8 import Int8Linear, int8_matmul, quantize_rows
    gen = torch.Generator(device="cuda").manual_seed(10)
    w = torch.randn((500, 300), generator=gen, device="cuda")
    layer = Int8Linear.from_float(w)
    wide = torch.randn((40, 700), generator=gen, device="cuda").half()
    x = wide[::2, 100:400]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = layer(x)
        second = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, second)
    xq, xs = quantized(x)
    check_product(first, xq, xs, layer.weight, layer.scale, None)
    q, s = quantize_rows(x)
    assert torch.equal(int8_matmul(q, s, layer.weight, layer.scale), first)


@gpu
def test_logits_feed_the_sampler():
    from miniserve_b200 import Sampler
    from miniserve_b200.int8 import Int8Linear
    gen = torch.Generator(device="cuda").manual_seed(11)
    head = Int8Linear.from_float(torch.randn((5003, 128), generator=gen, device="cuda"))
    logits = head(torch.randn((9, 128), generator=gen, device="cuda").bfloat16())
    tokens, _, status = Sampler().sample_batch(logits, temperature=0.0, uniforms=[0.5] * 9)
    assert not status.any() and torch.equal(tokens, logits.argmax(1))


@gpu
def test_refusals():
    from miniserve_b200.int8 import Int8Linear, int8_matmul, quantize_rows
    x = torch.zeros((4, 32), device="cuda")
    q, s = quantize_rows(x)
    w, ws = quantize_rows(torch.ones((6, 32), device="cuda"))
    layer = Int8Linear(w, ws)
    for err, call in [
        (TypeError, lambda: quantize_rows(x.cpu())), (TypeError, lambda: quantize_rows(x.double())),
        (ValueError, lambda: quantize_rows(x[0])), (ValueError, lambda: quantize_rows(x.T)),
        (ValueError, lambda: quantize_rows(x[:1].expand(4, 32))),
        (ValueError, lambda: quantize_rows(torch.zeros((1, 131073), device="cuda"))),
        (TypeError, lambda: int8_matmul(x, s, w, ws)), (ValueError, lambda: int8_matmul(q, s[:2], w, ws)),
        (ValueError, lambda: int8_matmul(q[:, :16], s, w, ws)), (TypeError, lambda: int8_matmul(q, s.double(), w, ws)),
        (ValueError, lambda: int8_matmul(q[:, 1:], s, w[:, 1:], ws)),
        (ValueError, lambda: int8_matmul(torch.zeros((4, 33), dtype=torch.int8, device="cuda")[:, :32], s, w, ws)),
        (TypeError, lambda: int8_matmul(q, s, w, ws, out_dtype=torch.int32)),
        (ValueError, lambda: int8_matmul(q, s, w, ws, out=torch.zeros((4, 5), device="cuda"))),
        (ValueError, lambda: int8_matmul(q, s, w, ws, bias=ws[:5])),
        (ValueError, lambda: layer(x[:, :31])), (TypeError, lambda: layer(x.double())),
        (TypeError, lambda: layer(x, out=torch.zeros((4, 6), device="cuda"), out_dtype=torch.float16)),
        (ValueError, lambda: layer(x, out=torch.zeros((1, 6), device="cuda").expand(4, 6))),
        (TypeError, lambda: Int8Linear(x, s)),
    ]:
        with pytest.raises(err):
            call()


def test_c_entries_refuse_bad_arguments():
    L = _lib.lib()
    F32 = _lib.MS_DTYPE_F32
    assert L.ms_quantize_rows(None, 9, 1, 1, 1, None, 16, None, None) == -2
    assert L.ms_quantize_rows(None, F32, 1, 1, 1, None, 16, None, None) == -1
    assert L.ms_quantize_rows(None, F32, 1, 200000, 200000, None, 200000, None, None) == -4
    assert L.ms_quantize_rows(None, F32, 0, 1, 1, None, 16, None, None) == 0
    assert L.ms_int8_matmul(None, 16, None, 1, None, 16, None, 1, 1, None, None, F32, 1, None) == -1
    assert L.ms_int8_matmul(16, 16, 16, 1, 16, 15, 16, 1, 1, None, 16, F32, 1, None) == -1   # row stride
    assert L.ms_int8_matmul(8, 16, 16, 1, 16, 16, 16, 1, 1, None, 16, F32, 1, None) == -1    # base
    assert L.ms_int8_matmul(16, 16, 16, 1, 16, 16, 16, 2, 1, None, 16, F32, 1, None) == -1   # ldo
    assert L.ms_int8_matmul(16, 16, 16, 1, 16, 16, 16, 1, 1, None, 16, 7, 1, None) == -2
    assert L.ms_int8_linear(16, F32, 1, 1, 16, 16, 16, 1, 1, None, 16, F32, 1, None, None) == -1
    assert L.ms_int8_workspace(3, 33) == 16 + 3 * 48 and L.ms_int8_workspace(-1, 4) == 0
