"""The merge of attention's partial records against the definition, and what it
reports for records that stand for no result: a page outside the cache, and a
wait that ran out.  The kernel is the library's, compiled here into a small
library that takes records from the test."""
import ctypes
import math
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from miniserve_b200 import _lib, build  # noqa: E402

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def merge(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("merge") / "attn_merge.so")
    done = subprocess.run([build.nvcc(), *build.ARCH, "-O1", "-std=c++17", "-Xcompiler", "-fPIC", "-shared", "-o", path,
                           os.path.join(HERE, "attn_merge.cu")], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    L = ctypes.CDLL(path)
    L.record_bad_page.restype = L.record_late.restype = ctypes.c_float
    L.merge_records.argtypes = [ctypes.c_int] * 5 + [ctypes.c_void_p] * 9
    return L


@pytest.mark.parametrize("wide", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,splits", [(4, 2, 1), (14, 2, 3), (8, 1, 70)])
def test_flags_of_records(merge, heads, kv_heads, splits, wide):
    """Rows: fine, a late record, a bad page, both, empty, a late one in the
    last head alone, fine.  A record (m, l, O) stands for O / l with weight 2^m l; the
    merge's fp32 sums over the records and bf16's rounding bound the rest."""
    B, G = 7, heads // kv_heads
    gen = torch.Generator(device="cuda").manual_seed(splits)
    o = torch.randn((splits, kv_heads, B * G, 64), generator=gen, device="cuda")
    ml = torch.rand((splits, kv_heads, B * G, 2), generator=gen, device="cuda") * 9 + 0.5
    late, bad = merge.record_late(), merge.record_bad_page()
    rows = ml.view(splits, kv_heads, B, G, 2)
    rows[0, :, 1, :] = torch.tensor([0.0, late], device="cuda")
    rows[-1, :, 2, :, 1] = bad
    rows[0, :, 3, :, 1] = bad
    rows[-1, :, 3, :] = torch.tensor([0.0, late], device="cuda")
    if splits == 1:
        rows[0, 0, 3, 0, 1] = bad
    rows[:, :, 4, :] = torch.tensor([-math.inf, 0.0], device="cuda")
    rows[splits // 2, -1, 5, -1] = torch.tensor([0.0, late], device="cuda")
    o.view(splits, kv_heads, B, G, 64)[0, :, 1] = math.nan  # what a late record's entries hold is anything
    o.view(splits, kv_heads, B, G, 64)[:, :, 4] = 0.0
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    base = torch.zeros(B, dtype=torch.int64, device="cuda")
    header = torch.full((4,), 3, dtype=torch.int64, device="cuda")
    out = torch.full((B, heads, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, heads), 7.0, device="cuda")
    status = torch.zeros(B, dtype=torch.int32, device="cuda")  # the lengths' part of it: all good
    rc = merge.merge_records(wide, B, heads, kv_heads, splits, *(t.data_ptr() for t in (
        o, ml, lengths, base, header, out, lse, status)), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    W, P = _lib.MS_ROW_WAIT_TIMEOUT, _lib.MS_ROW_BAD_PAGE
    assert status.tolist() == [0, W, P, W | P, 0, W, 0]
    assert not out[1:5].any() and bool((lse[1:5] == -math.inf).all())
    assert not out[5, -1].any() and float(lse[5, -1]) == -math.inf
    weight = ml[..., 0].double().exp2()
    total = (weight * ml[..., 1].double()).sum(0)                         # [kv_heads, B * G]
    want = (weight[..., None] * o.double()).sum(0) / total[..., None]
    room = (weight[..., None] * o.double().abs()).sum(0) / total[..., None]
    want, room = (t.view(kv_heads, B, G, 64).transpose(0, 1).reshape(B, heads, 64) for t in (want, room))
    exact_lse = (total.log2() * math.log(2)).view(kv_heads, B, G).transpose(0, 1).reshape(B, heads)
    for b, h in ((0, heads), (5, heads - 1), (6, heads)):
        bound = want[b].abs() * 2.0 ** -8 + room[b] * (splits + 16) * 2.0 ** -22 + 2.0 ** -25
        assert bool(((out[b].double() - want[b]).abs() <= bound)[:h].all())
        assert bool(((lse[b].double() - exact_lse[b]).abs()[:h] <= (splits + 16) * 2.0 ** -22 + 2.0 ** -20).all())
