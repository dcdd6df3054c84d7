"""The decode-step operators, case by case: appending rotated keys and values
to a paged cache, attention of a batch over a shared prefix and its rows' own
pages, and the 8-bit integer product that ends in the logits.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits, rounded once at the end) or, with ``own`` set, through the
package's public entry points; ``exact`` computes it from its definition in
64 bits.  Every case is a dict of plain values; ``prepare`` makes its inputs
on the GPU from a seed alone.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of the eight-row sampling batch: a launch's latency
        dict(name="append_decode_8", op="append", dtype="bf16", tokens=8, heads=14, kv_heads=2, dim=64, rotary=64,
             interleaved=False, page=16, pages=512, order="nhd", fused=True, padding=0.0),
        # one decode step of a large batch, pair-wise rotation of half of each head
        dict(name="append_decode_512", op="append", dtype="fp16", tokens=512, heads=32, kv_heads=8, dim=128, rotary=64,
             interleaved=True, page=64, pages=256, order="hnd", fused=False, padding=0.0),
        # prompts of many requests appended in one call, some tokens padding
        dict(name="append_prompts", op="append", dtype="bf16", tokens=30011, heads=14, kv_heads=2, dim=64, rotary=64,
             interleaved=False, page=16, pages=2048, order="nhd", fused=True, padding=0.02),
        # the eight-row batch behind a short instruction
        dict(name="attention_short_8", op="attention", dtype="bf16", rows=8, heads=14, kv_heads=2, dim=64, prefix=512,
             own_min=1, own_max=200, lengths=1, page=16, order="nhd"),
        # chats behind one system prompt whose last page is part full
        dict(name="attention_chat_128", op="attention", dtype="fp16", rows=128, heads=32, kv_heads=8, dim=128,
             prefix=2011, own_min=0, own_max=1024, lengths=2, page=16, order="nhd"),
        # the benchmark's 512 rows behind a long tool and schema description
        dict(name="attention_schema_512", op="attention", dtype="bf16", rows=512, heads=14, kv_heads=2, dim=64,
             prefix=8192, own_min=1, own_max=256, lengths=3, page=16, order="nhd"),
        # nothing shared: ragged histories, some rows just started (empty)
        dict(name="attention_own_64", op="attention", dtype="bf16", rows=64, heads=16, kv_heads=4, dim=128, prefix=0,
             own_min=0, own_max=8192, lengths=4, page=64, order="hnd"),
        # a few questions on one very long document
        dict(name="attention_document_4", op="attention", dtype="bf16", rows=4, heads=32, kv_heads=8, dim=128,
             prefix=131072, own_min=1, own_max=64, lengths=5, page=64, order="hnd"),
        # one row's logits over the benchmark's vocabulary
        dict(name="int8_head_1", op="int8", dtype="bf16", out="fp32", rows=1, inner=896, outer=151936, bias=False),
        # the benchmark's 512 rows of logits
        dict(name="int8_head_512", op="int8", dtype="bf16", out="fp32", rows=512, inner=896, outer=151936, bias=False),
        # sizes that are multiples of nothing
        dict(name="int8_odd_77", op="int8", dtype="fp16", out="fp16", rows=77, inner=1001, outer=32003, bias=True),
        # a prompt's wide projection
        dict(name="int8_prompt_2048", op="int8", dtype="bf16", out="bf16", rows=2048, inner=4096, outer=8192,
             bias=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "int8"])
    half = rng.choice(["bf16", "fp16"])
    if op == "append":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 96, 128])
        tokens = _log_int(rng, 1, 30000)
        page = rng.choice([8, 16, 24, 64])
        return dict(op=op, dtype=half, tokens=tokens, heads=kv * rng.randint(1, 4), kv_heads=kv, dim=dim,
                    rotary=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.5, page=page,
                    pages=(tokens + tokens // 3) // page + 2, order=rng.choice(["nhd", "hnd"]),
                    fused=rng.random() < 0.5, padding=rng.choice([0.0, 0.05]))
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128])
        group = rng.choice([1, 3, 4, 7, 8])
        rows = _log_int(rng, 1, 512)
        prefix = 0 if rng.random() < 0.15 else _log_int(rng, 1, 65536)
        own_max = _log_int(rng, 1, 8192)
        # no more scores than the listed 512 rows have, no more own keys than the listed 64 rows have
        while rows * kv * group * prefix > 512 * 14 * 8192:
            prefix //= 2
        while rows * kv * own_max > 64 * 4 * 8192 or rows * kv * group * own_max > 64 * 16 * 8192:
            own_max //= 2
        return dict(op=op, dtype=half, rows=rows, heads=kv * group, kv_heads=kv, dim=dim, prefix=prefix,
                    own_min=rng.choice([0, 1]), own_max=max(own_max, 1), lengths=rng.randrange(1 << 30),
                    page=rng.choice([8, 16, 24, 64]), order=rng.choice(["nhd", "hnd"]))
    rows = _log_int(rng, 1, 2048)
    inner = _log_int(rng, 256, 8192)
    outer = _log_int(rng, 1000, 151936)
    while rows * inner * outer > 512 * 896 * 151936 or rows * outer > 512 * 151936 or inner * outer > 4096 * 65536:
        outer = outer * 3 // 4
    return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), out=rng.choice(["fp32", "bf16", "fp16"]), rows=rows,
                inner=inner, outer=outer, bias=rng.random() < 0.5)


def _own_lengths(case):
    rng = random.Random(case["lengths"])
    return [rng.randint(case["own_min"], case["own_max"]) for _ in range(case["rows"])]


def _slots(case, seed):
    """Cache slot of every token (-1: padding), distinct where not negative:
    whole pages in a random order, as a block allocator deals them out."""
    rng = np.random.default_rng([seed, 11])
    page, T = case["page"], case["tokens"]
    order = rng.permutation(case["pages"])
    if T <= case["pages"]:  # decode: every row writes into a page of its own
        slots = order[:T] * page + rng.integers(0, page, T)
    else:
        slots = (order[:, None] * page + np.arange(page)[None]).reshape(-1)[:T]
    return np.where(rng.random(T) < case["padding"], -1, slots).astype(np.int64)


# ------------------------------------------------------------------ inputs
def _cache(gen, case, pages, dtype):
    """A [pages, page, kv_heads, dim] view of a cache stored in either order."""
    shape = ((pages, case["page"], case["kv_heads"], case["dim"]) if case["order"] == "nhd" else
             (pages, case["kv_heads"], case["page"], case["dim"]))
    t = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)
    return t if case["order"] == "nhd" else t.transpose(1, 2)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "int8": _prepare_int8}[case["op"]](
        case, seed, gen)


def _rope(rotary, positions=4096, base=1000000.0):
    """[positions, 2, rotary / 2] fp32: cosines, then sines."""
    half = rotary // 2
    inv = base ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) * 2 / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], 1).float()


def _prepare_append(case, seed, gen):
    dt, T, D = DTYPES[case["dtype"]], case["tokens"], case["dim"]
    Hq, Hkv = case["heads"], case["kv_heads"]
    if case["fused"]:  # slices of one projection's output, as a fused QKV product leaves them
        qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=gen, device=DEVICE).to(dt)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        q, k, v = (torch.randn((T, h, D), generator=gen, device=DEVICE).to(dt) for h in (Hq, Hkv, Hkv))
    return dict(case=case, q=q, k=k, v=v, cache_k=_cache(gen, case, case["pages"], dt),
                cache_v=_cache(gen, case, case["pages"], dt), slots=torch.from_numpy(_slots(case, seed)).to(DEVICE),
                positions=torch.randint(0, 4096, (T,), generator=gen, device=DEVICE), rope=_rope(case["rotary"]))


def _prepare_attention(case, seed, gen):
    dt, B, page = DTYPES[case["dtype"]], case["rows"], case["page"]
    lens = _own_lengths(case)
    width = max(1, -(-max(lens) // page))
    n_prefix = -(-case["prefix"] // page)
    used = [-(-n // page) for n in lens]
    total = n_prefix + sum(used)
    order = np.random.default_rng([seed, 12]).permutation(max(total, 1)).astype(np.int32)
    table = np.zeros((B, width), np.int32)
    at = n_prefix
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn((B, case["heads"], case["dim"]), generator=gen, device=DEVICE)
    # queries that prefer some keys, as trained heads do: scores spread over several units
    q = (q * 2.0).to(dt)
    return dict(case=case, q=q, cache_k=_cache(gen, case, max(total, 1), dt), cache_v=_cache(gen, case, max(total, 1), dt),
                pages=torch.from_numpy(table).to(DEVICE),
                lengths=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
                prefix_pages=torch.from_numpy(order[:n_prefix].copy()).to(DEVICE))


def _prepare_int8(case, seed, gen):
    M, K, N = case["rows"], case["inner"], case["outer"]
    x = torch.randn((M, K), generator=gen, device=DEVICE)
    x[:, :: 97] *= 6.0  # a hidden state's few large channels
    wq = (torch.randn((N, K), generator=gen, device=DEVICE) * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    ws = (torch.rand((N,), generator=gen, device=DEVICE) + 0.5) * 5e-4
    bias = torch.randn((N,), generator=gen, device=DEVICE) if case["bias"] else None
    state = dict(case=case, x=x.to(DTYPES[case["dtype"]]), wq=wq, ws=ws, bias=bias)
    if own:
        from miniserve_b200.int8 import Int8Linear
        state["linear"] = Int8Linear(wq, ws, bias=bias)
        del state["wq"]
    return state


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    return {"append": _append, "attention": _attention, "int8": _int8}[case["op"]](case, state)


def _append(case, s):
    if own:
        from miniserve_b200.kvcache import append_kv
        q_out, status = append_kv(s["cache_k"], s["cache_v"], s["k"], s["v"], s["slots"], q=s["q"],
                                  positions=s["positions"], rope=s["rope"], interleaved=case["interleaved"])
        return dict(q=q_out, cache_k=s["cache_k"], cache_v=s["cache_v"], status=status)
    q = _rotate(s["q"].float(), s["rope"][s["positions"]], case).to(s["q"].dtype)
    k = _rotate(s["k"].float(), s["rope"][s["positions"]], case).to(s["k"].dtype)
    live = s["slots"] >= 0
    at = s["slots"][live]
    page, off = at // case["page"], at % case["page"]
    s["cache_k"][page, off] = k[live]
    s["cache_v"][page, off] = s["v"][live]
    status = torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE)
    return dict(q=q, cache_k=s["cache_k"], cache_v=s["cache_v"], status=status)


def _rotate(x, table, case):
    """x [T, H, D] rotated in its first ``rotary`` entries by the tokens'
    rows of the table [T, 2, rotary / 2]."""
    r = case["rotary"]
    cos, sin = table[:, None, 0], table[:, None, 1]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _attention(case, s):
    if own:
        from miniserve_b200.attention import prefix_attention
        out, lse, status = prefix_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["lengths"],
                                            prefix_pages=s["prefix_pages"], prefix_length=case["prefix"])
        return dict(out=out, lse=lse, status=status)
    B, H, Hkv, D, P = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    q = s["q"].float().reshape(B, Hkv, H // Hkv, D) * D ** -0.5

    def keys(cache, table):  # [..., pages] -> [..., keys, Hkv, D]
        return cache[table.long()].float().flatten(-4, -3)

    kp, vp = keys(s["cache_k"], s["prefix_pages"])[:P], keys(s["cache_v"], s["prefix_pages"])[:P]
    ko, vo = keys(s["cache_k"], s["pages"]), keys(s["cache_v"], s["pages"])
    live = torch.arange(ko.shape[1], device=DEVICE) < s["lengths"][:, None]
    vo = vo * live[:, :, None, None]
    prefix = torch.einsum("bhgd,phd->bhgp", q, kp)
    mine = torch.einsum("bhgd,bkhd->bhgk", q, ko).masked_fill_(~live[:, None, None], -math.inf)
    scores = torch.cat([prefix, mine], -1)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = (scores - top).exp()
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bhgp,phd->bhgd", weight[..., :P], vp) + torch.einsum("bhgk,bkhd->bhgd", weight[..., P:], vo)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (total.log() + top).reshape(B, H)
    return dict(out=out.reshape(B, H, D).to(s["q"].dtype), lse=lse,
                status=torch.zeros(B, dtype=torch.int32, device=DEVICE))


def _int8(case, s):
    out_dtype = DTYPES[case["out"]]
    if own:
        return s["linear"](s["x"], out_dtype=out_dtype)
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / torch.full((1, 1), 127.0, device=DEVICE)
    xq = torch.where(scale > 0, (x / scale).round().clamp(-127, 127), 0.0)
    y = (xq @ s["wq"].float().T) * (scale * s["ws"])
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(out_dtype)


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "append":
        T, D, size = case["tokens"], case["dim"], 2
        live = T * (1 - case["padding"])
        moved = 2 * size * D * (T * case["heads"] + live * 2 * case["kv_heads"])
        table = min(T, 4096) * case["rotary"] * 4
        turned = case["rotary"] * (T * case["heads"] + live * case["kv_heads"])
        return dict(bytes=moved + table + T * (8 + 8 + 4), flops=3 * turned)
    if case["op"] == "attention":
        lens = _own_lengths(case)
        B, H, Hkv, D, P = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        keys = P + sum(lens)
        pages = -(-P // case["page"]) + sum(-(-n // case["page"]) for n in lens)
        return dict(bytes=keys * Hkv * D * 2 * 2 + B * H * D * 2 * 2 + B * H * 4 + pages * 4 + B * 8,
                    flops=4 * D * H * (B * P + sum(lens)))
    M, K, N = case["rows"], case["inner"], case["outer"]
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    return dict(bytes=M * K * size[case["dtype"]] + N * K + N * 4 * (2 if case["bias"] else 1)
                + M * N * size[case["out"]], flops=2 * M * N * K)


# ------------------------------------------------------------------- exact
def exact(case, seed):
    global own
    saved, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = saved
    return {"append": _exact_append, "attention": _exact_attention, "int8": _exact_int8}[case["op"]](case, s)


def _exact_append(case, s):
    """Pair (a, b) of a head is the complex number a + ib, turned by
    cos + i sin; the other entries and the values are copied."""
    r, half = case["rotary"], case["rotary"] // 2
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    table = s["rope"].double()[s["positions"]]
    turn = torch.complex(table[:, 0], table[:, 1])[:, None]
    outs = []
    for x in (s["q"], s["k"]):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        outs.append(y)
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    kept = torch.nonzero(s["slots"] >= 0)[:, 0]
    at = s["slots"][kept]
    where = (torch.div(at, case["page"], rounding_mode="floor"), at.remainder(case["page"]))
    ck.index_put_(where, outs[1][kept])
    cv.index_put_(where, s["v"].double()[kept])
    return dict(q=outs[0], cache_k=ck, cache_v=cv,
                status=torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE))


def _exact_attention(case, s):
    """Row by row and head group by head group: softmax over the keys that
    the row sees, the prefix's first, then its own."""
    lens = _own_lengths(case)
    B, H, Hkv, D, page = case["rows"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    G = H // Hkv
    out = torch.zeros((B, H, D), dtype=torch.float64, device=DEVICE)
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=DEVICE)

    def fetch(cache, table, n):  # [Hkv, n, D]
        k = torch.arange(n, device=DEVICE)
        return cache[table.long()[torch.div(k, page, rounding_mode="floor")], k % page].double().transpose(0, 1)

    kp, vp = (fetch(s[c], s["prefix_pages"], case["prefix"]) if case["prefix"] else None
              for c in ("cache_k", "cache_v"))
    for b in range(B):
        parts = []
        if case["prefix"]:
            parts.append((kp, vp))
        if lens[b]:
            parts.append(tuple(fetch(s[c], s["pages"][b], lens[b]) for c in ("cache_k", "cache_v")))
        if not parts:
            continue
        qb = s["q"][b].double().reshape(Hkv, G, D)
        scores = torch.cat([torch.bmm(qb, k.transpose(1, 2)) for k, _ in parts], -1) / math.sqrt(D)
        stat = torch.logsumexp(scores, -1)
        p = (scores - stat[..., None]).exp()
        o, at = 0.0, 0
        for _, v in parts:
            o = o + torch.bmm(p[..., at:at + v.shape[1]], v)
            at += v.shape[1]
        out[b], lse[b] = o.reshape(H, D), stat.reshape(H)
    return dict(out=out, lse=lse, status=torch.zeros(B, dtype=torch.int32, device=DEVICE))


def _exact_int8(case, s):
    """A token's scale is its largest magnitude over 127 and its integers are
    the quotients by that scale, both rounded to 32-bit floats (a quotient of
    two 32-bit floats taken in 64 bits and rounded once is the same), then to
    the nearest integer, ties to even; the rest is in 64 bits."""
    x = s["x"].double()
    scale = (x.abs().max(1).values / 127.0).float().double()[:, None]
    quotient = torch.where(scale > 0, x / torch.where(scale > 0, scale, 1.0), 0.0).float().double()
    xq = quotient.round().clamp(-127, 127)
    parts = []
    for n in range(0, case["outer"], 16384):
        w = s["wq"][n:n + 16384].double()
        y = torch.mm(xq, w.T) * scale * s["ws"][n:n + 16384].double()
        if s["bias"] is not None:
            y = y + s["bias"][n:n + 16384].double()
        parts.append(y)
    return torch.cat(parts, 1)
