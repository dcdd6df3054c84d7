"""A drafted-token decode step over a 4-bit cache, case by case: keys and values
quantised as they are written and read back, attention of one or several
tokens a row over the 4-bit cache, and the verification of drafted tokens.

``run`` computes each operator in its plain form (elementary torch operations
in 32 bits, verification in 64, rounded once at the end) or, with ``own`` set,
through the package's public entry points; ``exact`` computes it from its
definition in 64 bits.  Every case is a dict of plain values; ``prepare`` makes
its inputs on the GPU from a seed alone.

A cache is four tensors: ``codes`` uint8 [pages, kv_heads, page_size, padded /
2], byte j holding entries 2j (low four bits) and 2j + 1, and ``params`` fp16
[pages, kv_heads, page_size, groups, 2], the scale and the middle of every 32
entries, of the keys and of the values each.  Entry i stands for ``middle +
scale * (code - 8)``.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
GROUP = 32


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of the eight-row sampling batch: a launch's latency
        dict(name="store_decode_8", op="store", dtype="bf16", tokens=8, heads=14, kv_heads=2, dim=64, rotary=64,
             interleaved=False, page=16, pages=512, fused=True, padding=0.0),
        # prompts of odd sizes: heads of 80, half of them rotated pair-wise, pages of 24
        dict(name="store_odd_777", op="store", dtype="fp16", tokens=777, heads=15, kv_heads=5, dim=80, rotary=40,
             interleaved=True, page=24, pages=64, fused=False, padding=0.05),
        # prompts of many requests quantised in one call and handed on to a prompt's attention
        dict(name="store_prompts", op="store", dtype="bf16", tokens=20011, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, page=64, pages=320, fused=True, padding=0.02),
        # a matched prefix of a short request, read back
        dict(name="read_prefix_500", op="read", dtype="bf16", tokens=500, kv_heads=2, dim=64, page=16, pages=64,
             padding=0.0),
        # long histories read back for a model that attends in 16 bits
        dict(name="read_history", op="read", dtype="fp16", tokens=65536, kv_heads=8, dim=128, page=64, pages=1100,
             padding=0.01),
        # the eight-row batch with short histories
        dict(name="attention_short_8", op="attention", dtype="bf16", rows=8, tokens=1, heads=14, kv_heads=2, dim=64,
             min_keys=1, max_keys=700, lengths=1, page=16),
        # ragged histories, some rows just started (empty)
        dict(name="attention_own_64", op="attention", dtype="fp16", rows=64, tokens=1, heads=16, kv_heads=4, dim=128,
             min_keys=0, max_keys=8192, lengths=2, page=64),
        # two questions on very long documents
        dict(name="attention_long_2", op="attention", dtype="bf16", rows=2, tokens=1, heads=32, kv_heads=8, dim=128,
             min_keys=120000, max_keys=131072, lengths=3, page=64),
        # four drafted tokens and the last accepted one of many chats
        dict(name="attention_drafted_128", op="attention", dtype="bf16", rows=128, tokens=5, heads=14, kv_heads=2,
             dim=64, min_keys=1, max_keys=4096, lengths=4, page=16),
        # one request's drafts: latency over the benchmark's vocabulary
        dict(name="verify_one", op="verify", dtype="fp32", rows=1, drafts=4, vocab=151936, probs=True, sharp=2.5,
             counts=5, greedy=0.0),
        # a batch's drafts of a draft model
        dict(name="verify_64", op="verify", dtype="fp32", rows=64, drafts=4, vocab=151936, probs=True, sharp=2.5,
             counts=6, greedy=0.2),
        # drafts looked up in the prompt, an odd vocabulary
        dict(name="verify_lookup_200", op="verify", dtype="bf16", rows=200, drafts=3, vocab=32003, probs=False,
             sharp=5.0, counts=7, greedy=0.3),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attention", "attention", "verify"])
    half = rng.choice(["bf16", "fp16"])
    kv = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([48, 64, 80, 96, 112, 128])
    page = rng.choice([8, 16, 24, 64])
    if op == "store":
        tokens = _log_int(rng, 1, 20000)
        return dict(op=op, dtype=half, tokens=tokens, heads=kv * rng.randint(1, 4), kv_heads=kv, dim=dim,
                    rotary=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.5, page=page,
                    pages=(tokens + tokens // 3) // page + 2, fused=rng.random() < 0.5,
                    padding=rng.choice([0.0, 0.05]))
    if op == "read":
        tokens = _log_int(rng, 1, 65536)
        return dict(op=op, dtype=half, tokens=tokens, kv_heads=kv, dim=dim, page=page,
                    pages=tokens // page + rng.randint(2, 50), padding=rng.choice([0.0, 0.05]))
    if op == "attention":
        group = rng.choice([1, 3, 4, 7, 8])
        rows, tokens = _log_int(rng, 1, 256), rng.choice([1, 1, 2, 3, 4, 6, 8])
        keys = _log_int(rng, 1, 131072)
        # no more keys and scores than the listed cases have
        while rows * kv * keys > 2 * 8 * 131072 or rows * tokens * kv * group * keys > 128 * 5 * 14 * 4096:
            keys = keys * 2 // 3
        return dict(op=op, dtype=half, rows=rows, tokens=tokens, heads=kv * group, kv_heads=kv, dim=dim,
                    min_keys=rng.choice([0, 1, max(keys, 1) // 2]), max_keys=max(keys, 1),
                    lengths=rng.randrange(1 << 30), page=page)
    rows, drafts, vocab = _log_int(rng, 1, 256), rng.randint(1, 8), _log_int(rng, 1000, 151936)
    while rows * (drafts + 1) * vocab > 64 * 5 * 151936:
        rows = rows * 2 // 3
    return dict(op=op, dtype=rng.choice(["fp32", "bf16"]), rows=rows, drafts=drafts, vocab=vocab,
                probs=rng.random() < 0.6, sharp=rng.choice([2.5, 5.0]), counts=rng.randrange(1 << 30),
                greedy=rng.choice([0.0, 0.25]))


def _row_keys(case):
    """Keys of every row, its newest token's among them."""
    rng = random.Random(case["lengths"])
    return [rng.randint(case["min_keys"], case["max_keys"]) for _ in range(case["rows"])]


def _row_drafts(case):
    """Drafts of every row: most have all, some fewer or none."""
    rng = random.Random(case["counts"])
    return [case["drafts"] if rng.random() < 0.7 else rng.randint(0, case["drafts"]) for _ in range(case["rows"])]


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


# -------------------------------------------------------------- the format
def _padded(dim):
    return max(64, -(-dim // GROUP) * GROUP)


def _groups(dim):
    n = _padded(dim) // GROUP
    return 4 if n == 3 else n


def _in_groups(x):
    """x [..., dim] as [..., groups, 32], the last group filled up by repeating
    its first entry (which moves no minimum or maximum)."""
    dim = x.shape[-1]
    at = torch.arange(-(-dim // GROUP) * GROUP, device=x.device)
    at = torch.where(at < dim, at, (dim - 1) // GROUP * GROUP)
    return x[..., at].unflatten(-1, (-1, GROUP))


def _quantised(y):
    """(codes uint8 [..., padded / 2], params fp16 [..., groups, 2]) of y [..., dim] fp32."""
    dim, lead = y.shape[-1], y.shape[:-1]
    g = _in_groups(y)
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) * (1.0 / 15.0)).half().float()
    middle = (lo + 8.0 * scale).half().float()
    fine = scale.isfinite() & middle.isfinite()
    scale, middle = torch.where(fine, scale, 0.0), torch.where(fine, middle, math.nan)
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    code = ((g - middle[..., None]) * inverse[..., None]).nan_to_num(0.0).round() + 8.0
    code = code.clamp(0, 15).to(torch.uint8).flatten(-2)
    whole = torch.zeros((*lead, _padded(dim)), dtype=torch.uint8, device=y.device)
    whole[..., :dim] = code[..., :dim]
    params = torch.zeros((*lead, _groups(dim), 2), dtype=torch.float16, device=y.device)
    params[..., :scale.shape[-1], 0] = scale.half()
    params[..., :scale.shape[-1], 1] = middle.half()
    return whole[..., 0::2] | (whole[..., 1::2] << 4), params


def _values(codes, params, dim):
    """What codes [..., padded / 2] and params [..., groups, 2] stand for: [..., dim] fp32."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :dim].float()
    group = torch.arange(dim, device=codes.device) // GROUP
    return params[..., 1].float()[..., group] + params[..., 0].float()[..., group] * (code - 8.0)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"store": _prepare_store, "read": _prepare_read, "attention": _prepare_attention,
            "verify": _prepare_verify}[case["op"]](case, seed, gen)


def _cache(gen, case, pages):
    """The four tensors of a cache of normal entries, some of the keys' channels
    larger than the others, and what a program holds of them."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    keys = torch.randn(shape, generator=gen, device=DEVICE)
    keys[..., ::37] *= 4.0
    k = _quantised(keys)
    v = _quantised(torch.randn(shape, generator=gen, device=DEVICE, out=keys))
    state = dict(k=k, v=v)
    if own:
        from miniserve_b200.kvcache4 import KvCache4
        state["cache"] = KvCache4(*k, *v, head_dim=case["dim"], dtype=DTYPES[case["dtype"]])
    return state


def _rope(rotary, positions=4096, base=1000000.0):
    """[positions, 2, rotary / 2] fp32: cosines, then sines."""
    half = rotary // 2
    inv = base ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) * 2 / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], 1).float()


def _prepare_store(case, seed, gen):
    dt, T, D = DTYPES[case["dtype"]], case["tokens"], case["dim"]
    Hq, Hkv = case["heads"], case["kv_heads"]
    if case["fused"]:  # slices of one projection's output, as a fused QKV product leaves them
        qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=gen, device=DEVICE).to(dt)
        q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    else:
        q, k, v = (torch.randn((T, h, D), generator=gen, device=DEVICE).to(dt) for h in (Hq, Hkv, Hkv))
    return dict(case=case, q=q, new_k=k, new_v=v, slots=torch.from_numpy(_slots(case, seed)).to(DEVICE),
                positions=torch.randint(0, 4096, (T,), generator=gen, device=DEVICE), rope=_rope(case["rotary"]),
                **_cache(gen, case, case["pages"]))


def _prepare_read(case, seed, gen):
    return dict(case=case, slots=torch.from_numpy(_slots(case, seed)).to(DEVICE), **_cache(gen, case, case["pages"]))


def _prepare_attention(case, seed, gen):
    B, T, page = case["rows"], case["tokens"], case["page"]
    keys = _row_keys(case)
    used = [-(-n // page) for n in keys]
    order = np.random.default_rng([seed, 12]).permutation(max(sum(used), 1)).astype(np.int32)
    table = np.zeros((B, max(1, max(used))), np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    # a row's tokens see the keys before them and their own, the last one all of them
    lengths = np.maximum(np.array(keys)[:, None] - np.arange(T - 1, -1, -1)[None], 0).astype(np.int32)
    # queries that prefer some keys, as trained heads do: scores spread over several units
    q = (torch.randn((B, T, case["heads"], case["dim"]), generator=gen, device=DEVICE) * 2.0).to(DTYPES[case["dtype"]])
    lengths = torch.from_numpy(lengths).to(DEVICE)
    return dict(case=case, q=q if T > 1 else q[:, 0], lengths=lengths if T > 1 else lengths[:, 0].contiguous(),
                pages=torch.from_numpy(table).to(DEVICE), **_cache(gen, case, max(sum(used), 1)))


def _prepare_verify(case, seed, gen):
    B, n, V = case["rows"], case["drafts"], case["vocab"]
    logits = torch.randn((B, n + 1, V), generator=gen, device=DEVICE) * case["sharp"]
    temperature = 0.6 + 0.4 * torch.rand((B,), generator=gen, device=DEVICE, dtype=torch.float64)
    temperature[torch.rand((B,), generator=gen, device=DEVICE) < case["greedy"]] = 0.0
    heat = torch.where(temperature > 0, temperature, 0.7).float()[:, None, None]
    # a draft model's probabilities: the target's logits, somewhat off; looked-up drafts follow the target's
    near = logits[:, :n] + (0.7 if case["probs"] else 0.0) * torch.randn((B, n, V), generator=gen, device=DEVICE)
    probs = torch.softmax(near / heat, -1)
    race = torch.empty_like(probs).exponential_(generator=gen)
    drafts = (probs / race).argmax(-1)
    count = torch.tensor(_row_drafts(case), device=DEVICE)
    drafts = torch.where(torch.arange(n, device=DEVICE) < count[:, None], drafts, -1)
    return dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), drafts=drafts,
                draft_probs=probs if case["probs"] else None, temperature=temperature,
                uniforms=torch.rand((B, n + 1), generator=gen, device=DEVICE, dtype=torch.float64))


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    return {"store": _store, "read": _read, "attention": _attention, "verify": _verify}[case["op"]](case, state)


def _store(case, s):
    """New tokens into the cache, and what the cache then stands for in their slots."""
    if own:
        from miniserve_b200.kvcache4 import append_kv4, read_kv4
        q_out, status = append_kv4(s["cache"], s["new_k"], s["new_v"], s["slots"], q=s["q"], positions=s["positions"],
                                   rope=s["rope"], interleaved=case["interleaved"])
        k, v, read = read_kv4(s["cache"], s["slots"])
        return dict(q=q_out, k=k, v=v, status=status, read=read)
    table = s["rope"][s["positions"]]
    live = s["slots"] >= 0
    at = s["slots"][live]
    page, off = at // case["page"], at % case["page"]
    s["k"][0][page, :, off], s["k"][1][page, :, off] = _quantised(_rotate(s["new_k"].float(), table, case)[live])
    s["v"][0][page, :, off], s["v"][1][page, :, off] = _quantised(s["new_v"].float()[live])
    out = _read(case, s)
    return dict(q=_rotate(s["q"].float(), table, case).to(s["q"].dtype), k=out["k"], v=out["v"],
                status=torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE), read=out["status"])


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


def _read(case, s):
    if own:
        from miniserve_b200.kvcache4 import read_kv4
        k, v, status = read_kv4(s["cache"], s["slots"])
        return dict(k=k, v=v, status=status)
    live = s["slots"] >= 0
    at = torch.where(live, s["slots"], 0)
    page, off = at // case["page"], at % case["page"]

    def back(codes, params):
        y = _values(codes[page, :, off], params[page, :, off], case["dim"])
        return torch.where(live[:, None, None], y, 0.0).to(DTYPES[case["dtype"]])

    return dict(k=back(*s["k"]), v=back(*s["v"]), status=torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE))


def _attention(case, s):
    if own:
        from miniserve_b200.attention4 import attention_kv4
        out, lse, status = attention_kv4(s["q"], s["cache"], s["pages"], s["lengths"])
        return dict(out=out, lse=lse, status=status)
    B, T, H, Hkv, D = case["rows"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    q = s["q"].float().reshape(B, T, Hkv, H // Hkv, D) * D ** -0.5
    table = s["pages"].long()

    def entries(codes, params):  # [B, Hkv, keys, D]
        return _values(codes[table], params[table], D).transpose(1, 2).flatten(2, 3)

    scores = torch.einsum("bthgd,bhkd->bthgk", q, entries(*s["k"]))
    seen = torch.arange(scores.shape[-1], device=DEVICE) < s["lengths"].view(B, T, 1)
    scores = scores.masked_fill_(~seen[:, :, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = (scores - top).exp()
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bthgk,bhkd->bthgd", weight, entries(*s["v"]))
    out = torch.where(total > 0, out / total, 0.0).reshape(B, T, H, D).to(s["q"].dtype)
    lse = (total.log() + top).reshape(B, T, H)
    return dict(out=out if T > 1 else out[:, 0], lse=lse if T > 1 else lse[:, 0],
                status=torch.zeros(B, dtype=torch.int32, device=DEVICE))


def _verify(case, s):
    if own:
        from miniserve_b200.verify import verify_drafts
        tokens, probs, counts, status = verify_drafts(s["logits"], s["drafts"], s["uniforms"],
                                                      draft_probs=s["draft_probs"], temperature=s["temperature"])
        return dict(tokens=tokens, probs=probs, counts=counts, status=status)
    B, n, V = case["rows"], case["drafts"], case["vocab"]
    x = s["logits"].double()
    heat = s["temperature"][:, None, None]
    top = x.amax(-1, keepdim=True)
    p = ((x - top) / torch.where(heat > 0, heat, 1.0)).exp()
    p = p / p.sum(-1, keepdim=True)
    vocab = torch.arange(V, device=DEVICE)
    p = torch.where(heat > 0, p, (vocab == x.argmax(-1, keepdim=True)).double())  # greedy: the first maximum alone
    drafted = s["drafts"] >= 0
    d = torch.where(drafted, s["drafts"], 0)
    p_d = p[:, :n].gather(2, d[..., None])[..., 0]
    q_d = s["draft_probs"].gather(2, d[..., None])[..., 0].double() if s["draft_probs"] is not None else 1.0
    kept = (drafted & (s["uniforms"][:, :n] * q_d < p_d)).long().cumprod(1)
    count = kept.sum(1)
    rows = torch.arange(B, device=DEVICE)
    last = p[rows, count]
    at = count.clamp(max=n - 1)
    refused = (count < n) & drafted[rows, at]
    if s["draft_probs"] is not None:
        rest = (last - s["draft_probs"][rows, at].double()).clamp(min=0.0)
    else:
        rest = torch.where(vocab == d[rows, at][:, None], 0.0, last)
    weight = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, last)
    mass = weight.cumsum(1)
    final = (mass <= s["uniforms"][:, n:] * mass[:, -1:]).sum(1)
    final = torch.minimum(final, torch.where(weight > 0, vocab, 0).amax(1))
    place = torch.arange(n + 1, device=DEVICE)
    padded = torch.cat([d, torch.zeros_like(d[:, :1])], 1)
    tokens = torch.where(place < count[:, None], padded, -1)
    tokens[rows, count] = final
    probs = p.gather(2, tokens.clamp(min=0)[..., None])[..., 0]
    return dict(tokens=tokens, probs=torch.where(tokens >= 0, probs, 0.0).float(), counts=(count + 1).int(),
                status=torch.zeros(B, dtype=torch.int32, device=DEVICE))


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "verify":
        size = {"fp32": 4, "bf16": 2}[case["dtype"]]
        counts, V = _row_drafts(case), case["vocab"]
        rows = sum(n + 1 for n in counts)
        read = rows * V * size + (sum(1 for n in counts if n) * V * 4 if case["probs"] else 0)
        return dict(bytes=read + case["rows"] * ((case["drafts"] + 1) * 28 + 16), flops=4 * rows * V)
    D, Hkv = case["dim"], case["kv_heads"]
    entry = D / 2 + -(-D // GROUP) * 4  # of one token and head of the keys or the values
    if case["op"] == "attention":
        B, T, H = case["rows"], case["tokens"], case["heads"]
        keys = _row_keys(case)
        pages = sum(-(-n // case["page"]) for n in keys)
        scores = sum(max(0, n - t) for n in keys for t in range(T))
        return dict(bytes=sum(keys) * Hkv * entry * 2 + B * T * H * (D * 4 + 4) + pages * 4 + B * T * 4 + B * 4,
                    flops=4 * D * H * scores)
    T = case["tokens"]
    live = T * (1 - case["padding"])
    read = live * 2 * Hkv * entry + T * 2 * Hkv * D * 2 + T * (8 + 4)
    if case["op"] == "read":
        return dict(bytes=read, flops=2 * live * 2 * Hkv * D)
    written = T * case["heads"] * D * 4 + live * 2 * Hkv * (D * 2 + entry)
    table = min(T, 4096) * case["rotary"] * 4
    return dict(bytes=read + written + table + T * (8 + 8 + 4),
                flops=3 * case["rotary"] * (T * case["heads"] + live * Hkv) + 8 * live * 2 * Hkv * D)


# ------------------------------------------------------------------- exact
def exact(case, seed):
    global own
    saved, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = saved
    return {"store": _exact_store, "read": _exact_read, "attention": _exact_attention,
            "verify": _exact_verify}[case["op"]](case, s)


def _decoded(codes, params, dim):
    """Entry i of a head is four bits of byte i // 2; its group's scale and
    middle are numbers 2 (i // 32) and the next."""
    i = torch.arange(dim, device=DEVICE)
    nibble = torch.bitwise_right_shift(codes[..., torch.div(i, 2, rounding_mode="floor")].to(torch.int32), 4 * (i % 2))
    flat = params.flatten(-2).double()
    at = 2 * torch.div(i, GROUP, rounding_mode="floor")
    return flat[..., at + 1] + flat[..., at] * ((nibble & 15).double() - 8)


def _exact_read(case, s):
    out = {}
    for name in ("k", "v"):
        y = torch.zeros((case["tokens"], case["kv_heads"], case["dim"]), dtype=torch.float64, device=DEVICE)
        kept = torch.nonzero(s["slots"] >= 0)[:, 0]
        at = s["slots"][kept]
        page, off = torch.div(at, case["page"], rounding_mode="floor"), at.remainder(case["page"])
        y[kept] = _decoded(s[name][0][page, :, off], s[name][1][page, :, off], case["dim"])
        out[name] = y
    return dict(k=out["k"], v=out["v"], status=torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE))


def _exact_store(case, s):
    """Pair (a, b) of a head is the complex number a + ib, turned by cos + i
    sin.  A group's scale and middle are rounded to fp16 (they are what the
    cache holds); everything else is in 64 bits."""
    r, half, D = case["rotary"], case["rotary"] // 2, case["dim"]
    i = torch.arange(half, device=DEVICE)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    table = s["rope"].double()[s["positions"]]
    turn = torch.complex(table[:, 0], table[:, 1])[:, None]
    turned = []
    for x in (s["q"], s["new_k"]):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        turned.append(y)
    live = (s["slots"] >= 0)[:, None, None]
    held = []
    for y in (turned[1], s["new_v"].double()):
        z = torch.zeros_like(y)
        for g in range(0, D, GROUP):
            part = y[..., g:g + GROUP]
            low = part.min(-1, keepdim=True).values
            step = ((part.max(-1, keepdim=True).values - low) / 15).half().double()
            mid = (low + 8 * step).half().double()
            count = torch.where(step > 0, (part - mid) / torch.where(step > 0, step, 1.0), 0.0).round().clamp(-8, 7)
            z[..., g:g + GROUP] = mid + step * count
        held.append(torch.where(live, z, 0.0))
    zero = torch.zeros(case["tokens"], dtype=torch.int32, device=DEVICE)
    return dict(q=turned[0], k=held[0], v=held[1], status=zero, read=zero)


def _exact_attention(case, s):
    """Row by row and token by token: softmax over the keys that the token sees."""
    B, T, H, Hkv, D, page = (case[k] for k in ("rows", "tokens", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros((B, T, H, D), dtype=torch.float64, device=DEVICE)
    lse = torch.full((B, T, H), -math.inf, dtype=torch.float64, device=DEVICE)
    q = s["q"].double().reshape(B, T, Hkv, H // Hkv, D)
    for b, n in enumerate(_row_keys(case)):
        if n == 0:
            continue
        j = torch.arange(n, device=DEVICE)
        where = s["pages"][b].long()[torch.div(j, page, rounding_mode="floor")], slice(None), j % page
        k, v = (_decoded(s[name][0][where], s[name][1][where], D).transpose(0, 1) for name in ("k", "v"))
        for t in range(T):
            m = n - (T - 1 - t)
            if m <= 0:
                continue
            scores = torch.bmm(q[b, t], k[:, :m].transpose(1, 2)) / math.sqrt(D)
            stat = torch.logsumexp(scores, -1)
            out[b, t] = torch.bmm((scores - stat[..., None]).exp(), v[:, :m]).reshape(H, D)
            lse[b, t] = stat.reshape(H)
    return dict(out=out if T > 1 else out[:, 0], lse=lse if T > 1 else lse[:, 0],
                status=torch.zeros(B, dtype=torch.int32, device=DEVICE))


def _exact_verify(case, s):
    """Row by row and draft by draft, each step of the definition in turn."""
    B, n, V = case["rows"], case["drafts"], case["vocab"]
    drafts, uniforms, heats = s["drafts"].tolist(), s["uniforms"].tolist(), s["temperature"].tolist()
    tokens = torch.full((B, n + 1), -1, dtype=torch.int64, device=DEVICE)
    probs = torch.zeros((B, n + 1), dtype=torch.float64, device=DEVICE)
    counts = torch.zeros(B, dtype=torch.int32, device=DEVICE)

    def target(b, i):
        x = s["logits"][b, i].double()
        if heats[b] == 0:
            p = torch.zeros(V, dtype=torch.float64, device=DEVICE)
            p[torch.nonzero(x == x.max())[0, 0]] = 1.0
            return p
        return torch.softmax(x / heats[b], 0)

    for b in range(B):
        i = 0
        p = target(b, 0)
        weight = p
        while i < n and drafts[b][i] >= 0:
            d = drafts[b][i]
            q = s["draft_probs"][b, i].double() if s["draft_probs"] is not None else None
            if uniforms[b][i] * (float(q[d]) if q is not None else 1.0) >= float(p[d]):
                rest = torch.relu(p - q) if q is not None else p.index_fill(0, torch.tensor([d], device=DEVICE), 0.0)
                weight = rest if float(rest.sum()) > 0 else p
                break
            tokens[b, i], probs[b, i] = d, p[d]
            i += 1
            p = target(b, i)
            weight = p
        mass = torch.cumsum(weight, 0)
        past = torch.nonzero(mass > uniforms[b][n] * mass[-1])
        t = past[0, 0] if len(past) else torch.nonzero(weight > 0)[-1, 0]
        tokens[b, i], probs[b, i], counts[b] = t, p[t], i + 1
    return dict(tokens=tokens, probs=probs, counts=counts, status=torch.zeros(B, dtype=torch.int32, device=DEVICE))
