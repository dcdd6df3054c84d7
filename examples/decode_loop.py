"""A decode loop on the GPU operators: a batch of rows behind one shared prompt.

    python examples/decode_loop.py --rows 16 --steps 32

A one-layer attention model with random weights stands in for a checkpoint; the
calls are those of a real decode step:

    hidden -> QKV projection (Int8Linear) -> append_kv (rotation, paged cache)
           -> prefix_attention (the prompt's pages once, each row's own pages)
           -> output projection (Int8Linear) -> logits (Int8Linear, fp32)
           -> Sampler.sample_batch

The prompt's keys and values are appended once for all rows.  The step runs as
a CUDA graph: the positions, slots, lengths and uniforms that change from step
to step are device tensors, and nothing is read back between the steps.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from miniserve_b200 import Sampler  # noqa: E402
from miniserve_b200.attention import prefix_attention  # noqa: E402
from miniserve_b200.int8 import Int8Linear  # noqa: E402
from miniserve_b200.kvcache import append_kv, rope_table  # noqa: E402


class ToyModel:
    """Embedding, one attention layer, head: random weights of the given sizes."""

    def __init__(self, vocab=5003, hidden=896, heads=14, kv_heads=2, dim=64, positions=4096, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(rows, cols):
            return torch.randn((rows, cols), generator=gen, device=device) * cols ** -0.5

        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.embedding = torch.randn((vocab, hidden), generator=gen, device=device).bfloat16()
        self.qkv = Int8Linear.from_float(weight((heads + 2 * kv_heads) * dim, hidden))
        self.out = Int8Linear.from_float(weight(hidden, heads * dim))
        self.head = Int8Linear.from_float(weight(vocab, hidden) * 4.0)
        self.rope = rope_table(positions, dim, base=1e6, device=device)

    def project(self, tokens):
        """(hidden, q, k, v) of tokens [T]; q, k and v are slices of one product."""
        hidden = self.embedding[tokens]
        qkv = self.qkv(hidden, out_dtype=torch.bfloat16).view(len(tokens), -1, self.dim)
        return hidden, *qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)


class DecodeLoop:
    """``rows`` sequences behind one prompt: the prompt's pages first in the
    cache, then every row's own, reserved for ``steps`` tokens."""

    def __init__(self, model: ToyModel, prompt, rows: int, steps: int, page_size: int = 16) -> None:
        dev = model.embedding.device
        shared = -(-len(prompt) // page_size)
        each = -(-steps // page_size)
        shape = (shared + rows * each, page_size, model.kv_heads, model.dim)
        self.model, self.prefix_length, self.page_size = model, len(prompt), page_size
        self.cache_k = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
        self.cache_v = torch.zeros_like(self.cache_k)
        self.prefix_pages = torch.arange(shared, dtype=torch.int32, device=dev)
        self.pages = torch.arange(shared, shape[0], dtype=torch.int32, device=dev).view(rows, each)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.tokens = torch.as_tensor(prompt[-1:], dtype=torch.int64, device=dev).repeat(rows)
        self.uniforms = torch.zeros(rows, dtype=torch.float64, device=dev)
        self.rows = torch.arange(rows, device=dev)
        # the prompt: slots 0.. of the shared pages; a one-layer model's keys need no attention
        tokens = torch.as_tensor(prompt, dtype=torch.int64, device=dev)
        place = torch.arange(len(prompt), device=dev)
        _, _, k, v = model.project(tokens)
        _, status = append_kv(self.cache_k, self.cache_v, k, v, place, positions=place, rope=model.rope)
        assert not bool(status.any())

    def logits(self):
        """One step up to the logits [rows, vocab] fp32, the new tokens appended."""
        m = self.model
        hidden, q, k, v = m.project(self.tokens)
        n = self.lengths.long()
        slots = self.pages[self.rows, n // self.page_size].long() * self.page_size + n % self.page_size
        q, _ = append_kv(self.cache_k, self.cache_v, k, v, slots, q=q, positions=self.prefix_length + n, rope=m.rope)
        self.lengths += 1
        mixed, _, _ = prefix_attention(q, self.cache_k, self.cache_v, self.pages, self.lengths,
                                       prefix_pages=self.prefix_pages, prefix_length=self.prefix_length)
        hidden = hidden + m.out(mixed.flatten(1), out_dtype=torch.bfloat16)
        return m.head(hidden)

    def step(self, sampler: Sampler, **params):
        logits = self.logits()
        tokens, _, _ = sampler.sample_batch(logits, uniforms=self.uniforms, **params)
        self.tokens.copy_(tokens)

    def capture(self, sampler: Sampler, **params):
        """The step as a CUDA graph (the loop's state is left as it is)."""
        keep = [t.clone() for t in (self.lengths, self.tokens)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step(sampler, **params)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.step(sampler, **params)
        for t, k in zip((self.lengths, self.tokens), keep):
            t.copy_(k)
        return graph


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=500, help="tokens of the shared prompt")
    args = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    model = ToyModel()
    prompt = torch.randint(0, model.embedding.shape[0], (args.prompt,), generator=gen).tolist()
    loop = DecodeLoop(model, prompt, args.rows, args.steps + 1)
    params = dict(temperature=torch.full((args.rows,), 0.8, dtype=torch.float64, device="cuda"),
                  top_k=torch.full((args.rows,), 50, dtype=torch.int32, device="cuda"),
                  top_p=torch.full((args.rows,), 0.95, dtype=torch.float64, device="cuda"))
    graph = loop.capture(Sampler(), **params)
    uniforms = torch.rand((args.steps, args.rows), generator=gen, dtype=torch.float64).cuda()
    history = torch.empty((args.steps, args.rows), dtype=torch.int64, device="cuda")
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for i in range(args.steps):
        loop.uniforms.copy_(uniforms[i])
        graph.replay()
        history[i].copy_(loop.tokens)
    stop.record()
    torch.cuda.synchronize()
    for b, row in enumerate(history.T.tolist()[:4]):
        print(f"row {b}:", *row[:12], "...")
    print(f"{args.rows} rows, {args.steps} steps: {start.elapsed_time(stop) / args.steps * 1000:.0f} us a step")


if __name__ == "__main__":
    main()
