"""A decode loop that drafts: several tokens a row and step, over a 4-bit cache.

    python examples/drafted_loop.py --rows 16 --steps 200 --drafts 4

The model is the random one of decode_loop.py.  Every row proposes what followed
its newest tokens the last time they occurred in its text, and the step checks
all proposals at once:

    newest token + drafts -> QKV projection (Int8Linear)
        -> append_kv4 (rotation, quantised as written) -> attention_kv4 (each
           token with a length of its own) -> output projection -> logits
        -> verify_drafts (drafts kept, one more token drawn)

A rejected draft's slot is written again by the next step.  The step runs as a
CUDA graph; nothing is read back between the steps.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch  # noqa: E402

from decode_loop import ToyModel  # noqa: E402
from miniserve_b200 import KvCache4, append_kv4, attention_kv4, verify_drafts  # noqa: E402


class DraftedLoop:
    """One sequence a prompt, each with pages for ``steps`` steps of up to
    ``drafts`` + 1 tokens."""

    def __init__(self, model: ToyModel, prompts, steps: int, drafts: int = 4, page_size: int = 16) -> None:
        dev = model.embedding.device
        vocab, rows = model.embedding.shape[0], len(prompts)
        each = -(-(max(map(len, prompts)) + steps * (drafts + 1)) // page_size)
        self.model, self.drafts, self.page_size, self.vocab = model, drafts, page_size, vocab
        self.cache = KvCache4.empty(rows * each, page_size, model.kv_heads, model.dim, dtype=torch.bfloat16, device=dev)
        self.pages = torch.randperm(rows * each, device=dev).int().view(rows, each)
        self.lengths = torch.tensor([len(p) - 1 for p in prompts], device=dev)  # in the cache: all but the newest token
        self.newest = torch.tensor([p[-1] for p in prompts], device=dev)
        self.uniforms = torch.zeros((rows, drafts + 1), dtype=torch.float64, device=dev)
        self.rows = torch.arange(rows, device=dev)
        # what followed a token the last time (the last column takes what is none)
        self.follows = torch.full((rows, vocab + 1), -1, device=dev)
        for b, prompt in enumerate(prompts):
            if len(prompt) == 1:
                continue
            text = torch.as_tensor(prompt, device=dev)
            for at in range(len(prompt) - 1):
                self.follows[b, prompt[at]] = prompt[at + 1]
            place = torch.arange(len(prompt) - 1, device=dev)
            _, _, k, v = model.project(text[:-1])
            _, status = append_kv4(self.cache, k, v, self.slots(place[None], self.rows[b:b + 1])[0], positions=place, rope=model.rope)
            assert not bool(status.any())

    def slots(self, place, rows):
        return self.pages[rows[:, None], place // self.page_size].long() * self.page_size + place % self.page_size

    def propose(self):
        """[rows, drafts]: a chain of followers, -1 from where there is none."""
        out, token = [], self.newest
        for _ in range(self.drafts):
            token = self.follows[self.rows, torch.where(token < 0, self.vocab, token)]
            out.append(token)
        return torch.stack(out, 1)

    def logits(self, drafts):
        """[rows, drafts + 1, vocab] fp32 after the newest token and after each
        draft; the tokens are in the cache then."""
        m, (rows, n) = self.model, drafts.shape
        fed = torch.cat([self.newest[:, None], drafts], 1)
        i = torch.arange(n + 1, device=fed.device)
        place = self.lengths[:, None] + i
        slots = torch.where(fed < 0, -1, self.slots(place, self.rows))  # no draft: padding, which sees no keys
        hidden, q, k, v = m.project(fed.clamp(min=0).flatten())
        q, _ = append_kv4(self.cache, k, v, slots.flatten(), q=q, positions=place.flatten(), rope=m.rope)
        seen = torch.where(fed < 0, 0, place + 1).int()
        mixed, _, _ = attention_kv4(q.view(rows, n + 1, m.heads, m.dim), self.cache, self.pages, seen)
        hidden = hidden + m.out(mixed.view(rows * (n + 1), -1), out_dtype=torch.bfloat16)
        return m.head(hidden).view(rows, n + 1, -1)

    def step(self, temperature=0.0):
        """Returns ([rows, drafts + 1] tokens, -1 behind the last, [rows] counts)."""
        drafts = self.propose()
        tokens, _, counts, _ = verify_drafts(self.logits(drafts), drafts, self.uniforms, temperature=temperature)
        before = self.newest
        for i in range(self.drafts + 1):  # in order: the last occurrence stays
            token = tokens[:, i]
            self.follows[self.rows, torch.where(token < 0, self.vocab, before)] = token
            before = torch.where(token < 0, before, token)
        self.follows[:, self.vocab] = -1
        self.newest.copy_(before)
        self.lengths += counts
        return tokens, counts

    def capture(self, temperature=0.0):
        """The step as a CUDA graph and its outputs (the loop's state is left as it is)."""
        state = (self.lengths, self.newest, self.follows)
        keep = [t.clone() for t in state]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step(temperature)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = self.step(temperature)
        for t, k in zip(state, keep):
            t.copy_(k)
        return graph, outputs


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=500, help="tokens of the longest prompt")
    ap.add_argument("--temperature", type=float, default=0.0)
    args = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    model = ToyModel()
    prompts = [torch.randint(0, model.embedding.shape[0], (max(1, args.prompt - 7 * b),), generator=gen).tolist()
               for b in range(args.rows)]
    loop = DraftedLoop(model, prompts, args.steps, args.drafts)
    heat = torch.full((args.rows,), args.temperature, dtype=torch.float64, device="cuda")
    graph, (tokens, counts) = loop.capture(heat)
    uniforms = torch.rand((args.steps, args.rows, args.drafts + 1), generator=gen, dtype=torch.float64).cuda()
    history, taken = [], torch.empty((args.steps, args.rows), dtype=torch.int32, device="cuda")
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for i in range(args.steps):
        loop.uniforms.copy_(uniforms[i])
        graph.replay()
        taken[i].copy_(counts)
        history.append(tokens.clone())
    stop.record()
    torch.cuda.synchronize()
    for b, row in enumerate(torch.cat(history, 1)[:4].tolist()):
        print(f"row {b}:", *[t for t in row if t >= 0][:12], "...")
    print(f"{args.rows} rows, {args.steps} steps: {float(taken.float().mean()):.2f} tokens a row and step, "
          f"{start.elapsed_time(stop) / args.steps * 1000:.0f} us a step")


if __name__ == "__main__":
    main()
