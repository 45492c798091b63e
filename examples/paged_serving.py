"""Continuous batching over a paged 4-bit cache: a small decoder with random
weights serves requests of different lengths.

    python examples/paged_serving.py [--requests 12] [--layers 4] [--dtype bf16]

Every step admits waiting requests while there are slots and pages, takes the
next chunk of each prompt (attention over the chunk and, read back from the
cache, the tokens before it) and decodes one token for every running sequence.
``Server.step`` returns the logits it sampled from.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from innerq_b200.paged import PagedCache  # noqa: E402
from innerq_b200.prompt import prompt_attention  # noqa: E402

HEAD_DIM = 128


class Decoder:
    """Pre-norm transformer layers whose attention is the cache's."""

    def __init__(self, layers=4, heads=8, kv_heads=2, hidden=512, vocab=1000, max_pos=8192, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *s: (torch.randn(s, device="cuda", generator=g) * s[-1] ** -0.5).to(dtype)  # noqa: E731
        self.heads, self.kv_heads, self.dtype = heads, kv_heads, dtype
        self.embed, self.unembed = w(vocab, hidden), w(vocab, hidden)
        self.layers = [dict(qkv=w((heads + 2 * kv_heads) * HEAD_DIM, hidden), o=w(hidden, heads * HEAD_DIM),
                            up=w(2 * hidden, hidden), down=w(hidden, 2 * hidden)) for _ in range(layers)]
        angle = torch.arange(max_pos, device="cuda")[:, None] * 10000.0 ** -(
            torch.arange(0, HEAD_DIM, 2, device="cuda") / HEAD_DIM)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    @staticmethod
    def norm(x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)

    def forward(self, ids, attend):
        """ids [T]; attend(layer, q, k, v) -> [T, heads, 128] rotates, stores and attends."""
        x = self.embed[ids]
        for i, w in enumerate(self.layers):
            qkv = (self.norm(x) @ w["qkv"].T).view(len(ids), -1, HEAD_DIM)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)  # views: no copies
            x = x + attend(i, q, k, v).flatten(1) @ w["o"].T
            x = x + torch.nn.functional.silu(self.norm(x) @ w["up"].T) @ w["down"].T
        return self.norm(x) @ self.unembed.T


class Request:
    def __init__(self, prompt, new_tokens):
        self.tokens, self.prompt_len, self.left = list(prompt), len(prompt), new_tokens
        self.cached = 0  # tokens in the cache
        self.slot, self.pages = -1, []


class Server:
    def __init__(self, model: Decoder, n_pages=256, n_slots=8, page_size=64, w_sink=32, w_recent=32, chunk=256):
        self.model, self.chunk = model, chunk
        self.caches = [PagedCache.allocate(n_pages, model.kv_heads, n_slots, page_size, w_sink, w_recent, model.dtype)
                       for _ in model.layers]  # one table serves every layer
        self.n_pages = n_pages
        self.free_pages, self.free_slots = list(range(n_pages)), list(range(n_slots))
        self.waiting, self.running = [], []

    def submit(self, prompt, new_tokens):
        """Queue a request; one that could never be served raises."""
        total = len(prompt) + new_tokens
        if not len(prompt) or new_tokens < 1:
            raise ValueError(f"a request needs tokens before and after: {len(prompt)} and {new_tokens}")
        if self.caches[0].pages_for(total) > self.n_pages or total - 1 > len(self.model.cos):
            raise ValueError(f"{total} tokens do not fit {self.n_pages} pages or {len(self.model.cos)} positions")
        r = Request(prompt, new_tokens)
        self.waiting.append(r)
        return r

    # ------------------------------------------------------------ scheduling
    def _pages(self, r, length):
        """Give r the pages that `length` tokens need; False if there are too few."""
        need = self.caches[0].pages_for(length) - len(r.pages)
        if need > len(self.free_pages):
            return False
        for _ in range(need):
            r.pages.append(self.free_pages.pop())
        return True

    def _admit(self):
        while self.waiting and self.free_slots:
            r = self.waiting[0]
            if not self._pages(r, r.prompt_len + r.left):  # all it will ever need: no preemption here
                break
            r.slot = self.free_slots.pop()
            self.running.append(self.waiting.pop(0))

    def _finish(self, r):
        self.free_pages += r.pages
        self.free_slots.append(r.slot)
        self.running.remove(r)

    def _batch(self, rs):
        """Page table, slots and lengths of these requests, on the device."""
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        width = max(1, max(len(r.pages) for r in rs))
        return i32([r.pages + [-1] * (width - len(r.pages)) for r in rs]), i32([r.slot for r in rs]), i32([r.cached for r in rs])

    # ----------------------------------------------------------------- steps
    def prefill(self, rs):
        """The next chunk of each of these prompts; logits of their last tokens."""
        new = [min(self.chunk, r.prompt_len - r.cached) for r in rs]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        table, slots, lens = self._batch(rs)
        cu = i32(start)
        before = [r.cached for r in rs]
        past = torch.tensor([0] + before, device="cuda").cumsum(0).int()
        cu_k = cu + past
        ids = torch.tensor([t for r, n in zip(rs, new) for t in r.tokens[r.cached:r.cached + n]], device="cuda")

        def attend(layer, q, k, v):
            c = self.caches[layer]
            q, k = c.append(q, k, v, table, slots, lens, cu, cos=self.model.cos, sin=self.model.sin, return_k=True)
            if any(before):  # the tokens before the chunks, as the cache holds them
                now = lens + cu.diff()
                pk, pv = c.read(table, slots, now, torch.zeros_like(lens), past, sum(before))
                join = lambda a, b: torch.cat([x for p, x2 in zip(a.split(before), b.split(new)) for x in (p, x2)])  # noqa: E731
                k, v = join(pk, k), join(pv, v)
            return prompt_attention(q, k, v, cu, cu_k)

        logits = self.model.forward(ids, attend)
        for r, n in zip(rs, new):
            r.cached += n
        return logits[cu[1:].long() - 1]

    def decode(self, rs):
        """One token of each of these sequences."""
        table, slots, lens = self._batch(rs)
        ids = torch.tensor([r.tokens[r.cached] for r in rs], device="cuda")
        after = lens + 1

        def attend(layer, q, k, v):
            c = self.caches[layer]
            q = c.append(q, k, v, table, slots, lens, cos=self.model.cos, sin=self.model.sin)
            return c.attend(q, table, slots, after)

        logits = self.model.forward(ids, attend)
        for r in rs:
            r.cached += 1
        return logits

    def step(self):
        """One scheduling step; [(request, logits)] of the tokens it produced."""
        self._admit()
        prompts = [r for r in self.running if r.cached < r.prompt_len]
        decodes = [r for r in self.running if r.cached >= r.prompt_len]
        produced = []
        if prompts:
            logits = self.prefill(prompts)
            produced += [(r, x) for r, x in zip(prompts, logits) if r.cached == r.prompt_len]
        if decodes:
            produced += list(zip(decodes, self.decode(decodes)))
        if produced:
            for (r, _), t in zip(produced, torch.stack([x for _, x in produced]).argmax(-1).tolist()):
                r.tokens.append(t)
                r.left -= 1
                if r.left == 0:
                    self._finish(r)
        return produced


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=12)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--dtype", default="bf16", choices=["fp16", "bf16"])
    a = ap.parse_args()
    model = Decoder(layers=a.layers, dtype=torch.bfloat16 if a.dtype == "bf16" else torch.float16)
    server = Server(model)
    g = torch.Generator().manual_seed(0)
    rs = [server.submit(torch.randint(0, 1000, (int(n),), generator=g).tolist(), 40)
          for n in torch.randint(1, 900, (a.requests,), generator=g)]
    t, steps, tokens = time.time(), 0, 0
    while server.running or server.waiting:
        tokens += len(server.step())
        steps += 1
    torch.cuda.synchronize()
    print(f"{len(rs)} requests, {sum(r.prompt_len for r in rs)} prompt tokens, {tokens} new tokens in {steps} steps, "
          f"{time.time() - t:.2f} s; pages and slots all free again: "
          f"{len(server.free_pages) == 256 and len(server.free_slots) == 8}")
    print("first request's tokens:", rs[0].tokens[rs[0].prompt_len:][:16])


if __name__ == "__main__":
    main()
