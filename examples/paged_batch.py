"""A continuous batch over paged KV caches: requests of different lengths share the pages of one
pool per layer, prompts and single new tokens go through the same step.

A small decoder with random Q8_0 weights and per-head norms of queries and keys. Each step takes up
to 128 rows: one row for every running request's new token, the rest for pieces of waiting prompts,
unused rows as padding (position -1). Per layer: projections (prefill_matmul), then
PagedKvCache.append (norms, rotation and the write into the pages in one pass), then
PagedKvCache.attention, every row over its own sequence up to its own position. Pages are handed out
as sequences grow and go back to the pool when a request ends; PagedKvCache.read saves its last
positions' keys and values first.

    python examples/paged_batch.py [--requests N] [--cache q8_0|q4_0|f16|bf16]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ssd-llm_b200"))

import torch  # noqa: E402

import ssdllm  # noqa: E402

ROWS = 128  # rows of a step (prefill_matmul takes multiples of 128)
CACHE = {"f16": ssdllm.F16, "bf16": ssdllm.BF16, "q8_0": ssdllm.Q8_0, "q4_0": ssdllm.Q4_0}


class Decoder:
    """n_layers of attention and SwiGLU with resident Q8_0 weights, and a paged cache per layer."""

    def __init__(self, ctx, n_layers=2, n_embd=512, n_head=8, n_head_kv=2, head_dim=64, n_ff=1024,
                 vocab=256, n_pages=96, page_size=16, cache="q8_0", max_positions=512, seed=0):
        self.ctx, self.dev = ctx, torch.device("cuda", ctx.device)
        self.n_embd, self.n_head, self.n_head_kv, self.head_dim = n_embd, n_head, n_head_kv, head_dim
        self.page_size, self.n_pages, self.max_positions = page_size, n_pages, max_positions
        ids = iter(range(1000))

        def weight(rows, cols):
            return ssdllm.Weight.synth(ctx, ssdllm.Q8_0, seed, next(ids), 0.05, cols, 0, rows, 0, cols)

        g = torch.Generator().manual_seed(seed)

        def norm(n):
            return (1 + 0.1 * torch.randn(n, generator=g)).to(self.dev)

        qkv = (n_head + 2 * n_head_kv) * head_dim
        self.layers = [{"qkv": weight(qkv, n_embd), "o": weight(n_embd, n_head * head_dim),
                        "gate": weight(n_ff, n_embd), "up": weight(n_ff, n_embd),
                        "down": weight(n_embd, n_ff), "attn_norm": norm(n_embd), "ffn_norm": norm(n_embd),
                        "q_norm": norm(head_dim), "k_norm": norm(head_dim),
                        "kv": ssdllm.PagedKvCache(ctx, n_pages, page_size, n_head_kv, head_dim, CACHE[cache])}
                       for _ in range(n_layers)]
        self.embed = torch.randn(vocab, n_embd, generator=g).to(self.dev)
        self.out = weight(vocab, n_embd)
        self.out_norm = norm(n_embd)
        self.rope = torch.empty(max_positions, head_dim // 2, 2, device=self.dev)
        ssdllm.rope_table(ctx, head_dim, 10000.0, max_positions, self.rope)
        self.work = self.layers[0]["kv"].attention_workspace()

    def _norm(self, x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w

    def _matmul(self, w, x):
        y = torch.empty(x.shape[0], w.rows, device=self.dev)
        ssdllm.prefill_matmul(self.ctx, w, x.contiguous(), y)
        return y

    def step(self, tokens, pos, seq, table):
        """One row per token (padding rows: position -1); returns the rows' logits."""
        h, hk, d = self.n_head, self.n_head_kv, self.head_dim
        x = self.embed[tokens]
        q = torch.empty(ROWS, h * d, device=self.dev)
        att = torch.empty(ROWS, h * d, device=self.dev)
        for la in self.layers:
            qkv = self._matmul(la["qkv"], self._norm(x, la["attn_norm"]))
            la["kv"].append(qkv[:, h * d:(h + hk) * d], qkv[:, (h + hk) * d:], pos, table, seq=seq,
                            q=qkv[:, :h * d], q_out=q, q_norm=la["q_norm"], k_norm=la["k_norm"],
                            rope=self.rope, rope_halves=True)
            la["kv"].attention(q, pos + 1, table, att, self.work, seq=seq)
            x = x + self._matmul(la["o"], att)
            n = self._norm(x, la["ffn_norm"])
            a = torch.nn.functional.silu(self._matmul(la["gate"], n)) * self._matmul(la["up"], n)
            x = x + self._matmul(la["down"], a)
        return self._matmul(self.out, self._norm(x, self.out_norm))


class Batch:
    """Requests over one Decoder: pages from a free list, a page table per slot."""

    def __init__(self, model, slots=16):
        self.model, self.slots = model, slots
        width = -(-model.max_positions // model.page_size)
        self.table = torch.full((slots, width), -1, dtype=torch.int32)
        self.free = list(range(model.n_pages))[::-1]
        self.run = [None] * slots  # the slot's request: tokens, how many are cached, its end
        self.saved = {}

    def _reserve(self, slot, upto):
        """Pages for positions below `upto`; how many positions the slot has pages for."""
        have = int((self.table[slot] >= 0).sum())
        while have * self.model.page_size < upto and self.free:
            self.table[slot, have] = self.free.pop()
            have += 1
        return have * self.model.page_size

    def _finish(self, slot):
        r, m = self.run[slot], self.model
        n = min(len(r["tokens"]) - 1, m.page_size)  # the last cached positions, as a user may keep them
        last = torch.arange(r["cached"] - n, r["cached"], dtype=torch.int32, device=m.dev)
        k = torch.empty(n, m.n_head_kv * m.head_dim, device=m.dev)
        v = torch.empty_like(k)
        m.layers[-1]["kv"].read(last, self.table.to(m.dev), k, v,
                                seq=torch.full((n,), slot, dtype=torch.int32, device=m.dev))
        self.saved[r["id"]] = (k, v)
        self.free += [int(p) for p in self.table[slot] if p >= 0]
        self.table[slot] = -1
        self.run[slot] = None

    def generate(self, requests):
        """requests: {id: (prompt tokens, new tokens)}; returns {id: generated tokens}."""
        waiting, done, m = list(requests.items()), {}, self.model
        most = min(m.max_positions, m.n_pages * m.page_size)
        for rid, (prompt, new) in waiting:  # none that no step would ever take up or end
            if not prompt or new < 1 or len(prompt) + new > most:
                raise ValueError(f"request {rid}: {len(prompt)} prompt and {new} new tokens, 1 or more of each "
                                 f"and {most} together are possible")
        while waiting or any(self.run):
            for slot in range(self.slots):  # admit
                if self.run[slot] is None and waiting:
                    rid, (prompt, new) = waiting[0]
                    if self._reserve(slot, len(prompt) + new) < len(prompt) + new:
                        self.free += [int(p) for p in self.table[slot] if p >= 0]
                        self.table[slot] = -1
                        break  # not enough pages yet
                    waiting.pop(0)
                    self.run[slot] = {"id": rid, "tokens": list(prompt), "cached": 0, "end": len(prompt) + new,
                                      "prompt": len(prompt)}
            rows, last = [], {}
            order = sorted((s for s in range(self.slots) if self.run[s]),
                           key=lambda s: len(self.run[s]["tokens"]) - self.run[s]["cached"])
            for slot in order:  # new tokens first, then as much of the prompts as fits
                r = self.run[slot]
                n = min(len(r["tokens"]) - r["cached"], ROWS - len(rows))
                rows += [(r["tokens"][p], p, slot) for p in range(r["cached"], r["cached"] + n)]
                r["cached"] += n
                if n and r["cached"] == len(r["tokens"]):
                    last[slot] = len(rows) - 1
            rows += [(0, -1, 0)] * (ROWS - len(rows))
            t = torch.tensor(rows, dtype=torch.int32).t().contiguous().to(m.dev)
            logits = m.step(t[0].long(), t[1].contiguous(), t[2].contiguous(), self.table.to(m.dev))
            best = logits.argmax(-1).cpu()
            for slot, row in last.items():
                r = self.run[slot]
                r["tokens"].append(int(best[row]))
                if len(r["tokens"]) >= r["end"]:
                    done[r["id"]] = r["tokens"][r["prompt"]:]
                    self._finish(slot)
        return done


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=24)
    ap.add_argument("--cache", choices=sorted(CACHE), default="q8_0")
    a = ap.parse_args()
    ctx = ssdllm.Context(0)
    model = Decoder(ctx, cache=a.cache)
    g = torch.Generator().manual_seed(1)
    requests = {}
    for i in range(a.requests):
        n = int(torch.randint(1, 200, (1,), generator=g))
        requests[i] = (torch.randint(0, 256, (n,), generator=g).tolist(), int(torch.randint(1, 24, (1,), generator=g)))
    batch = Batch(model)
    done = batch.generate(requests)
    torch.cuda.synchronize()
    assert ctx.device_status() == 0
    print(f"{len(done)} requests, {sum(len(p) for p, _ in requests.values())} prompt tokens, "
          f"{sum(len(t) for t in done.values())} generated, {len(batch.free)} of {model.n_pages} pages free")


if __name__ == "__main__":
    main()
