"""Speculative decoding of a batch over a paged, quantised KV cache, with the library's operators.

A small decoder with seeded random weights stands in for a model: what it shows is the order of the
calls. Per pass every sequence brings its last token and a prompt-lookup draft (plan.LookupDrafter,
src/draft.ts:60-98); each layer quantises the pass's keys and values into the sequences' pages
(store), attends over them (attention), and the batch's logits decide in one call which drafts
stand and what follows (verify_drafts). Rows of refused drafts stay in the pages: the sequence's
length says what counts, and the next pass writes over them.

    python examples/paged_speculation.py [--tokens 48] [--format int8] [--temperature 0.8]
"""
from __future__ import annotations

import argparse
import importlib
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import __graft_entry__ as entry  # noqa: E402

pkg = entry.load_package()
paged = importlib.import_module(pkg.__name__ + ".paged")


class Decoder:
    """Pre-norm layers of grouped attention and a gated MLP, f32, a tied head."""

    def __init__(self, layers=3, hidden=256, heads=8, kv_heads=2, head_dim=64, vocab=384, seed=11):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def w(n, k):
            return torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)

        self.heads, self.kv_heads, self.head_dim, self.vocab = heads, kv_heads, head_dim, vocab
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda")
        self.layers = [{"qkv": w((heads + 2 * kv_heads) * head_dim, hidden), "o": w(hidden, heads * head_dim),
                        "gate": w(2 * hidden, hidden), "up": w(2 * hidden, hidden), "down": w(hidden, 2 * hidden)}
                       for _ in range(layers)]

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def rotate(self, x, pos):
        half = self.head_dim // 2
        angle = pos[:, None].float() * torch.pow(1e4, -torch.arange(half, device=x.device) / half)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)


class Server:
    """Sequences of one Decoder whose caches share a pool of pages per layer."""

    def __init__(self, model: Decoder, sequences: int, max_context=512, page_size=16, format="int8", window=0):
        self.model, self.page_size, self.window, self.max_context = model, page_size, window, max_context
        pages = sequences * -(-max_context // page_size)
        self.pools = [paged.PagePool.create(pages, page_size, model.kv_heads, model.head_dim, format)
                      for _ in model.layers]
        self.free = list(range(pages))
        self.table = torch.full((sequences, -(-max_context // page_size)), -1, dtype=torch.int32)
        self.held = [0] * sequences
        self.length = [0] * sequences

    def reserve(self, b: int, positions: int) -> None:
        while self.held[b] * self.page_size < positions:
            self.table[b, self.held[b]] = self.free.pop()
            self.held[b] += 1

    def forward(self, tokens: list) -> torch.Tensor:
        """Logits of every token of `tokens` (a list per sequence), placed after what its sequence
        holds. The sequences' lengths move only by `accept`."""
        m, dev = self.model, "cuda"
        begin, pos = [0], []
        for b, ids in enumerate(tokens):
            self.reserve(b, self.length[b] + len(ids))
            begin.append(begin[-1] + len(ids))
            pos += range(self.length[b], self.length[b] + len(ids))
        seq = torch.tensor([b for b, ids in enumerate(tokens) for _ in ids])
        where = torch.tensor(pos)
        slots = (self.table[seq, where // self.page_size] * self.page_size + where % self.page_size).to(torch.int32).to(dev)
        table, where = self.table.to(dev), where.to(dev)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        q_begin, q_pos = ints(begin), ints(self.length)
        kv = [n + len(ids) for n, ids in zip(self.length, tokens)]
        kv_len = ints(kv)
        x = m.embed[torch.tensor([t for ids in tokens for t in ids], device=dev)]
        H, G, D = m.heads, m.kv_heads, m.head_dim
        for w, pool in zip(m.layers, self.pools):
            qkv = (m.norm(x) @ w["qkv"].T).view(-1, H + 2 * G, D)
            q = m.rotate(m.norm(qkv[:, :H]), where)
            k = m.rotate(m.norm(qkv[:, H:H + G]), where)
            pool.store(k, qkv[:, H + G:], slots)
            a = paged.attention(pool, q, q_begin, q_pos, kv_len, table, max(map(len, tokens)), max(kv),
                                window=self.window, scale=1 / math.sqrt(D))
            x = x + a.reshape(-1, H * D) @ w["o"].T
            h = m.norm(x)
            x = x + (torch.nn.functional.gelu(h @ w["gate"].T, approximate="tanh") * (h @ w["up"].T)) @ w["down"].T
        return 8.0 * m.norm(x) @ m.embed.T / math.sqrt(m.embed.shape[1])

    def accept(self, b: int, n: int) -> None:
        self.length[b] += n


def generate(model: Decoder, prompts: list, tokens: int, max_drafts: int, temperature=0.0, seed=5, **server):
    """`tokens` new tokens for each prompt; (their ids, passes, accepted drafts)."""
    B = len(prompts)
    s = Server(model, B, **server)
    g = torch.Generator(device="cuda").manual_seed(seed)
    drafter = pkg.plan.LookupDrafter()
    history, want = [list(p) for p in prompts], [len(p) + tokens for p in prompts]
    # The prompts but for their last tokens, in one ragged pass.
    s.forward([p[:-1] for p in history])
    for b in range(B):
        s.accept(b, len(history[b]) - 1)
    temp = torch.full((B,), float(temperature), device="cuda")
    passes = accepted = 0
    while any(len(h) < w for h, w in zip(history, want)):
        drafts = [drafter.propose(h, min(max_drafts, w - len(h) - 1)) if len(h) < w else [] for h, w in zip(history, want)]
        logits = s.forward([[h[-1], *d] if len(h) < w else [] for h, d, w in zip(history, drafts, want)])
        rows = [len(d) + 1 if len(h) < w else 0 for h, d, w in zip(history, drafts, want)]
        begin = [sum(rows[:b]) for b in range(B + 1)]
        # Row i of a sequence tests draft i; the last row's entry is not used.
        flat = [t for d, n in zip(drafts, rows) for t in ([*d, 0] if n else [])]
        gumbel = -torch.log(torch.empty(B, model.vocab, device="cuda").exponential_(generator=g))
        ids, _, counts = paged.verify_drafts(
            logits, torch.tensor(begin, dtype=torch.int32, device="cuda"),
            torch.tensor(flat, dtype=torch.int32, device="cuda"),
            torch.rand(len(flat), generator=g, device="cuda"), gumbel, temp, max_drafts)
        ids, counts = ids.tolist(), counts.tolist()
        for b, n in enumerate(counts):
            if n:
                history[b] += ids[b][:n]
                s.accept(b, n)          # the last token and the accepted drafts are cached now
                accepted += n - 1
        passes += 1
    if paged.errors():
        raise RuntimeError("a paged operator met bad pages or lengths")
    return [h[len(p):] for h, p in zip(history, prompts)], passes, accepted


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--format", default="int8", choices=["bf16", "int8", "e4m3"])
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--drafts", type=int, default=5)
    ap.add_argument("--window", type=int, default=0)
    a = ap.parse_args(argv)
    model = Decoder()
    rng = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, model.vocab, (n,), generator=rng).tolist() for n in (70, 2, 33)]
    kw = dict(format=a.format, window=a.window, temperature=a.temperature)
    plain, plain_passes, _ = generate(model, prompts, a.tokens, 0, **kw)
    ids, passes, accepted = generate(model, prompts, a.tokens, a.drafts, **kw)
    out = {"ids": ids, "plain": plain, "passes": passes, "plain_passes": plain_passes, "accepted": accepted}
    print(f"{a.tokens} tokens x {len(prompts)} sequences: {plain_passes} passes one token at a time, {passes} with "
          f"drafts ({accepted} accepted)" + (f"; the same ids: {ids == plain}" if a.temperature == 0 else ""))
    return out


if __name__ == "__main__":
    main()
