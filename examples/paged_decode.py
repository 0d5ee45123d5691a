"""A batch of prompts decoded greedily over one paged KV cache per layer, with the
log probability, entropy and runners-up of every answer token.

    python examples/paged_decode.py [--tokens 12] [--cache int8|bfloat16|float16]

The model is a small random decoder of the engine's shape (RMSNorm, INT8
projections, rotary grouped-query attention, SiLU); what the example shows is
how a server that drives its own batch uses the operators: pages are handed out
as sequences grow, the prompts of all sequences run as one ragged batch, every
later step has one row a sequence, and logits never leave the GPU.
"""

from __future__ import annotations

import argparse
import importlib.util
import sys
from pathlib import Path

import numpy as np
import torch

HOME = Path(__file__).resolve().parent.parent / "low-precision-transformer-accelerator-for-edge-llms_b200"


def load_package():
    if "lpta_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("lpta_b200", HOME / "__init__.py",
                                                      submodule_search_locations=[str(HOME)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["lpta_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["lpta_b200"]


class Decoder:
    """Random weights of a small decoder; every row of a step is computed by itself."""

    def __init__(self, pkg, hidden=256, heads=8, kv_heads=2, head_dim=64, inter=512, vocab=1000, layers=2,
                 max_positions=512, seed=0):
        self.pkg, self.lib = pkg, pkg.load_library()
        self.heads, self.kv_heads, self.head_dim, self.vocab, self.layers = heads, kv_heads, head_dim, vocab, layers
        rng = np.random.default_rng(seed)

        def linear(n_in, n_out):
            w = pkg.quantize_weight(rng.standard_normal((n_in, n_out)).astype(np.float32) / n_in ** 0.5, "channel")
            return (torch.from_numpy(np.ascontiguousarray(w.w.T)).cuda(),
                    torch.from_numpy(w.scale.astype(np.float32)).cuda())

        self.embed = torch.from_numpy(rng.standard_normal((vocab, hidden)).astype(np.float32)).cuda()
        self.norm = torch.ones(hidden, device="cuda")
        self.blocks = [{"qkv": linear(hidden, (heads + 2 * kv_heads) * head_dim), "o": linear(heads * head_dim, hidden),
                        "gate": linear(hidden, inter), "up": linear(hidden, inter), "down": linear(inter, hidden)}
                       for _ in range(layers)]
        self.head = linear(hidden, vocab)
        cos, sin = pkg.rope_tables(max_positions, head_dim, 10000.0)
        self.cos, self.sin = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()

    def _call(self, name, *args):
        self.pkg.shim.check(getattr(self.lib, name)(*args, torch.cuda.current_stream().cuda_stream), name)

    def rms_norm(self, x):
        out = torch.empty_like(x)
        self._call("tl_rmsnorm", x.data_ptr(), self.norm.data_ptr(), 1e-5, out.data_ptr(), *x.shape)
        return out

    def linear(self, x, weight):
        """INT8 x INT8 product with one scale a row and one a column."""
        x = x.contiguous()
        (n, k), (w, scale) = x.shape, weight
        q = torch.empty((n, k), dtype=torch.int8, device="cuda")
        peak = torch.empty(n, device="cuda")
        acc = torch.empty((n, w.shape[0]), dtype=torch.int32, device="cuda")
        self._call("tl_quantize_int8", x.data_ptr(), n, k, 1, q.data_ptr(), peak.data_ptr())
        self._call("tl_gemm_i8", q.data_ptr(), w.data_ptr(), acc.data_ptr(), n, w.shape[0], k)
        return acc.float() * (torch.where(peak == 0, 127.0, peak) / 127).unsqueeze(1) * scale

    def step(self, caches, table, tokens, seq, pos):
        """Logits [rows, vocab] of rows (token, sequence, position); their keys and values enter the caches."""
        n, h, kv = tokens.numel(), self.heads, self.kv_heads
        x, lengths = self.embed[tokens.long()], pos + 1
        for block, cache in zip(self.blocks, caches):
            qkv = self.linear(self.rms_norm(x), block["qkv"]).view(n, h + 2 * kv, self.head_dim)
            # all rows are stored before any attends: a prompt's row sees the positions up to its own
            q = cache.append(qkv[:, h:h + kv], qkv[:, h + kv:], table, seq, pos, self.cos, self.sin, q=qkv[:, :h])
            x = x + self.linear(cache.attend(q, table, lengths, seq=seq).view(n, -1), block["o"])
            y = self.rms_norm(x)
            x = x + self.linear(torch.nn.functional.silu(self.linear(y, block["gate"])) * self.linear(y, block["up"]),
                                block["down"])
        return self.linear(self.rms_norm(x), self.head)


class Pages:
    """Hands out a pool's pages; the block table lives on the host and is copied when it changes."""

    def __init__(self, num_pages, page_size, sequences, max_pages):
        self.free, self.page_size = list(range(num_pages))[::-1], page_size
        self.table = np.full((sequences, max_pages), -1, np.int32)
        self.held = [0] * sequences

    def grow(self, sequence, length):
        """Makes room for ``length`` positions of a sequence."""
        while self.held[sequence] * self.page_size < length:
            self.table[sequence, self.held[sequence]] = self.free.pop()
            self.held[sequence] += 1


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def generate(model, prompts, n_tokens, cache_dtype=torch.int8, page_size=16, top_k=3):
    """Greedy continuation of every prompt: per token a dict of id, logprob, entropy and the ``top_k`` (id, logprob)."""
    pkg, n = model.pkg, len(prompts)
    longest = max(map(len, prompts)) + n_tokens
    per_seq = -(-longest // page_size)
    pages = Pages(n * per_seq, page_size, n, per_seq)
    caches = [pkg.PagedKVCache(n * per_seq, page_size, model.kv_heads, model.head_dim, cache_dtype)
              for _ in range(model.layers)]
    for s, p in enumerate(prompts):
        pages.grow(s, len(p))
    rows = [(t, s, i) for s, p in enumerate(prompts) for i, t in enumerate(p)]
    logits = model.step(caches, torch.from_numpy(pages.table).cuda(), *(int32(c) for c in zip(*rows)))
    logits = logits[int32(np.cumsum([len(p) for p in prompts]) - 1).long()]  # each prompt's last row
    answers = [[] for _ in prompts]
    for i in range(n_tokens):
        r = pkg.token_logprobs(logits, top_k=top_k)
        token = r.top_ids[:, 0].contiguous()
        for s, (ids, lps, ent) in enumerate(zip(r.top_ids.tolist(), r.top_logprobs.tolist(), r.entropy.tolist())):
            answers[s].append({"id": ids[0], "logprob": lps[0], "entropy": ent, "top": list(zip(ids, lps))})
        if i + 1 == n_tokens:
            break
        at = [len(p) + i for p in prompts]
        for s, p in enumerate(at):
            pages.grow(s, p + 1)
        logits = model.step(caches, torch.from_numpy(pages.table).cuda(), token, int32(list(range(n))), int32(at))
    return answers, caches, pages


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=12)
    ap.add_argument("--cache", choices=("int8", "bfloat16", "float16"), default="int8")
    a = ap.parse_args()
    model = Decoder(load_package())
    prompts = [[1, 5, 9, 2], [7] * 33, [3], list(range(100, 117))]
    answers, _, pages = generate(model, prompts, a.tokens, getattr(torch, a.cache))
    for prompt, answer, held in zip(prompts, answers, pages.held):
        print(f"prompt of {len(prompt)} tokens, {held} pages")
        for t in answer:
            others = ", ".join(f"{i} {p:.2f}" for i, p in t["top"][1:])
            print(f"  {t['id']:5d}  logprob {t['logprob']:7.3f}  entropy {t['entropy']:.3f}  next: {others}")


if __name__ == "__main__":
    main()
