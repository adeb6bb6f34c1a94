"""Several sampled continuations of one prompt, decoded as one batch over a paged cache.

Runs the paged serving operators together: the prompt is read once, its sequence is forked (the forks share
the prompt's pages until they write), and every step rotates and appends the new token's keys and values
(rope_append_device), attends over the pages (paged_attn_device) and draws the next ids from given uniform
numbers (sample_device); copy_pages_device copies a shared page before it is written.  The Q4 matrices go
through gemm_q4_device, the rest of the layer (norms, SiLU) through torch.

    python examples/paged_sampling.py [config] [--forks 8] [--new 64] [--temperature 0.8] [--cache bf16]

``config`` names a shape of the package's CONFIGS (llama ones); weights are seeded random numbers.
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
P = importlib.import_module("microllm-lab_b200")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class PagedDecoder:
    """A llama-shaped Q4 model over one page pool per layer.  ``step`` runs one new token of each sequence."""

    def __init__(self, data, n_pages: int, page_len: int = 16, cache: str = "f32", max_seqs: int = 16):
        self.bundle = b = P.parse_pgw(data)
        c = self.cfg = b.cfg
        self.d, self.heads, self.kv_heads = c["dModel"], c["nHeads"], c["nKvHeads"]
        self.dim = self.d // self.heads
        dev = lambda a: torch.from_numpy(np.array(a)).cuda()
        self.q4 = {n: (dev(b.u8(n)), dev(b.scales(n)), *t["shape"]) for n, t in b.tensors.items() if t["storage"] == "q4"}
        self.gain = {n: dev(b.f32(n)) for n, t in b.tensors.items() if t["storage"] == "f32"}
        self.embed = dev(b.dequant("lm_head"))
        rope_dim = int(self.dim * c["ropePct"]) // 2 * 2
        self.cos, self.sin = (dev(a) for a in P.rope_tables(c["maxSeqLen"], rope_dim, c["ropeTheta"]))
        self.rope_dim = rope_dim
        self.pages = P.PageTable(n_pages, page_len)
        shape = (c["nLayers"], n_pages, self.kv_heads, page_len, self.dim)
        self.k, self.v = (torch.zeros(shape, dtype=TYPES[cache], device="cuda") for _ in range(2))
        self.kv = [P.paged_kv(self.k[i].data_ptr(), self.v[i].data_ptr(), cache, n_pages, page_len, self.kv_heads, self.dim)
                   for i in range(c["nLayers"])]
        self.max_seqs = max_seqs
        self.ws = torch.zeros(P.paged_attn_workspace(max_seqs, self.heads, self.dim), dtype=torch.uint8, device="cuda")

    def matmul(self, name: str, x: torch.Tensor) -> torch.Tensor:
        packed, scales, rows, cols = self.q4[name]
        x = x.contiguous()
        y = torch.empty(x.shape[0], rows, device="cuda")
        P.gemm_q4_device(packed.data_ptr(), scales.data_ptr(), x.data_ptr(), y.data_ptr(), rows, cols, x.shape[0])
        return y

    def norm(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * self.gain[name]

    def copy(self, moves) -> None:
        """Page copies that the bookkeeping asked for, in every layer."""
        if moves[0]:
            P.copy_pages_device(self.kv[0], *moves, n_layers=len(self.kv), layer_stride=self.k.stride(0))

    def step(self, seqs, ids: torch.Tensor) -> torch.Tensor:
        """Append one token to each of ``seqs`` (each once) and return the logits after it [len(seqs)][vocab].  Raises
        MemoryError, changing nothing, when the pool has too few free pages."""
        n = len(seqs)
        if n > self.max_seqs:
            raise ValueError(f"{n} sequences in a decoder made for {self.max_seqs}")
        if any(self.pages.length(s) >= self.cos.shape[0] for s in seqs):
            raise ValueError(f"a sequence holds its {self.cos.shape[0]} positions")
        pos = torch.tensor([self.pages.length(s) for s in seqs], dtype=torch.int32, device="cuda")
        self.copy(self.pages.grow_all(seqs))
        table = torch.from_numpy(self.pages.table(seqs)).cuda()
        length = pos + 1
        known = (ids >= 0) & (ids < self.embed.shape[0])  # an id that is none makes its own sequence NaN
        x = self.embed[ids.long().where(known, 0)].where(known[:, None], float("nan"))
        q = torch.empty(n, self.d, device="cuda")
        att = torch.empty(n, self.d, device="cuda")
        for i, kv in enumerate(self.kv):
            qkv = self.matmul(f"blocks.{i}.attn.qkv", self.norm(f"blocks.{i}.norm1", x))
            P.rope_append_device(kv, "f32", qkv.data_ptr(), qkv.stride(0), n, self.heads, 0, pos.data_ptr(), table.data_ptr(), n,
                                 table.stride(0), self.cos.data_ptr(), self.sin.data_ptr(), self.cos.shape[0], self.rope_dim,
                                 q.data_ptr(), q.stride(0))
            P.paged_attn_device(kv, "f32", q.data_ptr(), q.stride(0), n, self.heads, length.data_ptr(), table.data_ptr(),
                                table.stride(0), self.dim ** -0.5, att.data_ptr(), att.stride(0), self.ws.data_ptr(),
                                self.ws.numel())
            x = x + self.matmul(f"blocks.{i}.attn.proj", att)
            h = self.norm(f"blocks.{i}.norm2", x)
            x = x + self.matmul(f"blocks.{i}.mlp.w2",
                                torch.nn.functional.silu(self.matmul(f"blocks.{i}.mlp.w1", h)) * self.matmul(f"blocks.{i}.mlp.w3", h))
        return self.matmul("lm_head", self.norm("norm_f", x))

    def read(self, prompt) -> tuple[int, torch.Tensor]:
        """A new sequence that holds the prompt, and the logits after it."""
        prompt = [int(t) for t in prompt]
        if not 0 < len(prompt) <= self.cos.shape[0]:
            raise ValueError(f"a prompt of {len(prompt)} ids, not 1 to {self.cos.shape[0]}")
        if not all(0 <= t < self.embed.shape[0] for t in prompt):
            raise ValueError("a prompt id outside the vocabulary")
        s = self.pages.new()
        try:
            for t in prompt:
                logits = self.step([s], torch.tensor([t], device="cuda"))
        except Exception:
            self.pages.free(s)
            raise
        return s, logits


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None):
    """One id per row and its log-probability; the settings are one number each, or None."""
    n, v = logits.shape
    per_row = [None if a is None else torch.full((n,), a, dtype=t, device="cuda")
               for a, t in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32))]
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    logprob = torch.empty(n, device="cuda")
    P.sample_device("f32", logits.data_ptr(), logits.stride(0), n, v, u.data_ptr(), ids.data_ptr(), logprob.data_ptr(),
                    temperature_ptr=per_row[0].data_ptr() if per_row[0] is not None else 0,
                    top_k_ptr=per_row[1].data_ptr() if per_row[1] is not None else 0,
                    top_p_ptr=per_row[2].data_ptr() if per_row[2] is not None else 0,
                    min_p_ptr=per_row[3].data_ptr() if per_row[3] is not None else 0)
    return ids, logprob


def continuations(model: PagedDecoder, prompt, forks: int, new: int, seed: int = 0, **settings):
    """``forks`` continuations of ``new`` ids each, with their log-probabilities, as [forks][new] tensors."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    first, logits = model.read(prompt)
    seqs = [first] + [model.pages.fork(first) for _ in range(forks - 1)]
    logits = logits.expand(forks, -1).contiguous()
    ids, logprobs = [], []
    try:
        for i in range(new):
            t, lp = sample(logits, torch.rand(forks, generator=gen, device="cuda"), **settings)
            ids.append(t)
            logprobs.append(lp)
            if i + 1 < new:
                logits = model.step(seqs, t)
    finally:
        for s in seqs:
            model.pages.free(s)
    return torch.stack(ids, 1), torch.stack(logprobs, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("config", nargs="?", default="smollm2-135m")
    ap.add_argument("--forks", type=int, default=8)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=64, help="seeded random prompt ids")
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--cache", choices=list(TYPES), default="bf16")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    data = P.synthetic_pgw(a.config, a.seed)
    pages = -(-a.prompt // 16) + a.forks * (-(-a.new // 16) + 1)
    model = PagedDecoder(data, pages, 16, a.cache, max(a.forks, 1))
    prompt = P.seeded_prompt(a.prompt, model.cfg["vocabSize"], a.seed)
    ids, logprobs = continuations(model, prompt, a.forks, a.new, a.seed, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p,
                                  min_p=a.min_p)
    for row, lp in zip(ids.tolist(), logprobs.sum(1).tolist()):
        print(f"{lp:9.2f}  {row}")


if __name__ == "__main__":
    main()
