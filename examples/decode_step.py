"""A decode loop over the C-ABI: quantized projections, rotation into a paged
cache, attention over its pages, the gated MLP, the output head and the choice
of a token, for a batch of sequences of different lengths.

    python examples/decode_step.py [--layers 2] [--seqs 8] [--steps 32] [--cache BF16]

Random weights (Q4_K, N(0, 1 / in_features)) at the attention block's sizes of
Llama-3-8B; prompts enter the cache one token a step beside sequences that are
already answering, as a serving batch mixes them.  Device memory and streams
come from PyTorch; every product, norm and choice is the library's.
"""
from __future__ import annotations

import argparse
import ctypes
import os
import sys
import time
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from ocelotl_amd import okq  # noqa: E402

Q4_K = 12
CACHE_TYPES = {"F32": 0, "F16": 1, "BF16": 30, "Q8_0": 8}


@dataclass
class Config:
    hidden: int = 4096
    intermediate: int = 14336
    vocab: int = 128256
    layers: int = 2
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    cache: str = "BF16"
    qk_norm: bool = False
    interleaved: bool = True
    page_tokens: int = 16
    max_tokens: int = 512  # of a sequence
    rope_base: float = 500000.0
    eps: float = 1e-5


@dataclass
class Generated:
    tokens: list
    seconds: float = 0.0


class Weight:
    """[rows, cols] of Q4_K blocks, made on the device."""

    def __init__(self, rows: int, cols: int, seed: int):
        self.rows, self.cols = rows, cols
        f = torch.empty(rows * cols, device="cuda")
        self.data = torch.empty(rows * cols // 256 * 144, dtype=torch.uint8, device="cuda")
        s = torch.cuda.current_stream().cuda_stream
        okq.call("okq_fill_normal", seed, 0, f.numel(), cols ** -0.5, f.data_ptr(), s)
        okq.call("okq_quantize", Q4_K, f.data_ptr(), f.numel(), self.data.data_ptr(), s)


class Layer:
    def __init__(self, c: Config, n_pages: int, seed: int):
        qw, kw = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        self.wq, self.wk, self.wv = (Weight(n, c.hidden, seed + i) for i, n in enumerate((qw, kw, kw)))
        self.wo = Weight(c.hidden, qw, seed + 3)
        self.gate, self.up = (Weight(c.intermediate, c.hidden, seed + 4 + i) for i in range(2))
        self.down = Weight(c.hidden, c.intermediate, seed + 6)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def norm(n):
            return 1 + 0.1 * torch.randn(n, generator=g, device="cuda")
        self.attn_norm, self.mlp_norm = norm(c.hidden), norm(c.hidden)
        self.q_norm, self.k_norm = (norm(c.head_dim), norm(c.head_dim)) if c.qk_norm else (None, None)
        row = c.head_dim // 32 * 34 if c.cache == "Q8_0" else c.head_dim * (4 if c.cache == "F32" else 2)
        page = c.kv_heads * c.page_tokens * row
        self.k, self.v = (torch.empty(n_pages * page, dtype=torch.uint8, device="cuda") for _ in range(2))
        self.pages = okq.KvPages(type=CACHE_TYPES[c.cache], n_pages=n_pages, page_tokens=c.page_tokens,
                                 kv_heads=c.kv_heads, head_dim=c.head_dim, page_stride=page,
                                 head_stride=c.page_tokens * row, token_stride=row, k=self.k.data_ptr(),
                                 v=self.v.data_ptr())


def _ptr(t):
    return None if t is None else t.data_ptr()


class Model:
    def __init__(self, config: Config, seqs: int, seed: int = 1):
        okq.call("okq_init", torch.cuda.current_device())
        c = self.c = config
        self.seqs = seqs
        per_seq = (c.max_tokens + c.page_tokens - 1) // c.page_tokens
        self.layers = [Layer(c, seqs * per_seq, 1000 * (seed + i)) for i in range(c.layers)]
        self.embedding, self.head = Weight(c.vocab, c.hidden, seed + 11), Weight(c.vocab, c.hidden, seed + 12)
        self.final_norm = torch.ones(c.hidden, device="cuda")
        half = c.head_dim // 2
        self.inv_freq = (c.rope_base ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
        # pages are handed out in no order, as a cache in use has them
        order = torch.randperm(seqs * per_seq, generator=torch.Generator().manual_seed(seed))
        self.table_host = order.view(seqs, per_seq).int()
        self.table = self.table_host.cuda()

        def buf(n):
            return torch.empty(seqs, n, device="cuda")
        qw, kw = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        self.x, self.q, self.k, self.v, self.attn = (buf(n) for n in (c.hidden, qw, kw, kw, qw))
        self.y, self.normed, self.g, self.u = (buf(n) for n in (c.hidden, c.hidden, c.intermediate, c.intermediate))
        self.logits = buf(c.vocab)

    def step(self, ids, positions) -> None:
        """One token of every sequence: ids and positions (host lists); leaves the head's logits in self.logits."""
        c, n, s = self.c, self.seqs, torch.cuda.current_stream().cuda_stream
        slots = [int(self.table_host[i, p // c.page_tokens]) * c.page_tokens + p % c.page_tokens
                 for i, p in enumerate(positions)]
        pos = torch.tensor(positions, dtype=torch.int32).cuda()
        slot = torch.tensor(slots, dtype=torch.int64).cuda()
        lengths = pos + 1
        okq.call("okq_get_rows_q", Q4_K, self.embedding.data.data_ptr(), self.embedding.data.numel(), c.hidden, c.vocab,
                 (ctypes.c_uint32 * n)(*ids), n, self.x.data_ptr(), s)
        for l in self.layers:
            self._project_qkv(l, s)
            self.rotate(l, pos, slot, s)
            self.attend(l, lengths, max(positions) + 1, s)
            self._linear(self.attn, l.wo, self.y, s)
            self.x += self.y
            okq.call("okq_rmsnorm", self.x.data_ptr(), n, c.hidden, l.mlp_norm.data_ptr(), c.eps,
                     self.normed.data_ptr(), s)
            okq.call("okq_mlp_gated_silu_q", self.normed.data_ptr(), n, c.hidden, c.intermediate, Q4_K,
                     l.gate.data.data_ptr(), l.gate.data.numel(), Q4_K, l.up.data.data_ptr(), l.up.data.numel(), Q4_K,
                     l.down.data.data_ptr(), l.down.data.numel(), self.g.data_ptr(), self.u.data_ptr(),
                     self.y.data_ptr(), s)
            self.x += self.y
        okq.call("okq_rmsnorm", self.x.data_ptr(), n, c.hidden, self.final_norm.data_ptr(), c.eps,
                 self.normed.data_ptr(), s)
        self._linear(self.normed, self.head, self.logits, s)

    def rotate(self, l: Layer, pos, slot, s: int) -> None:
        """Norm (if the model has it) and rotation of queries and keys; keys and values into the cache."""
        c = self.c
        qw, kw = c.q_heads * c.head_dim, c.kv_heads * c.head_dim
        okq.call("okq_qk_norm_rope", self.q.data_ptr(), qw, self.k.data_ptr(), kw, self.v.data_ptr(), kw, self.seqs,
                 c.q_heads, c.kv_heads, c.head_dim, _ptr(l.q_norm), _ptr(l.k_norm), c.eps, pos.data_ptr(),
                 self.inv_freq.data_ptr(), c.head_dim, int(c.interleaved), self.q.data_ptr(), qw, None, 0,
                 ctypes.byref(l.pages), slot.data_ptr(), s)

    def attend(self, l: Layer, lengths, longest: int, s: int) -> None:
        c = self.c
        qw = c.q_heads * c.head_dim
        okq.call("okq_paged_attention", self.q.data_ptr(), qw, self.seqs, c.q_heads, ctypes.byref(l.pages),
                 self.table.data_ptr(), self.table.shape[1], lengths.data_ptr(), longest, c.head_dim ** -0.5, 0.0, 0,
                 self.attn.data_ptr(), qw, None, s)

    def choose(self, hist, seen, start, rep, pres, best, s: int) -> None:
        """Penalties on self.logits, in place, and every sequence's token."""
        c = self.c
        okq.call("okq_logits_process", self.logits.data_ptr(), c.vocab, self.seqs, c.vocab, hist.data_ptr(),
                 hist.shape[1], seen.data_ptr(), start.data_ptr(), rep.data_ptr(), None, pres.data_ptr(), None, None, 0,
                 None, None, 0, self.logits.data_ptr(), c.vocab, best.data_ptr(), s)

    def _project_qkv(self, l: Layer, s: int) -> None:
        w, out = (l.wq, l.wk, l.wv), (self.q, self.k, self.v)
        okq.call("okq_rmsnorm_linear_q_multi", self.x.data_ptr(), self.seqs, self.c.hidden, l.attn_norm.data_ptr(),
                 self.c.eps, Q4_K, 3, (ctypes.c_void_p * 3)(*[m.data.data_ptr() for m in w]),
                 (ctypes.c_uint64 * 3)(*[m.data.numel() for m in w]), (ctypes.c_int64 * 3)(*[m.rows for m in w]), None,
                 (ctypes.c_void_p * 3)(*[t.data_ptr() for t in out]), s)

    def _linear(self, x, w: Weight, out, s: int) -> None:
        okq.call("okq_linear_out_by_in_q", x.data_ptr(), self.seqs, w.cols, Q4_K, w.data.data_ptr(), w.data.numel(),
                 w.rows, None, out.data_ptr(), s)

    def generate(self, prompts, steps: int, repetition: float = 1.1, presence: float = 0.0) -> Generated:
        """Greedy answers of `steps` tokens each.  A sequence's prompt goes in
        a token a step; once it has all of it, each step's choice is its next token."""
        c, n = self.c, self.seqs
        tokens = [list(p) for p in prompts]
        total = [len(p) + steps for p in prompts]
        assert len(prompts) == n and max(total) <= c.max_tokens and all(prompts)
        hist = torch.zeros(n, c.max_tokens, dtype=torch.int32, device="cuda")
        for i, p in enumerate(prompts):
            hist[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        start = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
        rep = torch.full((n,), repetition, device="cuda")
        pres = torch.full((n,), presence, device="cuda")
        best = torch.empty(n, dtype=torch.int32, device="cuda")
        got = Generated(tokens)
        torch.cuda.synchronize()
        began = time.perf_counter()
        for t in range(max(total) - 1):
            # a finished sequence repeats its last token in place
            at = [min(t, total[i] - 2) for i in range(n)]
            self.step([tokens[i][at[i]] for i in range(n)], at)
            seen = torch.tensor([max(a + 1, len(p)) for a, p in zip(at, prompts)], dtype=torch.int32).cuda()
            self.choose(hist, seen, start, rep, pres, best, torch.cuda.current_stream().cuda_stream)
            chosen = best.tolist()
            for i in range(n):
                if len(tokens[i]) == t + 1 and len(tokens[i]) < total[i]:
                    tokens[i].append(chosen[i])
                    hist[i, t + 1] = chosen[i]
        torch.cuda.synchronize()
        got.seconds = time.perf_counter() - began
        return got


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--cache", choices=sorted(CACHE_TYPES), default="BF16")
    a = ap.parse_args()
    model = Model(Config(layers=a.layers, cache=a.cache), a.seqs)
    prompts = [[(7 * i + j) % model.c.vocab for j in range(1 + 3 * i)] for i in range(a.seqs)]
    model.generate(prompts, 2)
    got = model.generate(prompts, a.steps)
    steps = max(len(t) for t in got.tokens) - 1
    print(f"{a.seqs} sequences, {a.layers} layers, {a.cache} cache: {steps} steps, {got.seconds / steps * 1e6:.0f} us a step")
    for i, (p, t) in enumerate(zip(prompts, got.tokens)):
        print(f"  {i}: prompt of {len(p)}, answer {t[len(p):][:8]} ...")


if __name__ == "__main__":
    main()
