"""The decode step as programs run it (needs an MI355X): the C++ mirror's
chain (tests/cpp/test_decode_step.cpp), and examples/decode_step.py with each
operator's outputs held against its definition in f64 on the same inputs.

(The chain as a whole is no measure of them: where a projection quantizes its
input, a difference of one f32 step turns into 2e-5 of its output and 3e-4 a
layer later.)  Bounds, u = 2^-24: rotation 16u (|a| + |b|); scores 8u scale
sum |q K|, outputs (2e + 8u + 8u sqrt(T)) max |V|; logits 5u of their parts.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


def test_cpp_mirror_decode_step():
    path = os.path.join(ROOT, "tests", "cpp", "_build", "test_decode_step")
    assert os.path.exists(path), f"{path} is not built: run __graft_entry__.build() (make -C tests/cpp)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture(scope="module")
def example():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_step
    return decode_step


def checked_model(example):
    import torch

    class Checked(example.Model):
        checks = 0

        def rows(self, l, i, n):
            """Keys and values of sequence i's first n tokens, as the cache holds them, f64 [n, kv heads, d]."""
            c = self.c
            out = []
            for raw in (l.k, l.v):
                p = raw.view(l.pages.n_pages, c.kv_heads, c.page_tokens, -1).cpu()
                r = torch.stack([p[int(self.table_host[i, t // c.page_tokens]), :, t % c.page_tokens] for t in range(n)])
                if c.cache == "Q8_0":
                    b = r.reshape(n, c.kv_heads, -1, 34)
                    r = (b[..., :2].contiguous().view(torch.float16).double() *
                         b[..., 2:].contiguous().view(torch.int8).double()).reshape(n, c.kv_heads, -1)
                else:
                    r = r.contiguous().view({"F32": torch.float32, "F16": torch.float16,
                                             "BF16": torch.bfloat16}[c.cache]).double()
                out.append(r)
            return out

        def rotate(self, l, pos, slot, s):
            c = self.c
            q, k, v = (t.cpu().double().view(self.seqs, -1, c.head_dim) for t in (self.q, self.k, self.v))
            super().rotate(l, pos, slot, s)
            ang = (pos.cpu().double()[:, None] * self.inv_freq.cpu().double())[:, None]
            i = torch.arange(c.head_dim // 2)
            a, b = (2 * i, 2 * i + 1) if c.interleaved else (i, i + c.head_dim // 2)

            def want(x, w):
                if w is not None:
                    x = x / (x.square().mean(-1, keepdim=True) + c.eps).sqrt() * w.cpu().double()
                y, size = torch.empty_like(x), torch.empty_like(x)
                y[..., a] = x[..., a] * ang.cos() - x[..., b] * ang.sin()
                y[..., b] = x[..., b] * ang.cos() + x[..., a] * ang.sin()
                size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
                return y, 16 * U * size

            y, tol = want(q, l.q_norm)
            assert ((self.q.cpu().double().view_as(y) - y).abs() <= tol).all()
            y, tol = want(k, l.k_norm)
            # half a step of the cache's type; a Q8_0 code and half a step of its f16 scale
            step = {"F32": U, "F16": 2.0 ** -11, "BF16": 2.0 ** -8}.get(c.cache, 0.0)

            def half(x):
                if c.cache != "Q8_0":
                    return step * x.abs()
                top = x.reshape(self.seqs, c.kv_heads, -1, 32).abs().amax(-1, keepdim=True)
                return (top * (0.5 / 127 + 2.0 ** -11)).expand(-1, -1, -1, 32).reshape_as(x)

            for j, p in enumerate(pos.tolist()):
                K, V = self.rows(l, j, p + 1)
                assert ((K[p] - y[j]).abs() <= half(y)[j] * (1 + 1e-5) + 2 * tol[j]).all()
                assert ((V[p] - v[j]).abs() <= half(v)[j] * (1 + 1e-5)).all()
            self.checks += 1

        def attend(self, l, lengths, longest, s):
            c = self.c
            super().attend(l, lengths, longest, s)
            scale, group = c.head_dim ** -0.5, c.q_heads // c.kv_heads
            for i, n in enumerate(lengths.tolist()):
                K, V = (x.repeat_interleave(group, 1) for x in self.rows(l, i, n))
                prod = K * self.q[i].cpu().double().view(-1, c.head_dim)
                p = torch.softmax(prod.sum(-1) * scale, 0)
                e = 8 * U * scale * prod.abs().sum(-1).amax()
                want = (p[..., None] * V).sum(0)
                got = self.attn[i].cpu().double().view_as(want)
                assert ((got - want).abs() <= (2 * e + 8 * U * (1 + n ** 0.5)) * V.abs().amax()).all()
            self.checks += 1

        def choose(self, hist, seen, start, rep, pres, best, s):
            y = self.logits.cpu().double()
            super().choose(hist, seen, start, rep, pres, best, s)
            size = 2 * y.abs()
            for i, (n, b) in enumerate(zip(seen.tolist(), start.tolist())):
                h, r, w = hist[i].tolist(), rep[i].item(), pres[i].item()
                for j in set(h[:n]):
                    y[i, j] = y[i, j] / r if y[i, j] > 0 else y[i, j] * r
                    size[i, j] *= r
                for j in set(h[b:n]):
                    y[i, j] -= w
                    size[i, j] += w
            got = self.logits.cpu()
            assert ((got.double() - y).abs() <= 5 * U * size).all()
            assert best.tolist() == got.argmax(-1).tolist()
            self.checks += 1

    return Checked


@pytest.mark.parametrize("cache,norm,interleaved", [("BF16", False, True), ("F16", True, False), ("F32", True, True),
                                                    ("Q8_0", False, False)])
def test_example_decodes_by_the_definitions(example, cache, norm, interleaved):
    """Three sequences of different prompts, nine answered tokens each."""
    config = example.Config(hidden=256, intermediate=512, vocab=1000, layers=2, q_heads=4, kv_heads=2, head_dim=64,
                            cache=cache, qk_norm=norm, interleaved=interleaved, page_tokens=8, max_tokens=32)
    prompts = [[5, 17, 900], [3], [999, 0, 1, 2, 3, 4, 5]]
    model = checked_model(example)(config, seqs=3, seed=7)
    got = model.generate(prompts, steps=9, repetition=1.2, presence=0.25)
    assert all(len(t) == len(p) + 9 and t[:len(p)] == p for t, p in zip(got.tokens, prompts))
    steps = max(len(t) for t in got.tokens) - 1
    assert model.checks == steps * (2 * config.layers + 1)
