"""The sparse layer as programs run it (needs an MI355X): the C++ mirror's chain
(tests/cpp/test_expert_layer.cpp), and examples/decode_step.py with experts,
each layer's mix checked against its definition in 64 bits.

Bounds: the sum of two f32 values is off by u = 2^-24 of it.  Weights of the
experts are held to 2^-18 of themselves: logits of rows of 256 values, whose
f32 norms are off by some 2^-20, through an exponential of logits around 1.  The
experts' results are held to 2^-13 of each row's largest: two products behind
one another with 2^-21 of sums of magnitudes some 30 times the result.
"""
import importlib.util
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
Q4_K = 12


def test_cpp_chain():
    path = os.path.join(ROOT, "tests", "cpp", "_build", "test_expert_layer")
    assert os.path.exists(path), f"{path} is not built: run __graft_entry__.build() (make -C tests/cpp)"
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.fixture(scope="module")
def example():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location("decode_step", os.path.join(ROOT, "examples", "decode_step.py"))
    module = importlib.util.module_from_spec(spec)
    import sys
    sys.modules["decode_step"] = module
    spec.loader.exec_module(module)
    return module


def _values(example, w):
    import torch
    out = torch.empty(w.rows * w.cols, device="cuda")
    example.okq.call("okq_dequantize", Q4_K, w.data.data_ptr(), out.numel(), out.data_ptr(),
                     torch.cuda.current_stream().cuda_stream)
    return out.view(w.rows, w.cols).double()


def test_example_mixes_by_the_definitions(example):
    """Three sequences of different prompts through two sparse layers."""
    import torch
    config = example.Config(hidden=256, vocab=1000, layers=2, q_heads=4, kv_heads=2, head_dim=64, page_tokens=8,
                            max_tokens=32, experts=12, top_k=3, expert_intermediate=512)

    class Checked(example.Model):
        checks = 0

        def mix(self, l, s):
            c = self.c
            x, y = self.x.double(), self.y.double()
            super().mix(l, s)
            total = x + y
            assert bool(((self.x.double() - total).abs() <= U * total.abs()).all())
            n = total / (total.square().mean(1, keepdim=True) + c.eps).sqrt() * l.mlp_norm.double()
            p = torch.softmax(n @ l.router.double().t().contiguous(), 1)
            ids = self.ids.long()
            chosen = p.gather(1, ids)
            rest = p.scatter(1, ids, 0.0)
            assert bool((chosen.amin(1) >= rest.amax(1) * (1 - 2.0 ** -18)).all())
            w = chosen / chosen.sum(1, keepdim=True)
            assert bool(((self.shares.double() - w).abs() <= 2.0 ** -18 * w).all())
            gate, up, down = (_values(example, m).view(c.experts, -1, m.cols) for m in (l.gate, l.up, l.down))
            want = torch.zeros_like(n)
            for r in range(len(n)):
                for j in range(c.top_k):
                    e = int(ids[r, j])
                    g = gate[e] @ n[r]
                    want[r] += w[r, j] * (down[e] @ (g * torch.sigmoid(g) * (up[e] @ n[r])))
            assert bool(((self.y.double() - want).abs() <= 2.0 ** -13 * want.abs().amax(1, keepdim=True)).all())
            self.checks += 1

    model = Checked(config, seqs=3, seed=7)
    prompts = [[5, 17, 900], [3], [999, 0, 1, 2, 3, 4, 5]]
    got = model.generate(prompts, steps=6)
    assert all(len(t) == len(p) + 6 and t[:len(p)] == p for t, p in zip(got.tokens, prompts))
    assert model.checks == (max(len(t) for t in got.tokens) - 1) * config.layers


def test_example_runs_from_the_command_line():
    r = subprocess.run(["python3", os.path.join(ROOT, "examples", "decode_step.py"), "--layers", "1", "--seqs", "3",
                        "--steps", "3", "--experts", "16"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "us a step" in r.stdout, r.stdout + r.stderr
