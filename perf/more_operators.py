"""The operators around and inside a layer's experts, and the work that they
are timed and compared on.

  norm    okq_residual_norm: the norm behind a block, its gate and scale, the
          residual sum, and the norm ahead of the next block
  route   okq_moe_route: the router's product, scores, groups, the choice of
          experts and their weights
  moe     okq_moe_mlp_q: the gated MLP of every token's experts over stacked
          GGUF tensors, and the weighted sum of their results

Hidden sizes are the Llama-3-8B block's 4096 (with its MLP of 14336) and the
Gemma4 embedding's 2560, with generic ones around them; numbers of experts are
generic.  Activations are f32, as the quantized projections read and write
them; expert weights are Q4_K, Q5_K, Q6_K or Q8_0.
"""
import math

import torch

own = False

F32, F16, BF16 = 0, 1, 30
Q8_0, Q4_K, Q5_K, Q6_K = 8, 12, 13, 14
FLOAT = {"F32": (F32, torch.float32), "F16": (F16, torch.float16), "BF16": (BF16, torch.bfloat16)}
QUANT = {"Q8_0": (Q8_0, 32, 34), "Q4_K": (Q4_K, 256, 144), "Q5_K": (Q5_K, 256, 176), "Q6_K": (Q6_K, 256, 210)}
EPS = 1e-6


def listed():
    return [
        # one token between two blocks: only latency counts
        dict(name="norm_token", op="norm", rows=1, hidden=4096, post=True, pre=True, gate="none", out="F32"),
        # a serving batch, a gate for every channel, bf16 rows for the next projections
        dict(name="norm_batch", op="norm", rows=48, hidden=2560, post=True, pre=True, gate="channel", out="BF16"),
        # a prompt of 4096 tokens
        dict(name="norm_prompt", op="norm", rows=4096, hidden=4096, post=True, pre=True, gate="none", out="F32"),
        # gates of every token and channel, a width that is no power of two
        dict(name="norm_gated", op="norm", rows=1531, hidden=1111, post=False, pre=True, gate="token", out="F16"),
        # one token of a chat
        dict(name="route_token", op="route", rows=1, hidden=2048, experts=128, top_k=8, score="softmax", groups=1,
             top_groups=1, group_best=1, balance=False, renormalise=True, weight="F32"),
        # a serving batch: sigmoid scores, a bias for balance, groups of experts
        dict(name="route_groups", op="route", rows=61, hidden=2560, experts=256, top_k=8, score="sigmoid", groups=8,
             top_groups=4, group_best=2, balance=True, renormalise=True, weight="F32"),
        # a prompt of 4096 tokens
        dict(name="route_prompt", op="route", rows=4096, hidden=2048, experts=128, top_k=8, score="softmax", groups=1,
             top_groups=1, group_best=1, balance=False, renormalise=True, weight="BF16"),
        # one token of a chat: the weights of its eight experts, once
        dict(name="moe_token", op="moe", rows=1, hidden=2048, inner=768, experts=128, top_k=8, gate_up="Q4_K",
             down="Q6_K", padded=False),
        # a serving batch with padded rows: nearly every expert has a few tokens
        dict(name="moe_serving", op="moe", rows=48, hidden=2048, inner=768, experts=128, top_k=8, gate_up="Q4_K",
             down="Q4_K", padded=True),
        # few wide experts, a small batch
        dict(name="moe_wide", op="moe", rows=13, hidden=4096, inner=14336, experts=8, top_k=2, gate_up="Q4_K",
             down="Q6_K", padded=False),
        # a short prompt, rows that are no multiple of 256 values
        dict(name="moe_q8", op="moe", rows=333, hidden=2560, inner=1440, experts=31, top_k=6, gate_up="Q8_0",
             down="Q8_0", padded=False),
        # a prompt of 4096 tokens
        dict(name="moe_prompt", op="moe", rows=4096, hidden=2048, inner=768, experts=128, top_k=8, gate_up="Q4_K",
             down="Q6_K", padded=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "route", "moe", "moe"])
    if op == "norm":
        hidden = spread(64, 16384)
        post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
        return dict(op=op, rows=max(1, min(spread(1, 4096), 4096 * 4096 // hidden)), hidden=hidden, post=post, pre=pre,
                    gate=rng.choice(["none", "none", "channel", "token"]), out=rng.choice(["F32", "F32", "BF16", "F16"]))
    if op == "route":
        groups = rng.choice([1, 1, 1, 4, 8])
        experts = groups * (spread(4, 32) if groups > 1 else spread(4, 256))
        top_groups = rng.randint(1, groups)
        hidden = spread(128, 4096)
        return dict(op=op, rows=max(1, min(spread(1, 4096), 4096 * 2048 * 128 // (hidden * experts))), hidden=hidden,
                    experts=experts, top_k=rng.randint(1, min(10, experts // groups * top_groups)),
                    score=rng.choice(["softmax", "sigmoid"]), groups=groups, top_groups=top_groups,
                    group_best=rng.choice([1, 2]), balance=rng.random() < 0.5, renormalise=rng.random() < 0.7,
                    weight=rng.choice(["F32", "F32", "F16", "BF16"]))
    gate_up = rng.choice(["Q4_K", "Q4_K", "Q5_K", "Q6_K", "Q8_0"])
    down = rng.choice(["Q4_K", "Q5_K", "Q6_K", "Q6_K", "Q8_0"])
    hidden = 256 * spread(2, 16) if gate_up != "Q8_0" else 32 * spread(16, 128)
    inner = 256 * spread(1, 12) if down != "Q8_0" else 32 * spread(8, 96)
    top_k = rng.randint(1, 8)
    experts = max(top_k, min(spread(4, 128), 128 * 2048 * 768 // (hidden * inner)))
    rows = max(1, min(spread(1, 4096), 4096 * 8 * 2048 * 768 // (top_k * hidden * inner)))
    return dict(op=op, rows=rows, hidden=hidden, inner=inner, experts=experts, top_k=top_k, gate_up=gate_up, down=down,
                padded=rng.random() < 0.3)


# ---- inputs -----------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, hidden):
    """Rows of a residual stream: a few channels stand out."""
    x = _normal(gen, rows, hidden)
    loud = torch.randperm(hidden, generator=gen, device="cuda")[:max(1, hidden // 256)]
    x[:, loud] *= 8.0
    return x


def _codes(gen, n, mean, deviation, lo, hi):
    return (torch.randn(n, generator=gen, device="cuda") * deviation + mean).round_().clamp_(lo, hi).to(torch.int16)


def _halves(v):
    """f32 [n] as the two bytes of their f16 values [n, 2]."""
    return v.to(torch.float16).view(torch.uint8).view(-1, 2)


def _blocks(gen, kind, n, columns):
    """n values of normal weights of deviation columns^-0.5 as GGUF blocks."""
    _, elems, size = QUANT[kind]
    nb, std = n // elems, columns ** -0.5
    vary = torch.rand(nb, generator=gen, device="cuda").mul_(0.6).add_(0.7)
    if kind == "Q8_0":
        q = _codes(gen, n, 0.0, 42.0, -127, 127).to(torch.int8).view(nb, 32)
        return torch.cat([_halves(vary * (std / 42.0)), q.view(torch.uint8)], 1)
    if kind == "Q6_K":
        q = _codes(gen, n, 32.0, 10.0, 0, 63).view(nb, 2, 4, 32)  # half, quarter, value
        low = (q[:, :, :2] & 15) | ((q[:, :, 2:] & 15) << 4)
        high = (q >> 4) << torch.tensor([0, 2, 4, 6], device="cuda", dtype=torch.int16).view(1, 1, 4, 1)
        scale = torch.randint(64, 128, (nb, 16), generator=gen, device="cuda")
        scale = scale * (1 - 2 * torch.randint(0, 2, (nb, 16), generator=gen, device="cuda"))
        return torch.cat([low.reshape(nb, 128).to(torch.uint8), high.sum(2).reshape(nb, 64).to(torch.uint8),
                          scale.to(torch.int8).view(torch.uint8), _halves(vary * (std / 960.0))], 1)
    five = kind == "Q5_K"
    q = _codes(gen, n, 15.5 if five else 7.5, 5.6 if five else 2.8, 0, 31 if five else 15).view(nb, 4, 2, 32)
    sc = torch.randint(32, 64, (nb, 8), generator=gen, device="cuda")
    m = (sc + torch.randint(-3, 4, (nb, 8), generator=gen, device="cuda")).clamp_(0, 63)
    s6 = torch.cat([sc[:, :4] | ((sc[:, 4:] >> 4) << 6), m[:, :4] | ((m[:, 4:] >> 4) << 6),
                    (sc[:, 4:] & 15) | ((m[:, 4:] & 15) << 4)], 1).to(torch.uint8)
    d = vary * (std / (48.0 * (5.6 if five else 2.8)))
    parts = [_halves(d), _halves(d * (15.5 if five else 7.5)), s6]
    if five:
        bit = torch.arange(8, device="cuda", dtype=torch.int16).view(1, 4, 2, 1)
        parts.append((((q >> 4) & 1) << bit).sum((1, 2)).to(torch.uint8))
    parts.append(((q[:, :, 0] & 15) | ((q[:, :, 1] & 15) << 4)).reshape(nb, 128).to(torch.uint8))
    return torch.cat(parts, 1)


def _stack(gen, kind, experts, rows, columns):
    """[experts, rows, bytes of a row] of a stacked tensor, some experts at a time."""
    _, elems, size = QUANT[kind]
    w = torch.empty(experts, rows, columns // elems * size, dtype=torch.uint8, device="cuda")
    some = max(1, (1 << 25) // (rows * columns))
    for e in range(0, experts, some):
        part = w[e:e + some]
        part.copy_(_blocks(gen, kind, part.shape[0] * rows * columns, columns).view(part.shape))
    return w


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    r, h = case["rows"], case["hidden"]
    s = {"x": _activations(gen, r, h)}
    if case["op"] == "norm":
        s["branch"] = _normal(gen, r, h).mul_(0.5)
        s["post"] = _normal(gen, h).mul_(0.2).add_(1.0) if case["post"] else None
        s["pre"] = _normal(gen, h).mul_(0.2).add_(1.0) if case["pre"] else None
        s["gate"] = {"none": None, "channel": (1, h), "token": (r, h)}[case["gate"]]
        if s["gate"]:
            s["gate"] = _normal(gen, *s["gate"]).mul_(0.5)
        return s
    e, k = case["experts"], case["top_k"]
    if case["op"] == "route":
        # popular experts have larger weight rows
        w = _normal(gen, e, h).mul_(1.5 * h ** -0.5) * torch.rand(e, 1, generator=gen, device="cuda").add_(0.5)
        s["w"] = w.to(FLOAT[case["weight"]][1])
        s["balance"] = _normal(gen, e).mul_(0.1) if case["balance"] else None
        return s
    # what a router gives: some experts more popular than others, weights that sum to 1
    logits = _normal(gen, r, e) + _normal(gen, 1, e).mul_(0.5)
    top = logits.topk(k, dim=1)
    s["ids"] = top.indices.to(torch.int32)
    s["weights"] = torch.softmax(top.values, 1).contiguous()
    if case["padded"]:  # rows of a batch that hold no token: the last ones and one between
        s["ids"][r - r // 5:] = -1
        s["ids"][r // 2] = -1
    n = case["inner"]
    s["gate_w"], s["up_w"] = _stack(gen, case["gate_up"], e, n, h), _stack(gen, case["gate_up"], e, n, h)
    s["down_w"] = _stack(gen, case["down"], e, h, n)
    return s


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    r, h = case["rows"], case["hidden"]
    if case["op"] == "norm":
        s["sum"] = torch.empty(r, h, device="cuda")
        s["normed"] = torch.empty(r, h, device="cuda", dtype=FLOAT[case["out"]][1]) if case["pre"] else None
    elif case["op"] == "route":
        s["ids"] = torch.empty(r, case["top_k"], device="cuda", dtype=torch.int32)
        s["weights"] = torch.empty(r, case["top_k"], device="cuda")
        s["logits"] = torch.empty(r, case["experts"], device="cuda")
    else:
        s["out"] = torch.empty(r, h, device="cuda")
    torch.cuda.synchronize()
    return s


def _results(s):
    op = s["case"]["op"]
    if op == "norm":
        return [s["sum"]] + ([] if s["normed"] is None else [s["normed"]])
    return [s["ids"], s["weights"], s["logits"]] if op == "route" else [s["out"]]


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        from ocelotl_amd import okq
        name, args = state["call"]
        okq.call(name, *args, torch.cuda.current_stream().cuda_stream)
        return _results(state)
    return {"norm": _plain_norm, "route": _plain_route, "moe": _plain_moe}[state["case"]["op"]](state)


# ---- the framework's calls ----------------------------------------------------

BRANCH_SCALE, RESIDUAL_SCALE, ROUTE_SCALE = 0.75, 1.125, 2.5


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(s):
    case = s["case"]
    r, h = case["rows"], case["hidden"]
    if case["op"] == "norm":
        return "okq_residual_norm", (
            _ptr(s["x"]), h, _ptr(s["branch"]), h, r, h, _ptr(s["post"]), _ptr(s["gate"]),
            h if case["gate"] == "token" else 0, BRANCH_SCALE, RESIDUAL_SCALE, _ptr(s["pre"]), EPS, _ptr(s["sum"]), h,
            _ptr(s["normed"]), FLOAT[case["out"]][0], h)
    e, k = case["experts"], case["top_k"]
    if case["op"] == "route":
        return "okq_moe_route", (
            _ptr(s["x"]), h, r, h, FLOAT[case["weight"]][0], _ptr(s["w"]), e, None, int(case["score"] == "sigmoid"),
            _ptr(s["balance"]), case["groups"], case["top_groups"], case["group_best"], k, int(case["renormalise"]),
            ROUTE_SCALE, _ptr(s["ids"]), _ptr(s["weights"]), _ptr(s["logits"]))
    return "okq_moe_mlp_q", (
        _ptr(s["x"]), h, r, h, case["inner"], e, k, _ptr(s["ids"]), _ptr(s["weights"]), QUANT[case["gate_up"]][0],
        _ptr(s["gate_w"]), s["gate_w"].numel(), _ptr(s["up_w"]), s["up_w"].numel(), QUANT[case["down"]][0],
        _ptr(s["down_w"]), s["down_w"].numel(), _ptr(s["out"]), h)


# ---- plain forms ----------------------------------------------------------------

def _plain_rms(x, w):
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w


def _plain_norm(s):
    b = s["branch"] if s["post"] is None else _plain_rms(s["branch"], s["post"])
    if s["gate"] is not None:
        b = b * s["gate"]
    total = s["x"] * RESIDUAL_SCALE + b * BRANCH_SCALE
    if s["pre"] is None:
        return [total]
    return [total, _plain_rms(total, s["pre"]).to(FLOAT[s["case"]["out"]][1])]


def _plain_choice(case, score, select):
    """ids and scores of the chosen experts, the larger selection score first, ties to the lowest index."""
    if case["groups"] > 1:
        g = select.unflatten(1, (case["groups"], -1))
        best = torch.sort(g, dim=2, descending=True).values[:, :, :case["group_best"]].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        select = torch.where(kept[:, :, None], g, -math.inf).flatten(1)
    ids = torch.sort(select, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    return ids, score.gather(1, ids)


def _plain_route(s):
    # in 64 bits: the choice is between scores that may lie next to each other
    case = s["case"]
    logits = torch.matmul(s["x"].double(), s["w"].double().t())
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        score = p / p.sum(1, keepdim=True)
    ids, w = _plain_choice(case, score, score if s["balance"] is None else score + s["balance"].double())
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return [ids.to(torch.int32), (w * ROUTE_SCALE).float(), logits.float()]


def _plain_weights(kind, blocks):
    """[rows, bytes of a row] as f32 [rows, columns]."""
    rows = blocks.shape[0]
    b = blocks.reshape(-1, QUANT[kind][2])

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).float()
    if kind == "Q8_0":
        return (half(0) * b[:, 2:].view(torch.int8).float()).view(rows, -1)
    if kind == "Q6_K":
        ql, qh = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 1, 32)
        low = torch.cat([ql & 15, ql >> 4], 2)
        shift = torch.tensor([0, 2, 4, 6], device="cuda", dtype=torch.uint8).view(1, 1, 4, 1)
        q = (low | (((qh >> shift) & 3) << 4)).float() - 32.0
        scale = half(208) * b[:, 192:208].contiguous().view(torch.int8).float()
        return (q.view(-1, 16, 16) * scale[:, :, None]).view(rows, -1)
    s6 = b[:, 4:16]
    sc = torch.cat([s6[:, :4] & 63, (s6[:, 8:] & 15) | ((s6[:, :4] >> 6) << 4)], 1).float()
    m = torch.cat([s6[:, 4:8] & 63, (s6[:, 8:] >> 4) | ((s6[:, 4:8] >> 6) << 4)], 1).float()
    qs = b[:, -128:].view(-1, 4, 1, 32)
    q = torch.cat([qs & 15, qs >> 4], 2)
    if kind == "Q5_K":
        shift = torch.arange(8, device="cuda", dtype=torch.uint8).view(1, 4, 2, 1)
        q = q | (((b[:, 16:48].view(-1, 1, 1, 32) >> shift) & 1) << 4)
    q = q.reshape(-1, 8, 32).float()
    return (q * (half(0) * sc)[:, :, None] - (half(2) * m)[:, :, None]).view(rows, -1)


def _plain_moe(s):
    case = s["case"]
    out = torch.zeros_like(s["x"])
    for e in s["ids"].unique().tolist():
        if e < 0:
            continue
        token, place = torch.where(s["ids"] == e)
        x = s["x"][token]
        gate = torch.matmul(x, _plain_weights(case["gate_up"], s["gate_w"][e]).t())
        up = torch.matmul(x, _plain_weights(case["gate_up"], s["up_w"][e]).t())
        y = torch.matmul(gate * (1.0 / (1.0 + torch.exp(-gate))) * up, _plain_weights(case["down"], s["down_w"][e]).t())
        out.index_add_(0, token, y * s["weights"][token, place][:, None])
    return [out]


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    r, h = case["rows"], case["hidden"]
    if case["op"] == "norm":
        gate = {"none": 0, "channel": 4 * h, "token": 4 * r * h}[case["gate"]]
        out = FLOAT[case["out"]][1].itemsize if case["pre"] else 0
        return {"bytes": r * h * (12 + out) + gate + 4 * h * (case["post"] + case["pre"]), "flops": 10 * r * h}
    e, k = case["experts"], case["top_k"]
    if case["op"] == "route":
        return {"bytes": 4 * r * h + e * h * FLOAT[case["weight"]][1].itemsize + r * (4 * e + 8 * k),
                "flops": 2 * r * h * e}
    n = case["inner"]
    tokens = r - (r // 5 + 1 if case["padded"] else 0)
    # experts that some token chose: nearly even odds, so that 1 - (1 - k / e)^tokens of them are read
    used = e * (1.0 - (1.0 - k / e) ** max(tokens, 0)) if k < e else e
    def size(kind):
        return h * n // QUANT[kind][1] * QUANT[kind][2]
    return {"bytes": int(used * (2 * size(case["gate_up"]) + size(case["down"])) + 8 * r * h + 8 * r * k),
            "flops": 6 * max(tokens, 0) * k * h * n}


# ---- the same in 64 bits ----------------------------------------------------------

def exact(case, seed):
    return {"norm": _exact_norm, "route": _exact_route, "moe": _exact_moe}[case["op"]](case, _inputs(case, seed))


def _exact_unit(x):
    return x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()


def _exact_norm(case, s):
    b = s["branch"].double()
    if case["post"]:
        b = _exact_unit(b) * s["post"].double()
    if s["gate"] is not None:
        b = b * s["gate"].double()
    y = RESIDUAL_SCALE * s["x"].double() + BRANCH_SCALE * b
    return [y, _exact_unit(y) * s["pre"].double()] if case["pre"] else [y]


def _exact_route(case, s):
    """One token after the other, the experts taken one at a time."""
    z = s["x"].double() @ s["w"].double().t().contiguous()
    p = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, 1)
    left = p.clone() if s["balance"] is None else p + s["balance"].double()
    r, size = case["rows"], case["experts"] // case["groups"]
    at = torch.arange(r, device="cuda")

    def lowest(v):  # the lowest index of each row's largest value
        top = v.amax(1, keepdim=True)
        return torch.where(v == top, torch.arange(v.shape[1], device="cuda"), v.shape[1]).amin(1)
    if case["groups"] > 1:
        g = left.view(r, case["groups"], size)
        best, rest = torch.zeros(r, case["groups"], dtype=torch.float64, device="cuda"), g.clone()
        for _ in range(min(case["group_best"], size)):
            i = rest.argmax(2, keepdim=True)
            best += rest.gather(2, i).squeeze(2)
            rest.scatter_(2, i, -math.inf)
        open_groups = torch.zeros(r, case["groups"], dtype=torch.bool, device="cuda")
        for _ in range(case["top_groups"]):
            i = lowest(best)
            open_groups[at, i] = True
            best[at, i] = -math.inf
        left = torch.where(open_groups[:, :, None], g, -math.inf).reshape(r, -1)
    ids = torch.empty(r, case["top_k"], dtype=torch.int64, device="cuda")
    for j in range(case["top_k"]):
        ids[:, j] = lowest(left)
        left[at, ids[:, j]] = -math.inf
    w = torch.stack([p[at, ids[:, j]] for j in range(case["top_k"])], 1)
    if case["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return [ids.to(torch.int32), ROUTE_SCALE * w, z]


def _exact_weights(kind, blocks):
    """[rows, bytes of a row] as f64 [rows, columns]: value k of every block in turn from its own bits."""
    rows = blocks.shape[0]
    b = blocks.reshape(-1, QUANT[kind][2]).to(torch.int32)
    k = torch.arange(QUANT[kind][1], device="cuda")

    def f16(at):
        bits = (b[:, at] | (b[:, at + 1] << 8))
        e, f = (bits >> 10) & 31, (bits & 1023).double()
        v = torch.where(e == 0, f * 2.0 ** -24, torch.ldexp(f / 1024.0 + 1.0, (e - 15).double()))
        return torch.where(bits >= 32768, -v, v)[:, None]

    def signed(v):
        return torch.where(v > 127, v - 256, v).double()
    if kind == "Q8_0":
        w = f16(0) * signed(b[:, 2:])
    elif kind == "Q6_K":
        half, quarter, l = k // 128, k // 32 % 4, k % 32
        low = (b[:, 64 * half + 32 * (quarter % 2) + l] >> (4 * (quarter // 2))) & 15
        high = (b[:, 128 + 32 * half + l] >> (2 * quarter)) & 3
        w = f16(208) * signed(b[:, 192 + k // 16]) * ((low + 16 * high) - 32).double()
    else:
        five = kind == "Q5_K"
        sub, l = k // 32, k % 32
        q = (b[:, (48 if five else 16) + 32 * (sub // 2) + l] >> (4 * (sub % 2))) & 15
        if five:
            q = q + 16 * ((b[:, 16 + l] >> sub) & 1)
        j, early = sub % 4, sub < 4
        sc = torch.where(early, b[:, 4 + j] & 63, (b[:, 12 + j] & 15) + 16 * (b[:, 4 + j] >> 6))
        m = torch.where(early, b[:, 8 + j] & 63, (b[:, 12 + j] >> 4) + 16 * (b[:, 8 + j] >> 6))
        w = f16(0) * (sc * q).double() - f16(2) * m.double()
    return w.reshape(rows, -1)


def _exact_moe(case, s):
    out = torch.zeros_like(s["x"], dtype=torch.float64)
    some = max(1, (1 << 24) // case["hidden"])  # rows of weights at a time
    for e in range(case["experts"]):
        pair = (s["ids"] == e).nonzero()
        if not len(pair):
            continue
        x = s["x"][pair[:, 0]].double()

        def times(v, kind, w):
            return torch.cat([v @ _exact_weights(kind, part).t().contiguous() for part in w.split(some)], 1)
        g = times(x, case["gate_up"], s["gate_w"][e])
        y = times(torch.sigmoid(g) * g * times(x, case["gate_up"], s["up_w"][e]), case["down"], s["down_w"][e])
        out.index_put_((pair[:, 0],), y * s["weights"][pair[:, 0], pair[:, 1]].double()[:, None], accumulate=True)
    return [out]
