"""The operators of a decode step around the quantized projections, and the
work that they are timed and compared on.

  rope    okq_qk_norm_rope: the RMS norm of every query and key head, the
          position rotation, and the store of keys and values into a paged cache
  attn    okq_paged_attention: one new token of each sequence against the
          cached keys and values of its pages
  logits  okq_logits_process: penalties for repeated tokens, biases and a
          grammar mask on the output head's logits, and the greedy token

Sizes are the Llama-3-8B attention block's (32 query heads on 8 key/value heads
of 128, vocabulary 128256) and the Gemma4 vocabulary of 262144, with generic
ones around them.  Activations and logits are f32, as the quantized projections
write them; caches are F32, F16, BF16 or Q8_0.
"""
import ctypes
import math

import torch

own = False

F32, F16, BF16, Q8_0 = 0, 1, 30, 8
CACHE = {"F32": (F32, torch.float32), "F16": (F16, torch.float16), "BF16": (BF16, torch.bfloat16), "Q8_0": (Q8_0, torch.uint8)}
EPS = 1e-6
Q8_BLOCK, Q8_BYTES = 32, 34


def listed():
    return [
        # one new token of a chat: rotation in GGUF's neighbouring pairs, far into its context
        dict(name="rope_token", op="rope", tokens=1, q_heads=32, kv_heads=8, head_dim=128, rotary=128, norm=False,
             interleaved=True, cache="BF16", page=16, far=100000),
        # one step of 48 sequences, normalised wide heads of which the first half turns
        dict(name="rope_serving", op="rope", tokens=48, q_heads=20, kv_heads=4, head_dim=256, rotary=128, norm=True,
             interleaved=False, cache="F16", page=24, far=30000),
        # a prompt of 4096 tokens entering the cache
        dict(name="rope_prompt", op="rope", tokens=4096, q_heads=32, kv_heads=8, head_dim=128, rotary=128, norm=True,
             interleaved=False, cache="BF16", page=16, far=0),
        # the first answer token of a short chat: little to read, latency counts
        dict(name="attn_token", op="attn", seqs=1, longest=517, ragged=False, q_heads=32, kv_heads=8, head_dim=128,
             cache="BF16", page=16, window=0, softcap=0.0),
        # one sequence at the far end of its context
        dict(name="attn_long", op="attn", seqs=1, longest=131072, ragged=False, q_heads=32, kv_heads=8, head_dim=128,
             cache="BF16", page=16, window=0, softcap=0.0),
        # a serving batch: contexts from nothing to thousands of tokens
        dict(name="attn_ragged", op="attn", seqs=64, longest=8192, ragged=True, q_heads=32, kv_heads=8, head_dim=128,
             cache="BF16", page=16, window=0, softcap=0.0),
        # a batch on a Q8_0 cache
        dict(name="attn_q8", op="attn", seqs=16, longest=5003, ragged=True, q_heads=32, kv_heads=8, head_dim=128,
             cache="Q8_0", page=32, window=0, softcap=0.0),
        # wide heads, a sliding window and capped scores
        dict(name="attn_window", op="attn", seqs=24, longest=6001, ragged=True, q_heads=16, kv_heads=4, head_dim=256,
             cache="F16", page=64, window=1024, softcap=50.0),
        # every head its own keys, a head size and a page size that are no power of two, an f32 cache
        dict(name="attn_f32_odd", op="attn", seqs=5, longest=3001, ragged=True, q_heads=20, kv_heads=20, head_dim=80,
             cache="F32", page=24, window=0, softcap=0.0),
        # sampling one token of a chat
        dict(name="logits_token", op="logits", rows=1, vocab=128256, history=1200, biases=20, mask=False),
        # a serving batch, long histories
        dict(name="logits_batch", op="logits", rows=64, vocab=128256, history=4000, biases=300, mask=False),
        # a large batch under grammars, the larger vocabulary
        dict(name="logits_grammar", op="logits", rows=200, vocab=262144, history=700, biases=0, mask=True),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rope", "attn", "attn", "logits"])
    if op == "logits":
        vocab = spread(1000, 262144)
        return dict(op=op, rows=min(spread(1, 256), 200 * 262144 // vocab), vocab=vocab, history=spread(1, 4000),
                    biases=rng.choice([0, spread(1, 300)]), mask=rng.random() < 0.5)
    cache = rng.choice(["BF16", "BF16", "F16", "F32"] + ["Q8_0"] * (op == "attn"))
    dim = rng.choice([64, 96, 128, 128, 256] if cache == "Q8_0" else [64, 80, 96, 112, 128, 128, 256])
    kv = spread(1, 16)
    group, page = rng.choice([1, 2, 3, 4, 5, 6, 8, 12]), rng.choice([8, 16, 24, 32, 64, 100])
    if op == "rope":
        tokens = max(1, min(spread(1, 4096), 4096 * 48 * 128 // (kv * (group + 2) * dim)))
        return dict(op=op, tokens=tokens, q_heads=kv * group, kv_heads=kv, head_dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.5, interleaved=rng.random() < 0.5,
                    cache=cache, page=page, far=rng.choice([0, spread(1, 200000)]))
    seqs = spread(1, 96)
    longest = max(1, min(spread(1, 131072), 131072 * 8 * 128 * 2 // (seqs * kv * dim * (4 if cache == "F32" else 2))))
    return dict(op=op, seqs=seqs, longest=longest, ragged=rng.random() < 0.7, q_heads=kv * group, kv_heads=kv,
                head_dim=dim, cache=cache, page=page, window=rng.choice([0, 0, spread(1, 4096)]),
                softcap=rng.choice([0.0, 0.0, 30.0]))


# ---- inputs -----------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _row_bytes(case):
    d = case["head_dim"]
    return d // Q8_BLOCK * Q8_BYTES if case["cache"] == "Q8_0" else d * CACHE[case["cache"]][1].itemsize


def _pages(gen, case, n):
    """n pages [page][kv head][token][row], filled as a cache in use is."""
    shape = (n, case["kv_heads"], case["page"])
    if case["cache"] != "Q8_0":
        return _normal(gen, *shape, case["head_dim"]).to(CACHE[case["cache"]][1])
    nb = case["head_dim"] // Q8_BLOCK
    codes = _normal(gen, *shape, nb, Q8_BLOCK).mul_(45).round_().clamp_(-127, 127).to(torch.int8)
    d = (_normal(gen, *shape, nb, 1).mul_(0.15).add_(1.0).clamp_(0.4, 2.0) / 45).to(torch.float16)
    return torch.cat([d.view(torch.uint8), codes.view(torch.uint8)], -1).reshape(*shape, nb * Q8_BYTES)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    if case["op"] == "logits":
        return _logits_inputs(case, gen)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        t, page = case["tokens"], case["page"]
        x = _normal(gen, t, (hq + 2 * hkv) * d)  # one row of q, k and v side by side, as one projection call leaves them
        x[:, :hq * d] *= 2.0
        n_pages = t // page + 3
        slots = torch.randperm(n_pages * page, generator=gen, device="cuda")[:t]
        pos = torch.arange(t, device="cuda", dtype=torch.int32)
        if case["far"]:
            pos = torch.randint(0, case["far"], (t,), generator=gen, device="cuda").to(torch.int32)
            pos[0] = case["far"]
        half = case["rotary"] // 2
        freq = (500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).to(torch.float32)
        empty = torch.zeros(2, n_pages, hkv, page, d, dtype=CACHE[case["cache"]][1], device="cuda")
        return {"x": x, "slots": slots, "pos": pos, "freq": freq, "kc": empty[0], "vc": empty[1],
                "qn": _normal(gen, d).mul_(0.2).add_(1.0) if case["norm"] else None,
                "kn": _normal(gen, d).mul_(0.2).add_(1.0) if case["norm"] else None}
    s, longest, page = case["seqs"], case["longest"], case["page"]
    lengths = torch.full((s,), longest, device="cuda", dtype=torch.int64)
    if case["ragged"]:  # spread over the logarithm from nothing (a sequence without context) to the longest
        u = torch.rand(s, generator=gen, device="cuda", dtype=torch.float64)
        lengths = torch.exp(u * math.log(longest + 1.0)).to(torch.int64) - 1
        lengths[s // 2] = longest
    need = (lengths + page - 1) // page
    width = (longest + page - 1) // page
    n_pages = int(need.sum()) + 1
    at = torch.arange(width, device="cuda")[None, :] + (need.cumsum(0) - need)[:, None]
    order = torch.randperm(n_pages, generator=gen, device="cuda")
    used = torch.arange(width, device="cuda")[None, :] < need[:, None]
    table = torch.where(used, order[at.clamp(max=n_pages - 1)], torch.full_like(at, -1)).to(torch.int32)
    return {"q": _normal(gen, s, hq, d).mul_(2.0), "kc": _pages(gen, case, n_pages), "vc": _pages(gen, case, n_pages),
            "table": table, "lengths": lengths.to(torch.int32)}


def _logits_inputs(case, gen):
    r, v, h, b = case["rows"], case["vocab"], case["history"], case["biases"]
    u = torch.rand(r, h, generator=gen, device="cuda", dtype=torch.float64)
    hist = (u.pow(3) * v).to(torch.int32).clamp_(max=v - 1)  # frequent tokens many times, rare ones once
    hist_len = torch.randint(0, h + 1, (r,), generator=gen, device="cuda").to(torch.int32)
    hist_len[0] = h
    start = (hist_len * torch.rand(r, generator=gen, device="cuda")).to(torch.int32)  # the prompt's part
    d = {"logits": _normal(gen, r, v).mul_(3.0), "hist": hist, "hist_len": hist_len, "start": start,
         "rep": torch.rand(r, generator=gen, device="cuda").mul_(0.4).add_(1.0),
         "freq": torch.rand(r, generator=gen, device="cuda").mul_(0.5),
         "pres": torch.rand(r, generator=gen, device="cuda").mul_(0.5), "bias_ids": None, "mask": None}
    if b:
        d["bias_ids"] = torch.rand(r, v, generator=gen, device="cuda").topk(b, dim=1).indices.to(torch.int32)
        d["bias"] = _normal(gen, r, b).mul_(4.0)
        d["bias_len"] = torch.randint(0, b + 1, (r,), generator=gen, device="cuda").to(torch.int32)
    if case["mask"]:  # grammars that allow one token in a hundred, half of them, or (a dead end) none
        share = torch.tensor([0.01, 0.5, 0.98], device="cuda")[torch.arange(r, device="cuda") % 3]
        if r > 2:
            share[r // 2] = 0.0
        words = (v + 31) // 32
        bits = torch.rand(r, words, 32, generator=gen, device="cuda") < share[:, None, None]
        w = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(2)
        d["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    return d


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if case["op"] == "rope":
        t, hq, d = case["tokens"], case["q_heads"], case["head_dim"]
        s["q_out"] = torch.empty(t, hq, d, device="cuda")
    elif case["op"] == "attn":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(case["seqs"], case["q_heads"], device="cuda")
    else:
        s["out"] = torch.empty_like(s["logits"])
        s["best"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        if "call" not in state:
            state["call"] = _call(state)
        from ocelotl_amd import okq
        name, args = state["call"]
        okq.call(name, *args, torch.cuda.current_stream().cuda_stream)
        if op == "rope":
            return [state["q_out"], state["kc"], state["vc"]]
        return [state["out"], state["lse" if op == "attn" else "best"]]
    return {"rope": _plain_rope, "attn": _plain_attention, "logits": _plain_logits}[op](state)


# ---- the framework's calls ----------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _kv_pages(case, s):
    from ocelotl_amd import okq
    row = _row_bytes(case)
    page, heads = case["page"], case["kv_heads"]
    return okq.KvPages(type=CACHE[case["cache"]][0], n_pages=s["kc"].shape[0], page_tokens=page, kv_heads=heads,
                       head_dim=case["head_dim"], page_stride=heads * page * row, head_stride=page * row,
                       token_stride=row, k=s["kc"].data_ptr(), v=s["vc"].data_ptr())


def _call(s):
    case = s["case"]
    if case["op"] == "logits":
        b = s["bias_ids"] is not None
        return "okq_logits_process", (
            _ptr(s["logits"]), case["vocab"], case["rows"], case["vocab"],
            _ptr(s["hist"]), case["history"], _ptr(s["hist_len"]), _ptr(s["start"]),
            _ptr(s["rep"]), _ptr(s["freq"]), _ptr(s["pres"]),
            _ptr(s["bias_ids"]), _ptr(s["bias"]) if b else None, case["biases"], _ptr(s["bias_len"]) if b else None,
            _ptr(s["mask"]), (case["vocab"] + 31) // 32, _ptr(s["out"]), case["vocab"], _ptr(s["best"]))
    cache = s["cache"] = _kv_pages(case, s)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        x, width = s["x"].data_ptr(), (hq + 2 * hkv) * d
        return "okq_qk_norm_rope", (
            x, width, x + 4 * hq * d, width, x + 4 * (hq + hkv) * d, width, case["tokens"], hq, hkv, d,
            _ptr(s["qn"]), _ptr(s["kn"]), EPS, _ptr(s["pos"]), _ptr(s["freq"]), case["rotary"],
            int(case["interleaved"]), _ptr(s["q_out"]), hq * d, None, 0, ctypes.byref(cache), _ptr(s["slots"]))
    return "okq_paged_attention", (
        _ptr(s["q"]), hq * d, case["seqs"], hq, ctypes.byref(cache), _ptr(s["table"]), s["table"].shape[1],
        _ptr(s["lengths"]), case["longest"], 1.0 / math.sqrt(d), case["softcap"], case["window"], _ptr(s["out"]),
        hq * d, _ptr(s["lse"]))


# ---- plain forms ----------------------------------------------------------------

def _plain_rotate(x, angle, case):
    half = case["rotary"] // 2
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if case["interleaved"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_norm(x, w):
    return x if w is None else x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w


def _plain_store(case, pages, slots, x):
    """Rows x [tokens, kv heads, head_dim] into their slots."""
    page, at = torch.div(slots, case["page"], rounding_mode="floor"), slots % case["page"]
    pages[page, :, at] = x.to(pages.dtype)


def _plain_rope(s):
    case = s["case"]
    t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    x = s["x"].view(t, hq + 2 * hkv, d)
    angle = s["pos"].double()[:, None] * s["freq"].double()
    q = _plain_rotate(_plain_norm(x[:, :hq], s["qn"]), angle, case)
    k = _plain_rotate(_plain_norm(x[:, hq:hq + hkv], s["kn"]), angle, case)
    _plain_store(case, s["kc"], s["slots"], k)
    _plain_store(case, s["vc"], s["slots"], x[:, hq + hkv:])
    return [q, s["kc"], s["vc"]]


def _plain_gather(case, pages, table):
    """The pages of every sequence as f32 [seqs, kv heads, tokens, head_dim]."""
    p = pages[table.clamp(min=0).long()]
    if case["cache"] == "Q8_0":
        p = p.unflatten(-1, (-1, Q8_BYTES))
        p = (p[..., :2].contiguous().view(torch.float16).float() * p[..., 2:].view(torch.int8).float()).flatten(-2)
    return p.float().transpose(1, 2).flatten(2, 3).contiguous()


def _plain_attention(s):
    case = s["case"]
    n, hkv, d = case["seqs"], case["kv_heads"], case["head_dim"]
    k, v = _plain_gather(case, s["kc"], s["table"]), _plain_gather(case, s["vc"], s["table"])
    q = s["q"].view(n, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    at, length = torch.arange(k.shape[2], device="cuda"), s["lengths"].long()[:, None]
    seen = at < length
    if case["window"]:
        seen = seen & (at >= length - case["window"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return [out.view(n, -1, d), (top + torch.log(total)).view(n, -1)]


def _plain_logits(s):
    case = s["case"]
    x, h = s["logits"], s["hist"].long()
    at = torch.arange(h.shape[1], device="cuda")
    past = at < s["hist_len"][:, None]
    count = torch.zeros(x.shape[0], x.shape[1], device="cuda")
    seen = count.scatter_add(1, h, past.float())
    count = count.scatter_add(1, h, (past & (at >= s["start"][:, None])).float())
    rep, freq, pres = s["rep"][:, None], s["freq"][:, None], s["pres"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * count
    x = torch.where(count > 0, x - pres, x)
    if s["bias_ids"] is not None:
        valid = torch.arange(case["biases"], device="cuda") < s["bias_len"][:, None]
        x = x.scatter_add(1, s["bias_ids"].long(), torch.where(valid, s["bias"], 0.0))
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :case["vocab"]] == 0, -math.inf)
    top, best = x.max(1)
    first = torch.where(x == top[:, None], torch.arange(x.shape[1], device="cuda"), x.shape[1]).amin(1)
    best = torch.where(top > -math.inf, first, -1)
    return [x, best.to(torch.int32)]


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    if case["op"] == "logits":
        r, v = case["rows"], case["vocab"]
        b = r * (8 * v + 2 * case["history"] + 4 * case["biases"] + (v // 8 if case["mask"] else 0) + 28)
        return {"bytes": b, "flops": 2 * r * v}
    hq, hkv, d, row = case["q_heads"], case["kv_heads"], case["head_dim"], _row_bytes(case)
    if case["op"] == "rope":
        t = case["tokens"]
        return {"bytes": t * (4 * (2 * hq + 2 * hkv) * d + 2 * hkv * row + 12) + 2 * case["rotary"],
                "flops": t * (hq + hkv) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    s, longest = case["seqs"], case["longest"]
    # ragged lengths are spread over their logarithm, one of them the longest
    mean = longest / math.log(longest + 1.0) if case["ragged"] else longest
    if case["window"]:
        w = min(case["window"], longest)
        mean = w / math.log(longest + 1.0) + w * (1 - math.log(w + 1.0) / math.log(longest + 1.0)) if case["ragged"] else w
    tokens = (s - 1) * mean + min(longest, case["window"] or longest)
    return {"bytes": int(tokens * hkv * 2 * row + s * (8 * hq * d + 4 * hq + 4)), "flops": int(tokens * 4 * hq * d)}


# ---- the same in 64 bits ----------------------------------------------------------

def exact(case, seed):
    return {"rope": _exact_rope, "attn": _exact_attention, "logits": _exact_logits}[case["op"]](case, _inputs(case, seed))


def _exact_cached(case, slots, rows):
    """A cache after rows [tokens, heads, dim] went to their slots, in f64."""
    n_slots = (case["tokens"] // case["page"] + 3) * case["page"]
    flat = torch.zeros(n_slots, case["kv_heads"], case["head_dim"], dtype=torch.float64, device="cuda")
    flat[slots] = rows
    return flat.view(-1, case["page"], case["kv_heads"], case["head_dim"]).permute(0, 2, 1, 3).contiguous()


def _exact_rope(case, s):
    t, hq, hkv, d, half = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary"] // 2
    x = s["x"].double().reshape(t, hq + 2 * hkv, d)
    if case["norm"]:
        unit = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
        x = torch.cat([unit[:, :hq] * s["qn"].double(), unit[:, hq:hq + hkv] * s["kn"].double(), x[:, hq + hkv:]], 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["freq"].double())
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    z = torch.complex(x[:, :hq + hkv, first], x[:, :hq + hkv, second]) * turn[:, None]
    y = x[:, :hq + hkv].clone()
    y[..., first], y[..., second] = z.real, z.imag
    return [y[:, :hq], _exact_cached(case, s["slots"], y[:, hq:]), _exact_cached(case, s["slots"], x[:, hq + hkv:])]


def _exact_rows(case, pages, ids, lo, hi):
    """Tokens lo..hi of one sequence's pages in f64 [kv heads, tokens, head_dim]."""
    p = pages[ids]
    if case["cache"] == "Q8_0":
        blocks = p.reshape(-1, Q8_BYTES)
        p = (blocks[:, 2:].view(torch.int8).double() * blocks[:, :2].contiguous().view(torch.float16).double())
        p = p.reshape(len(ids), case["kv_heads"], case["page"], case["head_dim"])
    return p.double().permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["head_dim"])[:, lo:hi]


def _exact_attention(case, s):
    hkv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(out.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["lengths"].tolist()):
        if not length:
            continue
        ids = s["table"][i, :(length + page - 1) // page].long()
        lo = max(0, length - case["window"]) if case["window"] else 0
        k, v = _exact_rows(case, s["kc"], ids, lo, length), _exact_rows(case, s["vc"], ids, lo, length)
        score = torch.bmm(s["q"][i].double().reshape(hkv, -1, d), k.transpose(1, 2).contiguous()) / math.sqrt(d)
        if case["softcap"]:
            score = torch.tanh(score / case["softcap"]) * case["softcap"]
        lse[i] = torch.logsumexp(score, -1).reshape(-1)
        out[i] = torch.bmm(torch.softmax(score, -1), v.contiguous()).reshape(-1, d)
    return [out, lse]


def _exact_logits(case, s):
    x = s["logits"].double()
    for i, (n, start) in enumerate(zip(s["hist_len"].tolist(), s["start"].tolist())):
        h = s["hist"][i, :n].long()
        ids = torch.unique(h)
        new, times = torch.unique(h[start:], return_counts=True)
        rep = s["rep"][i].double()
        x[i, ids] = torch.where(x[i, ids] > 0, x[i, ids] / rep, x[i, ids] * rep)
        x[i, new] -= s["freq"][i].double() * times + s["pres"][i].double()
        if s["bias_ids"] is not None:
            m = int(s["bias_len"][i])
            x[i, s["bias_ids"][i, :m].long()] += s["bias"][i, :m].double()
    if s["mask"] is not None:
        token = torch.arange(case["vocab"], device="cuda")
        x[((s["mask"][:, token // 32] >> (token % 32).to(torch.int32)) & 1) == 0] = -math.inf
    return [x, None]
