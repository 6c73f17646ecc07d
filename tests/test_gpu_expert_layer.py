"""okq_residual_norm, okq_moe_route and okq_moe_mlp_q against their definitions
in 64 bits (needs an MI355X).

Bounds, derived before the first run.  u = 2^-24 is half a step of f32.
  residual norm: a norm's factor is off by at most 24u relative (squares and
    sums of a row in a tree behind at most 16 in a thread; the long rows' sums
    of n / 1024 in a thread go like a random walk, 8 deviations: 8u sqrt(n /
    1024) more), each product and sum by u: sum within 4u (|rs x| + |t|) +
    (24u + walk) |t| with t = bs gate b; normed within that divided by the
    row's rms and times pre, and (26u + walk + that's own rms over the row's) of
    its value, and half a step of its type.
  route: 64 bits throughout: ids equal, weights and logits within half a step
    of f32 (and 2^-40 of the sum of magnitudes, far above any 64-bit sum's own).
  experts: a product x W is off by 2^-21 (two planes' roundings and the left
    out product of the low ones), sums go like a random walk of at most
    K / 8 f32 additions, 8 deviations: e = (2^-21 + 8u sqrt(K / 8)) sum |x| W',
    W' = |W| plus twice the largest |W| of its run of 32 (the integer part and
    the min term are summed apart).  silu's slope is at most 1.1, its own
    error 8u: h within 1.1 e_g |u| + |silu(g)| e_u + 8u |h|; the outputs sum
    those against |W_down| and add e of their own, a row's top_k results 2u
    each.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16, Q8_0, Q4_K, Q5_K, Q6_K = 0, 1, 30, 8, 12, 13, 14
BYTES = {Q8_0: (32, 34), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210)}
EPS = 1e-6


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    if not _t.cuda.is_available():
        pytest.skip("no GPU")
    return _t


@pytest.fixture(scope="module")
def okq(torch):
    from ocelotl_amd import okq as _okq
    _okq.call("okq_init", 0)
    return _okq


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _dtype(torch, t):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[t]


def _rows(torch, n, width, stride, offset=0, dtype=None, fill=None):
    """[n, width] rows `stride` apart, `offset` elements into their allocation; fill: what lies around them."""
    buf = torch.full((n * stride + offset,), math.nan if fill is None else fill, device="cuda",
                     dtype=dtype or torch.float32)
    return buf, buf[offset:].as_strided((n, width), (stride, 1), buf.storage_offset() + offset)


# ---- residual norm -------------------------------------------------------------

NORM = [  # rows, hidden, post, gate ("", "one", "row"), pre, type, sum ("new", "x", "branch", ""), pad, offset
    (1, 4096, True, "", True, F32, "new", 0, 0),
    (3, 2560, True, "one", True, BF16, "x", 0, 0),
    (5, 1111, False, "row", True, F16, "branch", 3, 1),
    (2, 1, True, "", True, F32, "new", 0, 0),
    (2, 3, True, "row", True, F16, "", 0, 0),
    (4, 64, False, "", False, F32, "new", 0, 0),
    (4, 64, True, "one", False, F32, "x", 4, 4),
    (3, 257, True, "row", True, BF16, "new", 0, 0),
    (2, 8192, True, "", True, F32, "", 8, 0),
    (2, 16384, True, "row", True, BF16, "x", 0, 0),
    (2, 16388, True, "row", True, BF16, "x", 0, 0),
    (2, 8193, True, "", True, F32, "branch", 0, 0),
    (1, 40001, True, "one", True, F16, "", 0, 3),
    (777, 512, True, "", True, F32, "x", 0, 0),
    (300, 4096, True, "one", True, BF16, "new", 0, 4),
]


def _norm_case(torch, okq, case, scales=(0.75, 1.125), spoil=None):
    rows, hidden, post, gate, pre, kind, where, pad, offset = case
    g = _gen(torch, rows * 31 + hidden)
    stride = hidden + pad
    _, x = _rows(torch, rows, hidden, stride, offset)
    _, b = _rows(torch, rows, hidden, stride, offset)
    x.copy_(torch.randn(rows, hidden, generator=g, device="cuda") * 3)
    b.copy_(torch.randn(rows, hidden, generator=g, device="cuda"))
    if spoil:
        spoil(x, b)
    w = [torch.randn(hidden, generator=g, device="cuda") * 0.2 + 1 if f else None for f in (post, pre)]
    gt = torch.randn(rows if gate == "row" else 1, hidden, generator=g, device="cuda") if gate else None
    total = {"new": _rows(torch, rows, hidden, stride, offset)[1], "x": x, "branch": b, "": None}[where]
    normed = _rows(torch, rows, hidden, stride, offset, dtype=_dtype(torch, kind))[1] if pre else None
    x64, b64 = x.double(), b.double()
    bs, rs = scales
    okq.call("okq_residual_norm", x.data_ptr(), stride, b.data_ptr(), stride, rows, hidden, _ptr(w[0]), _ptr(gt),
             hidden if gate == "row" else 0, bs, rs, _ptr(w[1]), EPS, _ptr(total), stride, _ptr(normed), kind, stride,
             _stream(torch))
    torch.cuda.synchronize()
    if post:
        b64 = b64 / (b64.square().mean(1, keepdim=True) + EPS).sqrt() * w[0].double()
    t = bs * b64 * (gt.double() if gate else 1.0)
    y = rs * x64 + t
    walk = 8 * U * math.sqrt(hidden / 1024) if hidden > 8192 else 0.0
    off = 4 * U * ((rs * x64).abs() + t.abs()) + (24 * U + walk) * t.abs() * post
    want = None
    if pre:
        rms = (y.square().mean(1, keepdim=True) + EPS).sqrt()
        want = y / rms * w[1].double()
        far = off / rms * w[1].double().abs()
        far = far + want.abs() * (26 * U + walk + off.square().mean(1, keepdim=True).sqrt() / rms)
        half = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}[kind]
        far = far + half * want.abs() + (2.0 ** -25 if kind == F16 else 0.0)
        want = (want, far)
    return total, normed, (y, off), want


def _within(got, want, bound, what):
    import torch
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), torch.nonzero(bad)[:3].tolist(),
                                 float((got - want).abs()[bad].max()), float(bound.expand_as(want)[bad].min()))


@pytest.mark.parametrize("case", NORM, ids=[str(c[:2]) for c in NORM])
def test_residual_norm(torch, okq, case):
    total, normed, (y, off), want = _norm_case(torch, okq, case)
    if total is not None:
        _within(total, y, off, "sum")
    if want is not None:
        _within(normed, *want, "normed")


def test_residual_norm_leaves_what_lies_between_rows(torch, okq):
    buf, s = _rows(torch, 3, 60, 64, 4, fill=7.0)
    x, b = torch.randn(3, 60, device="cuda"), torch.randn(3, 60, device="cuda")
    hbuf, h = _rows(torch, 3, 60, 68, 4, dtype=torch.bfloat16, fill=7.0)
    one = torch.ones(60, device="cuda")
    okq.call("okq_residual_norm", x.data_ptr(), 60, b.data_ptr(), 60, 3, 60, None, None, 0, 1.0, 1.0, one.data_ptr(), EPS,
             s.data_ptr(), 64, h.data_ptr(), BF16, 68, _stream(torch))
    assert torch.equal(s, x + b)
    for whole, part in ((buf, s), (hbuf, h)):
        part.fill_(7.0)
        assert bool((whole == 7.0).all())


def test_residual_norm_of_zero_rows_and_huge_ones(torch, okq):
    """Rows of zeros normalise to zeros; an infinity or NaN reaches its row and no other."""
    def spoil(x, b):
        x[0] = 0.0
        b[0] = 0.0
        x[1, 5] = math.inf
        b[2, 7] = math.nan
    total, normed, (y, off), want = _norm_case(torch, okq, (5, 1024, True, "", True, F32, "new", 0, 0), spoil=spoil)
    assert not bool(total[0].any()) and not bool(normed[0].any())
    assert math.isinf(float(total[1, 5])) and bool(torch.isnan(normed[1, 5]))
    assert bool(torch.isnan(total[2]).all()) and bool(torch.isnan(normed[2]).all())
    _within(total[3:], y[3:], off[3:], "sum")
    _within(normed[3:], want[0][3:], want[1][3:], "normed")


# ---- routing -------------------------------------------------------------------

ROUTE = [  # rows, hidden, experts, top_k, sigmoid, groups, top_groups, group_best, bias, choice, renorm, type, pad
    (1, 2048, 128, 8, False, 1, 1, 1, False, False, True, F32, 0),
    (5, 64, 8, 2, False, 1, 1, 1, True, False, True, BF16, 0),
    (61, 2560, 256, 8, True, 8, 4, 2, False, True, True, F32, 0),
    (17, 4096, 512, 10, False, 1, 1, 1, False, True, False, F16, 4),
    (3, 7, 1, 1, True, 1, 1, 1, False, False, True, F32, 0),
    (4, 1, 5, 5, False, 1, 1, 1, False, False, True, BF16, 0),
    (33, 999, 60, 4, False, 1, 1, 1, True, True, True, F32, 1),
    (2, 130, 64, 64, False, 1, 1, 1, False, False, False, F16, 0),
    (40, 1023, 96, 6, True, 4, 2, 1, True, True, False, BF16, 0),
    (9, 512, 64, 3, False, 64, 7, 2, False, False, True, F32, 0),
    (300, 1024, 33, 5, True, 3, 1, 2, False, True, True, F32, 0),
    (4096, 512, 128, 8, False, 1, 1, 1, False, False, True, BF16, 0),
    (2100, 100, 17, 2, True, 1, 1, 1, False, True, True, F32, 0),
    (2049, 256, 40, 4, False, 8, 3, 2, True, False, True, F16, 8),
]


def _route_want(torch, x, w, bias, choice, sigmoid, groups, top_groups, group_best, top_k, renorm, scale):
    """ids, weights and logits of the definition, row by row on the CPU."""
    z = x.double() @ w.double().t().contiguous()
    if bias is not None:
        z = z + bias.double()
    p = torch.sigmoid(z) if sigmoid else torch.softmax(z, 1)
    c = p if choice is None else p + choice.double()
    p, c = p.cpu(), c.cpu()
    rows, experts = p.shape
    ids = torch.full((rows, top_k), -1, dtype=torch.int32)
    weights = torch.zeros(rows, top_k, dtype=torch.float64)
    size = experts // groups
    pl, cl = p.tolist(), c.tolist()
    for r in range(rows):
        row = cl[r]
        if any(math.isnan(v) for v in row):
            weights[r] = math.nan
            continue
        if groups > 1:
            best = [sum(sorted(row[g * size:(g + 1) * size], reverse=True)[:group_best]) for g in range(groups)]
            stay = set(sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups])
            row = [v if e // size in stay else -math.inf for e, v in enumerate(row)]
        order = [e for e in sorted(range(experts), key=lambda e: (-row[e], e))[:top_k] if row[e] > -math.inf]
        total = sum(pl[r][e] for e in order)
        for j, e in enumerate(order):
            ids[r, j] = e
            weights[r, j] = scale * ((pl[r][e] / total if total > 0 else 0.0) if renorm else pl[r][e])
    return ids, weights, z


def _route(torch, okq, x, stride, w, kind, bias, choice, sigmoid, groups, top_groups, group_best, top_k, renorm, scale,
           logits=True):
    rows, hidden = x.shape
    experts = w.shape[0]
    ids = torch.full((rows, top_k), 12345, dtype=torch.int32, device="cuda")
    weights = torch.full((rows, top_k), 7.0, device="cuda")
    z = torch.full((rows, experts), 7.0, device="cuda") if logits else None
    okq.call("okq_moe_route", x.data_ptr(), stride, rows, hidden, kind, w.data_ptr(), experts, _ptr(bias), int(sigmoid),
             _ptr(choice), groups, top_groups, group_best, top_k, int(renorm), scale, ids.data_ptr(), weights.data_ptr(),
             _ptr(z), _stream(torch))
    torch.cuda.synchronize()
    return ids, weights, z


def _route_inputs(torch, case, seed=5):
    rows, hidden, experts, top_k, sigmoid, groups, top_groups, best, bias, choice, renorm, kind, pad = case
    g = _gen(torch, seed + rows)
    _, x = _rows(torch, rows, hidden, hidden + pad)
    x.copy_(torch.randn(rows, hidden, generator=g, device="cuda"))
    w = (torch.randn(experts, hidden, generator=g, device="cuda") * 1.5 * hidden ** -0.5).to(_dtype(torch, kind))
    b = torch.randn(experts, generator=g, device="cuda") * 0.5 if bias else None
    c = torch.randn(experts, generator=g, device="cuda") * 0.1 if choice else None
    return x, hidden + pad, w, kind, b, c, sigmoid, groups, top_groups, best, top_k, renorm, 2.5


def _check_route(torch, got, want, x, w):
    ids, weights, z = got
    wi, ww, wz = want
    assert torch.equal(ids.cpu(), wi)
    near = 2.0 ** -40
    assert bool(((weights.cpu().double() - ww).abs() <= (U + near) * ww.abs() + 2.0 ** -149).all())
    if z is not None:
        mag = x.double().abs() @ w.double().abs().t().contiguous()
        _within(z, wz, U * wz.abs() + near * mag, "logits")


@pytest.mark.parametrize("case", ROUTE, ids=[str(c[:4]) for c in ROUTE])
def test_route(torch, okq, case):
    args = _route_inputs(torch, case)
    got = _route(torch, okq, *args)
    x, _, w, _, b, c, *rest = args
    _check_route(torch, got, _route_want(torch, x, w, b, c, *rest), x, w)


def test_route_ties_go_to_the_lowest(torch, okq):
    x = torch.ones(20, 32, device="cuda")
    w = torch.zeros(48, 32, device="cuda")
    w[[7, 30, 41]] = 0.25
    ids, weights, _ = _route(torch, okq, x, 32, w, F32, None, None, False, 1, 1, 1, 6, True, 1.0)
    assert ids.tolist() == [[7, 30, 41, 0, 1, 2]] * 20
    # whole groups that tie, and inside them
    ids, _, _ = _route(torch, okq, x, 32, w, F32, None, None, True, 6, 2, 2, 6, True, 1.0)
    assert ids.tolist() == [[7, 30, 0, 1, 2, 3]] * 20


def test_route_masks_and_bad_rows(torch, okq):
    """-infinity in choice_bias shuts experts out, to the last one; NaN reaches its row only."""
    case = (37, 256, 24, 4, False, 1, 1, 1, False, False, True, F32, 0)
    x, stride, w, kind, _, _, *rest = _route_inputs(torch, case)
    lowest = torch.finfo(torch.float32).min
    for left in (24, 5, 3, 1, 0):
        choice = torch.zeros(24, device="cuda")
        choice[left:] = -math.inf
        got = _route(torch, okq, x, stride, w, kind, None, choice, *rest)
        _check_route(torch, got, _route_want(torch, x, w, None, choice, *rest), x, w)
    choice = torch.full((24,), lowest, device="cuda")  # the type's lowest value is no infinity: all tie
    ids, _, _ = _route(torch, okq, x, stride, w, kind, None, choice, *rest)
    assert ids.tolist() == [[0, 1, 2, 3]] * 37
    x[5, 9] = math.nan
    x[6, 9] = math.inf
    ids, weights, _ = _route(torch, okq, x, stride, w, kind, None, None, *rest)
    want = _route_want(torch, x, w, None, None, *rest)
    keep = [r for r in range(37) if r not in (5, 6)]
    assert ids[5].tolist() == [-1] * 4 and bool(torch.isnan(weights[5]).all())
    assert ids[6].tolist() == [-1] * 4 and bool(torch.isnan(weights[6]).all())
    assert torch.equal(ids.cpu()[keep], want[0][keep])


def test_route_scores_that_vanish(torch, okq):
    """A sum of scores that is 0 leaves weights of 0."""
    x = torch.ones(2, 16, device="cuda")
    w = torch.full((4, 16), -100.0, device="cuda")
    ids, weights, _ = _route(torch, okq, x, 16, w, F32, None, None, True, 1, 1, 1, 2, True, 1.0)
    assert ids.tolist() == [[0, 1]] * 2 and not bool(weights.any())


def test_route_does_not_depend_on_the_batch(torch, okq):
    case = (4096, 1000, 128, 8, False, 1, 1, 1, False, False, True, F32, 0)
    args = _route_inputs(torch, case)
    ids, weights, z = _route(torch, okq, *args)
    for n in (1, 16, 100, 1500):
        some = _route(torch, okq, args[0][:n], *args[1:])
        assert torch.equal(some[0], ids[:n])
        assert bool(((some[1] - weights[:n]).abs() <= 2 * U * weights[:n]).all())


# ---- the experts' products ---------------------------------------------------------

def _stack(torch, okq, kind, experts, rows, cols, seed, offset=0):
    """Stacked blocks and their values [experts, rows, cols] in f32."""
    n = experts * rows * cols
    elems, size = BYTES[kind]
    f = torch.empty(n, device="cuda")
    s = _stream(torch)
    okq.call("okq_fill_normal", seed, 0, n, cols ** -0.5, f.data_ptr(), s)
    q = torch.empty(n // elems * size, dtype=torch.uint8, device="cuda")
    okq.call("okq_quantize", kind, f.data_ptr(), n, q.data_ptr(), s)
    okq.call("okq_dequantize", kind, q.data_ptr(), n, f.data_ptr(), s)
    buf = torch.full((q.numel() + offset,), 0xFF, dtype=torch.uint8, device="cuda")
    buf[offset:] = q
    return buf[offset:], f.view(experts, rows, cols)


def _apart(w):
    """|W| plus twice the largest |W| of its run of 32, f64."""
    a = w.double().abs()
    runs = a.unflatten(-1, (-1, 32))
    return (runs + 2 * runs.amax(-1, keepdim=True)).flatten(-2)


def _moe_want(torch, x, ids, weights, gate, up, down):
    """The definition in f64, and the bound."""
    rows, hidden = x.shape
    out = torch.zeros(rows, hidden, dtype=torch.float64, device="cuda")
    far = torch.zeros_like(out)

    def e(k):
        return 2.0 ** -21 + 8 * U * math.sqrt(k / 8)

    def mm(a, b):
        return torch.matmul(a, b.t().contiguous())
    for ex in range(gate.shape[0]):
        at = (ids == ex).nonzero()
        if not len(at):
            continue
        t = at[:, 0]
        a = x[t].double()
        g, u = mm(a, gate[ex].double()), mm(a, up[ex].double())
        eg, eu = (e(hidden) * mm(a.abs(), _apart(w[ex])) for w in (gate, up))
        silu = g * torch.sigmoid(g)
        h = silu * u
        eh = 1.1 * eg * u.abs() + silu.abs() * eu + 8 * U * h.abs() + 1.1 * eg * eu
        d = down[ex].double()
        w = weights[t, at[:, 1]].double()[:, None]
        y = mm(h, d)
        far.index_add_(0, t, w.abs() * (mm(eh, d.abs()) + e(h.shape[1]) * mm(h.abs() + eh, _apart(down[ex]))) + 2 * U * (w * y).abs())
        out.index_add_(0, t, w * y)
    return out, far


class Experts:
    def __init__(self, torch, okq, experts, hidden, inner, gu, dn, seed=3, offset=0):
        self.gu, self.dn, self.hidden, self.inner, self.experts = gu, dn, hidden, inner, experts
        self.gate, self.gate_f = _stack(torch, okq, gu, experts, inner, hidden, seed, offset)
        self.up, self.up_f = _stack(torch, okq, gu, experts, inner, hidden, seed + 1, offset)
        self.down, self.down_f = _stack(torch, okq, dn, experts, hidden, inner, seed + 2, offset)

    def __call__(self, torch, okq, x, ids, weights, out=None, x_stride=None, out_stride=None, stream=None):
        rows, k = ids.shape
        out = torch.full((rows, self.hidden), math.nan, device="cuda") if out is None else out
        okq.call("okq_moe_mlp_q", x.data_ptr(), x_stride or self.hidden, rows, self.hidden, self.inner, self.experts, k,
                 ids.data_ptr(), weights.data_ptr(), self.gu, self.gate.data_ptr(), self.gate.numel(), self.up.data_ptr(),
                 self.up.numel(), self.dn, self.down.data_ptr(), self.down.numel(), out.data_ptr(),
                 out_stride or self.hidden, stream if stream is not None else _stream(torch))
        return out

    def want(self, torch, x, ids, weights):
        return _moe_want(torch, x, ids, weights, self.gate_f, self.up_f, self.down_f)


def _pairs(torch, rows, experts, k, seed):
    g = _gen(torch, seed)
    logits = torch.randn(rows, experts, generator=g, device="cuda") + 0.7 * torch.randn(1, experts, generator=g, device="cuda")
    top = logits.topk(k, 1)
    return top.indices.int().contiguous(), torch.softmax(top.values, 1).contiguous()


MOE = [  # rows, hidden, inner, experts, top_k, gate and up, down
    (1, 512, 256, 16, 2, Q4_K, Q6_K),
    (1, 2048, 768, 32, 8, Q4_K, Q4_K),
    (2, 256, 512, 4, 1, Q5_K, Q8_0),
    (5, 512, 352, 7, 3, Q8_0, Q8_0),     # rows of 1 3/8 items
    (7, 1056, 32, 5, 2, Q8_0, Q8_0),     # one block a row, and an odd row of 33
    (17, 256, 256, 1, 1, Q4_K, Q4_K),    # one expert, two turns of 16 rows
    (33, 768, 1280, 6, 2, Q6_K, Q5_K),
    (70, 512, 512, 9, 4, Q5_K, Q6_K),
    (3, 4096, 2560, 3, 2, Q4_K, Q6_K),   # two rounds of items a wave
    (260, 512, 768, 8, 2, Q4_K, Q6_K),
    (600, 512, 288, 5, 3, Q8_0, Q8_0),
    (515, 256, 512, 40, 8, Q6_K, Q4_K),
    (1, 256, 256, 64, 64, Q5_K, Q5_K),
]


@pytest.mark.parametrize("case", MOE, ids=[str(c) for c in MOE])
def test_moe(torch, okq, case):
    rows, hidden, inner, experts, k, gu, dn = case
    e = Experts(torch, okq, experts, hidden, inner, gu, dn)
    x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
    x[:, 3 % hidden] *= 20.0
    ids, weights = _pairs(torch, rows, experts, k, 9)
    got = e(torch, okq, x, ids, weights)
    _within(got, *e.want(torch, x, ids, weights), "out")


def _odd_ids(torch, ids, weights, experts):
    """Ids outside the experts (their weights NaN), a row without any, the same expert twice."""
    bad = ids.clone()
    rows = ids.shape[0]
    bad[0, 0] = -1
    bad[1 % rows, 1] = experts
    bad[2 % rows] = torch.tensor([2 ** 31 - 1, -2 ** 31] + [-1] * (ids.shape[1] - 2), device="cuda")
    bad[3 % rows, 1] = bad[3 % rows, 0]
    w = weights.clone()
    w[(bad < 0) | (bad >= experts)] = math.nan
    return bad, w


@pytest.mark.parametrize("rows", [4, 23, 150, 700])
@pytest.mark.parametrize("experts", [6, 200])
def test_moe_ids_outside_the_experts_add_nothing(torch, okq, rows, experts):
    e = Experts(torch, okq, experts, 256, 256, Q4_K, Q6_K)
    x = torch.randn(rows, 256, generator=_gen(torch, rows), device="cuda")
    ids, weights = _odd_ids(torch, *_pairs(torch, rows, experts, 3, 2), experts)
    got = e(torch, okq, x, ids, weights)
    _within(got, *e.want(torch, x, ids, weights), "out")
    assert not bool(got[2].any())
    ids.fill_(-1)
    got = e(torch, okq, x, ids, weights)
    assert not bool(got.any()) and not bool(torch.isnan(got).any())


@pytest.mark.parametrize("rows", [3, 90, 400])
def test_moe_strides_and_alignment(torch, okq, rows):
    """Padded rows of x and out, weights that start 4 bytes into their allocation, and between experts on a half word."""
    for kind, hidden, inner in ((Q8_0, 96, 288), (Q6_K, 256, 256), (Q4_K, 256, 512)):
        e = Experts(torch, okq, 3, hidden, inner, kind, kind, offset=4)
        _, x = _rows(torch, rows, hidden, hidden + 12, 4)
        x.copy_(torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda"))
        ids, weights = _pairs(torch, rows, 3, 2, 4)
        for pad, offset in ((8, 4), (3, 1)):
            buf, out = _rows(torch, rows, hidden, hidden + pad, offset, fill=7.0)
            e(torch, okq, x, ids, weights, out=out, x_stride=hidden + 12, out_stride=hidden + pad)
            _within(out, *e.want(torch, x, ids, weights), "out")
            out.fill_(7.0)
            assert bool((buf == 7.0).all())


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_moe_bad_rows_reach_nothing_else(torch, okq, rows):
    e = Experts(torch, okq, 5, 512, 256, Q4_K, Q6_K)
    x = torch.randn(rows, 512, generator=_gen(torch, rows), device="cuda")
    ids, weights = _pairs(torch, rows, 5, 2, 6)
    clean = e(torch, okq, x, ids, weights)
    x[0, 100] = math.inf
    x[rows - 1, 511] = math.nan
    got = e(torch, okq, x, ids, weights)
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[rows - 1]).all())
    assert torch.equal(got[1:rows - 1], clean[1:rows - 1])


@pytest.mark.parametrize("rows", [2, 300])
def test_moe_scales_exactly_with_powers_of_two(torch, okq, rows):
    """gate is linear in nothing, but a zero up leaves zeros, and weights scale the outputs exactly."""
    e = Experts(torch, okq, 4, 256, 256, Q4_K, Q6_K)
    x = torch.randn(rows, 256, generator=_gen(torch, 1), device="cuda")
    ids, weights = _pairs(torch, rows, 4, 2, 6)
    one = e(torch, okq, x, ids, weights)
    assert torch.equal(e(torch, okq, x, ids, weights * 2.0 ** -30), one * 2.0 ** -30)
    x.zero_()
    assert not bool(e(torch, okq, x, ids, weights).any())


@pytest.mark.parametrize("rows", [1, 20, 500])
def test_moe_is_deterministic(torch, okq, rows):
    e = Experts(torch, okq, 12, 512, 512, Q4_K, Q6_K)
    x = torch.randn(rows, 512, generator=_gen(torch, 1), device="cuda")
    ids, weights = _pairs(torch, rows, 12, 3, 6)
    first = e(torch, okq, x, ids, weights)
    for _ in range(5):
        assert torch.equal(e(torch, okq, x, ids, weights), first)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -20, 2.0 ** 10])
def test_moe_small_and_large_activations(torch, okq, scale):
    """A row's power of two goes into its planes' scale."""
    for rows in (4, 200):
        e = Experts(torch, okq, 3, 256, 256, Q5_K, Q8_0)
        x = torch.randn(rows, 256, generator=_gen(torch, 1), device="cuda") * scale
        ids, weights = _pairs(torch, rows, 3, 2, 6)
        want, far = e.want(torch, x, ids, weights)
        _within(e(torch, okq, x, ids, weights), want, far + 2.0 ** -140, "out")


# ---- together ----------------------------------------------------------------------

def _layer(torch, okq, e, router, norms, x, attn, out, scratch, stream):
    """norm and sum behind attention, router, experts, norm and sum behind them: one sparse layer's second half."""
    rows, hidden = x.shape
    ids, weights, normed, y, after = scratch
    okq.call("okq_residual_norm", x.data_ptr(), hidden, attn.data_ptr(), hidden, rows, hidden, norms[0].data_ptr(), None,
             0, 1.0, 1.0, norms[1].data_ptr(), EPS, after.data_ptr(), hidden, normed.data_ptr(), F32, hidden, stream)
    okq.call("okq_moe_route", normed.data_ptr(), hidden, rows, hidden, F32, router.data_ptr(), e.experts, None, 0, None,
             1, 1, 1, ids.shape[1], 1, 1.0, ids.data_ptr(), weights.data_ptr(), None, stream)
    e(torch, okq, normed, ids, weights, out=y, stream=stream)
    okq.call("okq_residual_norm", after.data_ptr(), hidden, y.data_ptr(), hidden, rows, hidden, norms[2].data_ptr(), None,
             0, 1.0, 1.0, norms[3].data_ptr(), EPS, after.data_ptr(), hidden, out.data_ptr(), F32, hidden, stream)


def _layer_want(torch, e, router, norms, x, attn, ids):
    """With the kernel's experts, which are the best up to what n in f32 leaves open."""
    def rms(v, w):
        return v / (v.square().mean(1, keepdim=True) + EPS).sqrt() * w.double()
    y = x.double() + rms(attn.double(), norms[0])
    n = rms(y, norms[1])
    p = torch.softmax(n @ router.double().t().contiguous(), 1)
    chosen = p.gather(1, ids.long())
    rest = p.scatter(1, ids.long(), 0.0)
    assert bool((chosen.amin(1) >= rest.amax(1) * (1 - 2.0 ** -14)).all())
    w = chosen / chosen.sum(1, keepdim=True)
    out, _ = _moe_want(torch, n, ids, w, e.gate_f, e.up_f, e.down_f)
    y = y + rms(out, norms[2])
    return y, rms(y, norms[3])


def _layer_inputs(torch, okq, rows, hidden=512, inner=256, experts=24, k=4, seed=1):
    e = Experts(torch, okq, experts, hidden, inner, Q4_K, Q6_K)
    g = _gen(torch, seed)
    router = torch.randn(experts, hidden, generator=g, device="cuda") * 2 * hidden ** -0.5
    norms = [torch.randn(hidden, generator=g, device="cuda") * 0.1 + 1 for _ in range(4)]
    x, attn = (torch.randn(rows, hidden, generator=g, device="cuda") for _ in range(2))
    out = torch.empty(rows, hidden, device="cuda")
    scratch = (torch.empty(rows, k, dtype=torch.int32, device="cuda"), torch.empty(rows, k, device="cuda"),
               *(torch.empty(rows, hidden, device="cuda") for _ in range(3)))
    return e, router, norms, x, attn, out, scratch


@pytest.mark.parametrize("rows", [1, 13, 260])
def test_a_sparse_layer(torch, okq, rows):
    """The operators one after the other, as a layer runs them: 2^-17 of the norm's rows of deviation 1 covers the
    experts' own bound (some 2^-19 here) and the norm behind them, which divides by their rms."""
    e, router, norms, x, attn, out, scratch = _layer_inputs(torch, okq, rows)
    _layer(torch, okq, e, router, norms, x, attn, out, scratch, _stream(torch))
    y, n = _layer_want(torch, e, router, norms, x, attn, scratch[0])
    _within(scratch[4], y, torch.full_like(y, 2.0 ** -15), "sum")
    _within(out, n, torch.full_like(n, 2.0 ** -15), "normed")


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_a_captured_layer_replays(torch, okq, rows):
    """Captured once, replayed on new inputs with eager calls between, each replay equal to the eager result."""
    e, router, norms, x, attn, out, scratch = _layer_inputs(torch, okq, rows)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _layer(torch, okq, e, router, norms, x, attn, out, scratch, s.cuda_stream)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            _layer(torch, okq, e, router, norms, x, attn, out, scratch, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for i in range(4):
        g = _gen(torch, 50 + i)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        attn.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        again, more = torch.empty_like(out), tuple(torch.empty_like(t) for t in scratch)
        _layer(torch, okq, e, router, norms, x, attn, again, more, _stream(torch))
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(scratch[0], more[0]) and torch.equal(scratch[4], more[4])


def test_two_streams_at_once(torch, okq):
    """Each stream has a workspace of its own."""
    jobs = [_layer_inputs(torch, okq, rows, seed=s) for rows, s in ((60, 2), (60, 3))]
    alone = []
    for j in jobs:
        e, router, norms, x, attn, out, scratch = j
        _layer(torch, okq, e, router, norms, x, attn, out, scratch, _stream(torch))
        alone.append(out.clone())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        for (e, router, norms, x, attn, out, scratch), s in zip(jobs, streams):
            _layer(torch, okq, e, router, norms, x, attn, out, scratch, s.cuda_stream)
    torch.cuda.synchronize()
    for j, a in zip(jobs, alone):
        assert torch.equal(j[5], a)


def test_a_larger_call_makes_room_for_a_smaller_captured_one(torch, okq):
    """Whatever kernels the two take: on a fresh stream, a call of many rows, then captures of fewer."""
    e, router, norms, x, attn, out, scratch = _layer_inputs(torch, okq, 5000, hidden=4096, inner=256, experts=8, k=2)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _layer(torch, okq, e, router, norms, x, attn, out, scratch, s.cuda_stream)
        s.synchronize()
        for rows in (1, 17, 100, 600):
            part = [x[:rows], attn[:rows], out[:rows], tuple(t[:rows] for t in scratch)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                _layer(torch, okq, e, router, norms, *part, torch.cuda.current_stream().cuda_stream)
            graph.replay()
            s.synchronize()
            again, more = torch.empty_like(part[2]), tuple(torch.empty_like(t) for t in part[3])
            _layer(torch, okq, e, router, norms, part[0], part[1], again, more, s.cuda_stream)
            s.synchronize()
            assert torch.equal(out[:rows], again)


def test_moe_in_several_passes(torch, okq):
    """More pairs than a pass takes, streamed and sorted: rows of a first and of a last pass, and of a batch of their own."""
    for rows, experts, k in ((9000, 8, 8), (1100, 4000, 64)):  # 72000 pairs; 70400 pairs of many experts
        hidden, inner = 64, 32
        e = Experts(torch, okq, experts, hidden, inner, Q8_0, Q8_0)
        x = torch.randn(rows, hidden, generator=_gen(torch, 3), device="cuda")
        ids = torch.randint(-1, experts, (rows, k), generator=_gen(torch, 4), device="cuda").int()
        weights = torch.rand(rows, k, generator=_gen(torch, 5), device="cuda") / k
        got = e(torch, okq, x, ids, weights)
        for at in (0, rows // 2, rows - 24):
            part = slice(at, at + 24)
            _within(got[part], *e.want(torch, x[part], ids[part], weights[part]), "out")


@pytest.mark.parametrize("rows", [3, 56000])
def test_moe_stacks_beyond_4_gib(torch, okq, rows):
    """The last two of 2000 experts, 4.7 GB into their stacks; what the others hold is not read."""
    experts, hidden, inner = 2000, 2048, 2048
    e = Experts(torch, okq, 2, hidden, inner, Q4_K, Q4_K)
    x = torch.randn(rows, hidden, generator=_gen(torch, 1), device="cuda")
    ids, weights = _pairs(torch, rows, 2, 1, 3)
    want, far = e.want(torch, x, ids, weights)
    for name in ("gate", "up", "down"):
        stack = torch.full((experts // 2, getattr(e, name).numel()), 0xFF, dtype=torch.uint8, device="cuda")
        stack[-1] = getattr(e, name)
        setattr(e, name, stack.view(-1))
    assert e.gate.numel() > 1 << 32
    e.experts = experts
    _within(e(torch, okq, x, ids + experts - 2, weights), want, far, "out")


def test_two_host_threads_on_one_stream(torch, okq):
    """Each call's launches go in as one sequence, so the stream's workspaces serve one call at a time."""
    import threading
    jobs = [_layer_inputs(torch, okq, 60, seed=s) for s in (2, 3)]
    alone, stream = [], torch.cuda.Stream()
    for e, router, norms, x, attn, out, scratch in jobs:
        _layer(torch, okq, e, router, norms, x, attn, out, scratch, stream.cuda_stream)
        torch.cuda.synchronize()
        alone.append(out.clone())

    def work(job):
        e, router, norms, x, attn, out, scratch = job
        for _ in range(20):
            _layer(torch, okq, e, router, norms, x, attn, out, scratch, stream.cuda_stream)
    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for j, a in zip(jobs, alone):
        assert torch.equal(j[5], a)


@pytest.mark.parametrize("case", [
    (1, 4096, 2560, 8, 2, Q6_K, Q4_K),      # one row, its items in two slices each way
    (2, 2304, 4608, 16, 2, Q5_K, Q6_K),     # nine items in slices of five and four, eighteen in three of six
    (1, 288, 8480, 5, 3, Q8_0, Q8_0),       # 33 and a half items: slices of seven and six, the last one cut
    (4, 1280, 768, 128, 8, Q4_K, Q5_K),     # rows that share some experts, unsorted
    (64, 2560, 256, 3, 1, Q5_K, Q4_K),      # more than 16 rows an expert
    (130, 4352, 1280, 2, 2, Q8_0, Q6_K),    # tiles of 128 and of 2 rows
], ids=str)
def test_moe_of_long_rows(torch, okq, case):
    rows, hidden, inner, experts, k, gu, dn = case
    e = Experts(torch, okq, experts, hidden, inner, gu, dn)
    x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
    ids, weights = _pairs(torch, rows, experts, k, 11)
    _within(e(torch, okq, x, ids, weights), *e.want(torch, x, ids, weights), "out")


def test_moe_rows_do_not_depend_on_each_other(torch, okq):
    """Alone (not sorted), in a batch (sorted), in another one: the same bits; so in batches of tiles."""
    e = Experts(torch, okq, 6, 512, 768, Q4_K, Q6_K)
    x = torch.randn(900, 512, generator=_gen(torch, 2), device="cuda")
    ids, weights = _pairs(torch, 900, 6, 2, 6)
    some = e(torch, okq, x[:70], ids[:70], weights[:70])
    assert torch.equal(e(torch, okq, x[20:60], ids[20:60], weights[20:60]), some[20:60])
    for r in (0, 33, 69):
        assert torch.equal(e(torch, okq, x[r:r + 1], ids[r:r + 1], weights[r:r + 1])[0], some[r])
    many = e(torch, okq, x, ids, weights)
    assert torch.equal(e(torch, okq, x[100:500], ids[100:500], weights[100:500]), many[100:500])


@pytest.mark.parametrize("rows", [2, 50, 400])
def test_moe_rows_without_experts_may_hold_anything(torch, okq, rows):
    e = Experts(torch, okq, 4, 256, 256, Q8_0, Q5_K)
    x = torch.randn(rows, 256, generator=_gen(torch, 2), device="cuda")
    ids, weights = _pairs(torch, rows, 4, 2, 6)
    clean = e(torch, okq, x, ids, weights)
    x[1] = math.nan
    x[rows - 1, 3] = math.inf
    weights[[1, rows - 1]] = math.inf
    ids[[1, rows - 1]] = -7
    got = e(torch, okq, x, ids, weights)
    assert not bool(got[1].any()) and not bool(got[rows - 1].any())
    assert torch.equal(got[2:rows - 1], clean[2:rows - 1]) and torch.equal(got[0], clean[0])


@pytest.mark.parametrize("behind", [0x7E00, 0xFC00, 0x7BFF], ids=["nan", "infinity", "largest"])
@pytest.mark.parametrize("rows", [1, 20, 400])
def test_moe_rows_of_q8_end_at_their_own_blocks(torch, okq, rows, behind):
    """Rows that are no multiple of 256 values: whatever the blocks behind them hold, the next expert's and the next
    row's, changes no bit."""
    for hidden, inner in ((288, 352), (32, 96), (1312, 2592)):
        e = Experts(torch, okq, 5, hidden, inner, Q8_0, Q8_0)
        x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
        ids, weights = _pairs(torch, rows, 3, 2, 8)
        ids *= 2  # experts 1 and 3 have no rows
        clean = e(torch, okq, x, ids, weights)
        _within(clean, *e.want(torch, x, ids, weights), "out")
        block = torch.tensor([behind & 255, behind >> 8] + [127] * 32, dtype=torch.uint8, device="cuda")
        for name in ("gate", "up", "down"):
            getattr(e, name).view(5, -1, 34)[1::2] = block
        assert torch.equal(e(torch, okq, x, ids, weights), clean)
        at = hidden // 2  # one output of expert 2 whose own weights are such blocks
        e.down.view(5, hidden, -1, 34)[2, at] = block
        got = e(torch, okq, x, ids, weights)
        keep = torch.arange(hidden, device="cuda") != at
        assert torch.equal(got[:, keep], clean[:, keep])
        used = (ids == 2).any(1)
        assert torch.equal(got[~used], clean[~used])
        if behind != 0x7BFF:
            assert not bool(torch.isfinite(got[used, at]).any())


@pytest.mark.parametrize("rows", [1, 20, 400])
@pytest.mark.parametrize("hidden,inner", [(512, 256), (288, 1312)])
def test_moe_q8_of_large_scales(torch, okq, rows, hidden, inner):
    """Blocks up to the largest scale and code beside ordinary ones: within the bound; and bit for bit those of
    ordinary scales alone, where what meets the others is zero."""
    e = Experts(torch, okq, 5, hidden, inner, Q8_0, Q8_0)
    x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
    ids, weights = _pairs(torch, rows, 5, 2, 8)
    loud = torch.arange(hidden, device="cuda") // 32 % 4 == 1
    x[:, loud] = 0.0
    clean = e(torch, okq, x, ids, weights)
    g = _gen(torch, 7)
    for name, columns in (("gate", hidden), ("up", hidden), ("down", inner)):
        blocks = getattr(e, name).view(-1, columns // 32, 34)
        at = torch.arange(columns // 32, device="cuda") % 4 == 1
        if name == "down":  # some rows, which gives those outputs alone other values
            blocks = blocks[::7]
        d = torch.rand(blocks[:, at, 0].shape, generator=g, device="cuda") * 65000 + 200
        d[..., 0] = 65504.0
        q = torch.randint(0, 256, (*d.shape, 32), generator=g, device="cuda").to(torch.uint8)
        q[..., 0] = 128
        blocks[:, at] = torch.cat([d.half().view(torch.uint8).view(*d.shape, 2), q], -1)
        okq.call("okq_dequantize", Q8_0, getattr(e, name).data_ptr(), getattr(e, name + "_f").numel(),
                 getattr(e, name + "_f").data_ptr(), _stream(torch))
    got = e(torch, okq, x, ids, weights)
    _within(got, *e.want(torch, x, ids, weights), "out")
    small = (e.down_f.abs().amax((0, 2)) < 10.0)  # outputs that no expert's large blocks reach
    assert bool(small.any()) and torch.equal(got[:, small], clean[:, small])
    x[:, loud] = torch.randn(rows, int(loud.sum()), generator=g, device="cuda")
    _within(e(torch, okq, x, ids, weights), *e.want(torch, x, ids, weights), "out")


@pytest.mark.parametrize("rows", [(1 << 26) - 16, (1 << 26) - 15, 1 << 26])
def test_route_of_the_most_rows(torch, okq, rows):
    """2^26 rows are 2^22 tiles: of 1024 threads each they would be more than a launch has."""
    x = torch.randn(rows, 1, generator=_gen(torch, 1), device="cuda")
    w = torch.tensor([[1.0], [-1.0], [0.5]], device="cuda")
    ids, weights, _ = _route(torch, okq, x, 1, w, F32, None, None, True, 1, 1, 1, 1, False, 1.0, logits=False)
    want = (x[:, 0] < 0).int()
    assert torch.equal(ids[:, 0], want)
    off = (weights[:, 0] - torch.sigmoid(x[:, 0].abs().double())).abs()
    assert float(off.max()) <= U  # below 1: half a step is 2^-25, and torch's own f64


@pytest.mark.parametrize("case", [  # as ROUTE: whole rows a workgroup, in more than one round of 128 experts
    (2100, 256, 256, 8, True, 8, 4, 2, False, True, True, F32, 0),
    (2049, 130, 500, 10, False, 1, 1, 1, True, False, True, BF16, 1),
    (2033, 64, 129, 5, False, 3, 2, 1, False, True, False, F32, 0),
    (2050, 96, 512, 64, True, 64, 9, 2, True, True, True, F16, 4),
], ids=lambda c: str(c[:4]))
def test_route_of_many_rows_and_experts(torch, okq, case):
    args = _route_inputs(torch, case)
    got = _route(torch, okq, *args)
    x, _, w, _, b, c, *rest = args
    _check_route(torch, got, _route_want(torch, x, w, b, c, *rest), x, w)
    for n in (1, 300):  # split over expert tiles: the same experts
        some = _route(torch, okq, x[:n], *args[1:])
        assert torch.equal(some[0], got[0][:n])
        assert bool(((some[1] - got[1][:n]).abs() <= 2 * U * got[1][:n]).all())


@pytest.mark.parametrize("rows,k,experts,gu,dn", [
    (1, 64, 128, Q4_K, Q6_K),  # one row that names one expert 64 times
    (40, 1, 128, Q8_0, Q4_K),  # all rows with one expert, not sorted
    (8, 8, 128, Q6_K, Q5_K),   # all rows with the same eight
    (13, 4, 104, Q5_K, Q8_0),
])
def test_moe_pairs_of_few_experts_not_sorted(torch, okq, rows, k, experts, gu, dn):
    """An expert of more than 16 pairs goes in turns where nothing is sorted."""
    e = Experts(torch, okq, experts, 512, 768, gu, dn)
    x = torch.randn(rows, 512, generator=_gen(torch, rows), device="cuda")
    _, weights = _pairs(torch, rows, experts, k, 4)
    few = 1 if k in (1, 64) else k
    ids = (torch.arange(rows * k, device="cuda") % few * 11 + 7).int().view(rows, k)
    got = e(torch, okq, x, ids, weights)
    _within(got, *e.want(torch, x, ids, weights), "out")


def _off(k):
    """A product's relative error in root mean square over K values of independent sign: planes 2^-21 of each (the
    worst of all), sums as a random walk of K / 8 additions."""
    return 2.0 ** -21 + U * math.sqrt(k / 8)


@pytest.mark.parametrize("kind", [Q8_0, Q4_K, Q5_K, Q6_K])
@pytest.mark.parametrize("rows,hidden,inner,experts", [
    (1, 512, 768, 8), (24, 768, 512, 40), (9, 4352, 8704, 4),            # streamed: unsorted, sorted, in slices
    (300, 512, 256, 8), (400, 4352, 5120, 3), (200, 2048, 14336, 2)])    # tiles, of long rows too
def test_moe_is_as_near_as_its_planes(torch, okq, kind, rows, hidden, inner, experts):
    """The whole error beside the whole result: one plane of activations less would be 2^-12 of it.

    Q4_K and Q5_K sum q and the min apart: q's mean is 2.7 of its deviations, so each of the two sums is up to 2.9
    times the result, together 4.  silu's slope of at most 1.1 against its root mean square of 0.6 at deviation 1, and
    the factor up, make 3 of one product's error in the gated values, taken as 4."""
    e = Experts(torch, okq, experts, hidden, inner, kind, kind)
    x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
    ids, weights = _pairs(torch, rows, experts, 2, 12)
    want, _ = e.want(torch, x, ids, weights)
    got = e(torch, okq, x, ids, weights)
    off = float((got - want).square().mean().sqrt() / want.square().mean().sqrt())
    bound = (4 if kind in (Q4_K, Q5_K) else 1) * (4 * _off(hidden) + _off(inner))
    assert off <= bound, (off, bound)


@pytest.mark.parametrize("kind", [Q8_0, Q4_K, Q5_K, Q6_K])
@pytest.mark.parametrize("rows", [1, 30, 400])
def test_moe_bad_blocks_stay_in_their_outputs(torch, okq, kind, rows):
    """A block of weights that is no number: one output of down; every output where gate or up has it; of its expert's
    rows alone.  Experts without rows may hold anything."""
    hidden, inner = 768, 512
    e = Experts(torch, okq, 5, hidden, inner, kind, kind)
    x = torch.randn(rows, hidden, generator=_gen(torch, rows), device="cuda")
    ids, weights = _pairs(torch, rows, 3, 2, 8)
    ids *= 2
    clean = e(torch, okq, x, ids, weights)
    for name in ("gate", "up", "down"):
        getattr(e, name).view(5, -1)[1::2] = 0xFF
    assert torch.equal(e(torch, okq, x, ids, weights), clean)
    used = (ids == 2).any(1)
    elems, size = BYTES[kind]
    for name, outputs, columns in (("down", hidden, inner), ("gate", inner, hidden), ("up", inner, hidden)):
        blocks = getattr(e, name).view(5, outputs, columns // elems, size)
        at = outputs - 1  # beside the next expert's
        held = blocks[2, at, -1].clone()
        blocks[2, at, -1] = 0xFF
        got = e(torch, okq, x, ids, weights)
        blocks[2, at, -1] = held
        assert torch.equal(got[~used], clean[~used])
        if name == "down":
            keep = torch.arange(hidden, device="cuda") != at
            assert torch.equal(got[:, keep], clean[:, keep]) and bool(torch.isnan(got[used, at]).all())
        else:
            assert bool(torch.isnan(got[used]).all())
