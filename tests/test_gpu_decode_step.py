"""okq_qk_norm_rope, okq_paged_attention and okq_logits_process against their
definitions in 64 bits (needs an MI355X).

Bounds, derived before the first run.  u = 2^-24 is half a step of f32.
  rotation: cosine and sine are off by at most 2u (a remainder rounded once, a
    series, a rounding), the norm's factor by at most 12u relative (squares
    and sums of at most 512 values in a tree, square root, reciprocal), each
    product and sum by u: 16u (|y_a| + |y_b|); a cache adds half a step of its
    type (and f16's half step of 2^-24 below its normal range).
  scores: head_dim products and sums, whose roundings add up like a random
    walk: 8 deviations, e = 8u scale sum |q K| (+ 4u |s| for the scale and the
    base of the exponential, + 8u softcap where capped, whose slope is at most 1).
  outputs: each weight is off by 2e + 8u relative, and T of them are summed:
    (2e + 8u + 8u sqrt(T)) sum p |V| / sum p.  lse: e + 8u (1 + sqrt(T) + |lse|).
  logits: five operations: 5u (|x| rep + |x| + freq n + pres + |bias|).
"""
import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16, Q8_0 = 0, 1, 30, 8
TYPES = {"F32": F32, "F16": F16, "BF16": BF16, "Q8_0": Q8_0}


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


def _row_bytes(t, d):
    return {F32: 4 * d, F16: 2 * d, BF16: 2 * d, Q8_0: d // 32 * 34}[t]


def _dtype(torch, t):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[t]


def _decode(torch, t, rows, d):
    """Rows of cache bytes [..., row bytes] as f64 [..., d] (CPU)."""
    if t != Q8_0:
        return rows.contiguous().view(_dtype(torch, t)).double()
    b = rows.reshape(*rows.shape[:-1], d // 32, 34)
    return (b[..., :2].contiguous().view(torch.float16).double() * b[..., 2:].contiguous().view(torch.int8).double()
            ).reshape(*rows.shape[:-1], d)


def _encode(torch, okq, t, x):
    """f32 values [..., d] (GPU) as cache bytes [..., row bytes]."""
    if t != Q8_0:
        return x.to(_dtype(torch, t)).view(torch.uint8)
    x = x.contiguous()
    out = torch.empty(x.numel() // 32 * 34, dtype=torch.uint8, device="cuda")
    okq.call("okq_quantize", Q8_0, x.data_ptr(), x.numel(), out.data_ptr(), _stream(torch))
    return out.view(*x.shape[:-1], -1)


class Cache:
    """Pages filled with `filler` bytes, laid out head by head or token by
    token, `offset` bytes into their allocations and with `pad` bytes a row."""

    def __init__(self, torch, okq, t, n_pages, page, heads, d, token_major=False, offset=0, pad=0, filler=0xFF):
        row = _row_bytes(t, d) + pad
        self.row, self.t, self.d, self.heads, self.page, self.n_pages = _row_bytes(t, d), t, d, heads, page, n_pages
        self.ts, self.hs = (heads * row, row) if token_major else (row, page * row)
        self.ps = heads * page * row
        self.buf = torch.full((2, n_pages * self.ps + offset), filler, dtype=torch.uint8, device="cuda")
        self.views = [b[offset:].as_strided((n_pages, heads, page, self.row), (self.ps, self.hs, self.ts, 1),
                                            b.storage_offset() + offset) for b in self.buf]
        self.c = okq.KvPages(type=t, n_pages=n_pages, page_tokens=page, kv_heads=heads, head_dim=d,
                             page_stride=self.ps, head_stride=self.hs, token_stride=self.ts,
                             k=self.views[0].data_ptr(), v=self.views[1].data_ptr())

    def ref(self):
        return ctypes.byref(self.c)


# ---- the step before attention --------------------------------------------------

ROPE = [  # tokens, q_heads, kv_heads, head_dim, rotary, type, page, interleaved, norm, far
    (1, 32, 8, 128, 128, "BF16", 16, True, False, 100000),
    (5, 6, 2, 80, 40, "F16", 24, False, True, 0),
    (7, 3, 3, 64, 64, "F32", 8, False, True, 30000),
    (4, 8, 2, 256, 128, "F16", 100, False, True, 1 << 20),
    (3, 8, 4, 112, 112, "BF16", 16, True, True, 200000),
    (9, 5, 1, 96, 48, "BF16", 1, True, False, 77),
    (2, 2, 1, 33, 32, "F32", 5, False, True, 1000),
    (2, 2, 1, 7, 2, "F16", 5, True, False, 1000),
    (3, 4, 2, 512, 256, "BF16", 16, False, True, 5000),
    (3, 4, 2, 128, 0, "BF16", 16, False, True, 0),
    (300, 12, 4, 128, 128, "BF16", 16, False, True, 0),
    (301, 9, 3, 128, 128, "Q8_0", 32, True, True, 0),
    (3, 4, 2, 96, 48, "Q8_0", 24, False, False, 999),
    (2, 8, 8, 256, 256, "Q8_0", 8, False, True, 100000),
    (1100, 7, 1, 64, 64, "F32", 64, True, False, 4000),
]


def _rope_inputs(torch, n, hq, hkv, d, rotary, page, norm, far, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(n, (hq + 2 * hkv) * d, generator=g, device="cuda")
    n_pages = n // page + 3
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:n]
    pos = torch.randint(0, far + 1, (n,), generator=g, device="cuda").int() if far else torch.arange(n, device="cuda").int()
    if far:
        pos[0] = far
    freq = (500000.0 ** (-torch.arange(rotary // 2, device="cuda").double() / max(1, rotary // 2))).float()
    w = [torch.randn(d, generator=g, device="cuda") * 0.2 + 1 if norm else None for _ in range(2)]
    return x, n_pages, slots, pos, freq, w


def _rope_want(torch, x, w, eps, pos, freq, rotary, interleaved):
    """[tokens, heads, d] in f64, and the bound's |y_a| + |y_b|."""
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = rotary // 2
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    ang = (pos.double()[:, None] * freq.double())[:, None]
    u, v = y[..., a], y[..., b]
    out, size = y.clone(), y.abs()
    out[..., a], out[..., b] = u * ang.cos() - v * ang.sin(), v * ang.cos() + u * ang.sin()
    size[..., a] = size[..., b] = u.abs() + v.abs()
    return out, size


@pytest.mark.parametrize("case", ROPE, ids=[f"{c[0]}x{c[1]}+{c[2]}x{c[3]}r{c[4]}{c[5]}" for c in ROPE])
def test_rope_and_cache(torch, okq, case):
    n, hq, hkv, d, rotary, tn, page, inter, norm, far = case
    print(f"[gpu] rope {case}", flush=True)
    t, eps = TYPES[tn], 1e-6
    x, n_pages, slots, pos, freq, w = _rope_inputs(torch, n, hq, hkv, d, rotary, page, norm, far, 11 + d)
    if n > 2:
        slots[1], slots[2] = -1, n_pages * page  # not stored
    cache = Cache(torch, okq, t, n_pages, page, hkv, d, token_major=d % 3 == 0)
    before = [v.cpu().clone() for v in cache.views]
    q_out, k_out = torch.full((n, hq, d), math.nan, device="cuda"), torch.full((n, hkv, d), math.nan, device="cuda")
    p, width = x.data_ptr(), (hq + 2 * hkv) * d
    okq.call("okq_qk_norm_rope", p, width, p + 4 * hq * d, width, p + 4 * (hq + hkv) * d, width, n, hq, hkv, d,
             _ptr(w[0]), _ptr(w[1]), eps, _ptr(pos), _ptr(freq) if rotary else None, rotary, int(inter),
             q_out.data_ptr(), hq * d, k_out.data_ptr(), hkv * d, cache.ref(), slots.data_ptr(), _stream(torch))
    torch.cuda.synchronize()
    xc = x.cpu().view(n, -1, d)
    ws = [None if v is None else v.cpu() for v in w]
    q, qs = _rope_want(torch, xc[:, :hq], ws[0], eps, pos.cpu(), freq.cpu(), rotary, inter)
    k, ks = _rope_want(torch, xc[:, hq:hq + hkv], ws[1], eps, pos.cpu(), freq.cpu(), rotary, inter)
    assert ((q_out.cpu().double() - q).abs() <= 16 * U * qs + 1e-40).all()
    assert ((k_out.cpu().double() - k).abs() <= 16 * U * ks + 1e-40).all()
    # the cache holds exactly the call's own keys, and the values, in its type
    for view, was, rows in ((cache.views[0], before[0], k_out), (cache.views[1], before[1], x.view(n, -1, d)[:, hq + hkv:])):
        want = was.clone()
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < n_pages * page:
                want[s // page, :, s % page] = _encode(torch, okq, t, rows[i]).cpu()
        assert torch.equal(view.cpu(), want)


@pytest.mark.parametrize("d,rotary,tn,offset", [(128, 128, "BF16", 2), (128, 64, "F16", 6), (64, 64, "F32", 4),
                                                (128, 128, "Q8_0", 2), (120, 60, "BF16", 0), (68, 68, "F32", 0)])
def test_rope_of_odd_places(torch, okq, d, rotary, tn, offset):
    """Rows at 4-byte addresses, odd strides, padded cache rows at odd offsets,
    and queries turned in place: the same values as from aligned rows."""
    print(f"[gpu] rope odd {d} {rotary} {tn} {offset}", flush=True)
    n, hq, hkv, page, t = 6, 4, 2, 8, TYPES[tn]
    x, n_pages, slots, pos, freq, w = _rope_inputs(torch, n, hq, hkv, d, rotary, page, True, 5000, 7)

    def run(stride, shift, off, pad, inplace):
        buf = torch.zeros(n * stride + 8, device="cuda")
        at = buf[shift:shift + n * stride].view(n, stride)
        at[:, :x.shape[1]] = x
        cache = Cache(torch, okq, t, n_pages, page, hkv, d, offset=off, pad=pad, filler=0)
        q_out = at if inplace else torch.empty(n, hq * d, device="cuda")
        okq.call("okq_qk_norm_rope", at.data_ptr(), stride, at.data_ptr() + 4 * hq * d, stride,
                 at.data_ptr() + 4 * (hq + hkv) * d, stride, n, hq, hkv, d, _ptr(w[0]), _ptr(w[1]), 1e-6, _ptr(pos),
                 _ptr(freq), rotary, 0, q_out.data_ptr(), stride if inplace else hq * d, None, 0, cache.ref(),
                 slots.data_ptr(), _stream(torch))
        torch.cuda.synchronize()
        return q_out[:, :hq * d].clone(), [v.clone() for v in cache.views]

    q0, c0 = run(x.shape[1], 0, 0, 0, False)
    q1, c1 = run(x.shape[1] + 3, 1, offset, 4 if tn == "F32" else 2, True)
    # rows that no vector load reaches sum their squares in another order: 2 x 12u
    assert ((q0 - q1).double().abs() <= 2 * 16 * U * (2 * q0.double().abs().amax())).all()
    for a, b in zip(c0, c1):
        da, db = (_decode(torch, t, v.cpu(), d) for v in (a, b))
        step = {F32: 0.0, F16: 2.0 ** -10, BF16: 2.0 ** -7, Q8_0: 0.0}[t]
        block = da.abs().amax() / 100 if t == Q8_0 else 0.0  # one code
        assert ((da - db).abs() <= step * da.abs() + 32 * U * da.abs().amax() * 2 + block).all()


def test_rope_without_a_cache_and_with_its_norms_apart(torch, okq):
    n, hq, hkv, d = 3, 4, 2, 64
    x, _, _, pos, freq, w = _rope_inputs(torch, n, hq, hkv, d, d, 16, True, 0, 3)
    xc = x.cpu().view(n, -1, d)
    for qn, kn in ((w[0], None), (None, w[1])):
        q, k = torch.empty(n, hq, d, device="cuda"), torch.empty(n, hkv, d, device="cuda")
        okq.call("okq_qk_norm_rope", x.data_ptr(), (hq + 2 * hkv) * d, x.data_ptr() + 4 * hq * d, (hq + 2 * hkv) * d,
                 None, 0, n, hq, hkv, d, _ptr(qn), _ptr(kn), 1e-6, _ptr(pos), _ptr(freq), d, 0, q.data_ptr(), hq * d,
                 k.data_ptr(), hkv * d, None, None, _stream(torch))
        torch.cuda.synchronize()
        for got, rows, ww in ((q, xc[:, :hq], qn), (k, xc[:, hq:hq + hkv], kn)):
            want, size = _rope_want(torch, rows, None if ww is None else ww.cpu(), 1e-6, pos.cpu(), freq.cpu(), d, False)
            assert ((got.cpu().double() - want).abs() <= 16 * U * size).all()


# ---- attention over pages ---------------------------------------------------------

ATTN = [  # type, head_dim, kv_heads, group, page, lengths, window, softcap, token_major
    ("BF16", 128, 8, 4, 16, [517], 0, 0.0, False),
    ("BF16", 128, 2, 4, 16, [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000], 0, 0.0, False),
    ("BF16", 128, 1, 1, 24, [23, 24, 25, 2000], 0, 0.0, True),
    ("BF16", 80, 3, 5, 100, [7, 250, 0], 0, 30.0, False),
    ("BF16", 96, 2, 12, 8, [300, 2, 45], 40, 0.0, True),
    ("BF16", 112, 2, 3, 1, [1, 33, 70], 0, 0.0, False),
    ("BF16", 64, 4, 8, 64, [777, 64], 100, 50.0, False),
    ("BF16", 256, 2, 4, 32, [500, 31, 0], 0, 0.0, False),
    ("BF16", 512, 1, 4, 16, [100, 17], 0, 0.0, False),
    ("BF16", 128, 1, 40, 16, [200, 3], 0, 0.0, False),
    ("F16", 128, 2, 4, 16, [517, 0, 64], 0, 0.0, False),
    ("F16", 256, 2, 4, 64, [3000, 1025, 1024, 1023, 1], 1024, 50.0, False),
    ("F16", 80, 4, 1, 24, [100, 49], 1, 0.0, True),
    ("F16", 33, 2, 2, 7, [50, 8], 0, 0.0, False),
    ("F32", 80, 5, 1, 24, [1500, 0, 25], 0, 0.0, False),
    ("F32", 128, 2, 6, 16, [333, 1], 0, 30.0, True),
    ("F32", 64, 2, 2, 100, [99, 100, 101, 201], 17, 0.0, False),
    ("F32", 256, 1, 8, 8, [200, 9], 0, 0.0, False),
    ("F32", 112, 2, 2, 16, [60], 0, 0.0, False),
    ("F32", 1, 2, 2, 16, [60, 5], 0, 0.0, False),
    ("Q8_0", 128, 2, 4, 32, [600, 0, 33], 0, 0.0, False),
    ("Q8_0", 64, 3, 2, 24, [100, 24], 0, 0.0, True),
    ("Q8_0", 96, 1, 5, 16, [77, 300], 64, 20.0, False),
    ("Q8_0", 256, 2, 12, 100, [400, 1], 0, 0.0, False),
    ("Q8_0", 512, 1, 2, 16, [40], 0, 0.0, False),
]


def _attn_inputs(torch, okq, t, d, kv, group, page, lengths, token_major=False, offset=0, pad=0, seed=5):
    """Tokens past a length and pages of nobody hold bytes 0xFF (NaN in every type)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    need = [(n + page - 1) // page for n in lengths]
    n_pages = sum(need) + 2
    cache = Cache(torch, okq, t, n_pages, page, kv, d, token_major, offset, pad)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(max(need), 1) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for i, n in enumerate(lengths):
        for j in range(need[i]):
            table[i, j] = order.pop()
            m = min(page, n - j * page)
            for view in cache.views:
                rows = torch.randn(kv, m, d, generator=g, device="cuda")
                view[int(table[i, j]), :, :m] = _encode(torch, okq, t, rows)
    q = torch.randn(len(lengths), kv * group, d, generator=g, device="cuda") * 2
    return cache, table, q


def _attn_want(torch, cache, table, q, lengths, scale, softcap, window, group, limit=None):
    """out, lse in f64 and their bounds."""
    s, hq, d = q.shape
    K, V = (v.cpu() for v in cache.views)
    out, lse = torch.zeros(s, hq, d, dtype=torch.float64), torch.full((s, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for i, n in enumerate(lengths):
        n = min(n, table.shape[1] * cache.page, n if limit is None else limit)
        at = [j for j in range(max(0, n - window) if window else 0, n)
              if 0 <= int(table[i, j // cache.page]) < cache.n_pages]
        if not at:
            continue
        pg = torch.tensor([int(table[i, j // cache.page]) for j in at])
        sl = torch.tensor([j % cache.page for j in at])
        k, v = (_decode(torch, cache.t, c[pg, :, sl], d).repeat_interleave(group, 1) for c in (K, V))  # [T, hq, d]
        qi = q[i].cpu().double()
        x = (k * qi).sum(-1) * scale
        e = 8 * U * scale * (k * qi).abs().sum(-1) + 4 * U * x.abs()
        if softcap:
            x = softcap * torch.tanh(x / softcap)
            e = e + 8 * U * softcap
        p = torch.softmax(x, 0)
        e = e.amax(0)
        out[i] = (p[..., None] * v).sum(0)
        lse[i] = torch.logsumexp(x, 0)
        root = math.sqrt(len(at))
        tol[i] = (2 * e + 8 * U + 8 * U * root)[:, None] * (p[..., None] * v.abs()).sum(0)
        ltol[i] = e + 8 * U * (1 + root + lse[i].abs())
    return out, lse, tol, ltol


def _attention(torch, okq, cache, table, q, lengths, longest, scale, softcap=0.0, window=0, stream=None, out=None):
    s, hq, d = q.shape
    if out is None:
        out = torch.full((s, hq, d), math.nan, device="cuda")
    lse = torch.full((s, hq), math.nan, device="cuda")
    td, ld = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    okq.call("okq_paged_attention", q.data_ptr(), q.stride(0) if s > 1 else hq * d, s, hq, cache.ref(), td.data_ptr(),
             td.shape[1], ld.data_ptr(), longest, scale, softcap, window, out.data_ptr(),
             out.stride(0) if s > 1 else hq * d, lse.data_ptr(), _stream(torch) if stream is None else stream)
    return out, lse


def _attn_check(torch, got, want):
    (out, lse), (wo, wl, tol, ltol) = got, want
    out, lse = out.cpu().double(), lse.cpu().double()
    empty = wl == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out[empty] == 0).all()
    assert ((out - wo).abs() <= tol).all(), ((out - wo).abs() / tol.clamp(min=1e-300)).max()
    assert ((lse - wl).abs()[~empty] <= ltol[~empty]).all()


@pytest.mark.parametrize("case", ATTN, ids=[f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-p{c[4]}-w{c[6]}" for c in ATTN])
def test_attention(torch, okq, case):
    tn, d, kv, group, page, lengths, window, softcap, tm = case
    print(f"[gpu] attention {case}", flush=True)
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, kv, group, page, lengths, tm)
    scale = 1 / math.sqrt(d)
    got = _attention(torch, okq, cache, table, q, lengths, max(lengths), scale, softcap, window)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, scale, softcap, window, group))


@pytest.mark.parametrize("tn,d,kv,group,lengths", [
    ("BF16", 64, 1, 4, [70001]), ("F16", 64, 2, 1, [20011, 3, 0, 9000]), ("F32", 64, 1, 3, [30000, 1]),
    ("Q8_0", 64, 1, 5, [40013, 100]), ("BF16", 128, 1, 2, [1, 33000] + [5] * 30)])
def test_attention_split_over_a_long_cache(torch, okq, tn, d, kv, group, lengths):
    """One long sequence beside short ones; two calls agree bit for bit."""
    print(f"[gpu] attention long {tn} {d} {lengths[:3]}", flush=True)
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, kv, group, 64, lengths)
    got = [_attention(torch, okq, cache, table, q, lengths, max(lengths), d ** -0.5) for _ in range(2)]
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    _attn_check(torch, got[0], _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, group))


def test_attention_of_many_sequences(torch, okq):
    """More sequences than a workgroup has threads, most of them empty."""
    lengths = [(i * 37) % 50 if i % 3 == 0 else 0 for i in range(1500)]
    cache, table, q = _attn_inputs(torch, okq, BF16, 64, 1, 2, 16, lengths)
    got = _attention(torch, okq, cache, table, q, lengths, 4000, 0.125)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, 0.125, 0.0, 0, 2))


@pytest.mark.parametrize("tn,d,offset,pad", [("BF16", 128, 2, 2), ("F16", 64, 8, 8), ("F32", 128, 4, 4), ("Q8_0", 128, 2, 2),
                                             ("BF16", 120, 0, 0), ("F16", 100, 0, 0), ("F32", 66, 0, 0)])
def test_attention_of_odd_places(torch, okq, tn, d, offset, pad):
    """Cache rows at odd offsets and strides, q and out rows apart and not
    16-byte aligned."""
    print(f"[gpu] attention odd {tn} {d}", flush=True)
    lengths, group, kv = [75, 0, 200], 3, 2
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, kv, group, 16, lengths, offset=offset, pad=pad)
    wide = torch.full((2, 3 * (kv * group * d + 5) + 1), math.nan, device="cuda")
    qs, os = (w[1:].view(3, -1)[:, :kv * group * d].view(3, kv * group, d) for w in wide)
    qs.copy_(q)
    got = _attention(torch, okq, cache, table, qs, lengths, 200, d ** -0.5, out=os)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, group))
    assert wide[1].isnan().sum() == 16  # nothing written between the rows


@pytest.mark.parametrize("tn", ["Q8_0", "F16", "BF16", "F32"])
def test_attention_weights_keep_f32_precision(torch, okq, tn):
    """Hundreds of short sequences with scores near zero: the bound is a few
    steps of f32, so no weight of the 10^5 (tokens, heads, blocks) may lose
    bits, a step of f16 apart (2^-11 of an eighth) least of all."""
    lengths, d, kv, group = [8] * 256, 128, 4, 8
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, kv, group, 8, lengths)
    q = q * 0.1
    got = _attention(torch, okq, cache, table, q, lengths, 8, d ** -0.5)
    torch.cuda.synchronize()
    want = _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, group)
    assert want[2].max() < 2.0 ** -16
    _attn_check(torch, got, want)


def test_attention_hides_pages_outside_the_cache_and_clamps_lengths(torch, okq):
    """Table entries of -1, n_pages and far off; a length over max_length and
    over the table; a negative one; every page hidden."""
    lengths, page = [100, 100, 100, 40, 64], 16
    cache, table, q = _attn_inputs(torch, okq, BF16, 64, 2, 2, page, lengths)
    table[0, 1], table[0, 3], table[1, 0], table[1, 5] = -1, cache.n_pages, 2 ** 31 - 1, -2 ** 31
    table[3, :] = -1
    said = [100, 100, 2 ** 31 - 1, 40, -5]
    for longest in (100, 50, 10 ** 6, 0):
        got = _attention(torch, okq, cache, table, q, said, longest, 0.125)
        torch.cuda.synchronize()
        lens = [100, 100, longest, 40, 0]
        _attn_check_limited = _attn_want(torch, cache, table, q, [min(n, 112) for n in lens], 0.125, 0.0, 0, 2, longest)
        if longest >= 112:  # the third sequence's tokens past its pages are hidden with them
            assert int(table[2, 7]) == -1
            # its last page's rows past 100 are the caller's claim to hold tokens: NaN here
            assert got[0][2].isnan().all()
            got[0][2], got[1][2] = 0, 0
            for w, z in zip(_attn_check_limited, (0, 0, 1, 1)):
                w[2] = z
        _attn_check(torch, got, _attn_check_limited)


def test_attention_of_large_scores_and_infinities(torch, okq):
    """Scores of thousands do not overflow; a visible infinity, among values or
    keys, leaves no finite number in what it reaches and all else alone."""
    lengths = [64, 64]
    cache, table, q = _attn_inputs(torch, okq, BF16, 64, 2, 2, 16, lengths)
    q = q * 300
    want = _attn_want(torch, cache, table, q, lengths, 1.0, 0.0, 0, 2)
    _attn_check(torch, _attention(torch, okq, cache, table, q, lengths, 64, 1.0), want)
    page = int(table[1, 2])
    cache.views[1][page, 1, 5] = torch.full((64,), math.inf, device="cuda").to(torch.bfloat16).view(torch.uint8)
    out, lse = _attention(torch, okq, cache, table, q * 1e-3, lengths, 64, 1.0)
    torch.cuda.synchronize()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :2]).all() and torch.isfinite(lse).all()
    assert not torch.isfinite(out[1, 2:]).any()
    q.fill_(0)
    q[:, :, 0] = 1
    k = cache.views[0]
    for j in range(4):
        row = torch.zeros(16, 64, device="cuda")
        row[:, 0] = -math.inf
        k[int(table[0, j]), 0] = row.to(torch.bfloat16).view(torch.uint8)
    out, lse = _attention(torch, okq, cache, table, q, lengths, 64, 1.0)
    torch.cuda.synchronize()
    assert not torch.isfinite(lse[0, :2]).any()
    assert torch.isfinite(out[0, 2:]).all()


def test_attention_past_4_gib(torch, okq):
    """Pages whose byte offsets pass 32 bits."""
    page, d, row = 16, 64, 128
    stride = 3 << 30
    buf = torch.zeros(2, 2 * stride + page * row, dtype=torch.uint8, device="cuda")
    c = okq.KvPages(type=BF16, n_pages=3, page_tokens=page, kv_heads=1, head_dim=d, page_stride=stride, head_stride=0,
                    token_stride=row, k=buf[0].data_ptr(), v=buf[1].data_ptr())
    small, table, q = _attn_inputs(torch, okq, BF16, d, 1, 4, page, [16 * 1])
    pg = int(table[0, 0])
    for b, v in zip(buf, small.views):
        b[2 * stride:2 * stride + page * row] = v[pg].reshape(-1)
    big = type("C", (), {"ref": lambda self: ctypes.byref(c)})()
    t2 = torch.tensor([[2]], dtype=torch.int32)
    a = _attention(torch, okq, big, t2, q, [16], 16, 0.125)
    b = _attention(torch, okq, small, table[:, :1], q, [16], 16, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_attention_in_a_graph_and_on_another_stream(torch, okq):
    """Captured after one call on the stream; replayed with new queries and
    lengths between eager calls, each replay the eager result bit for bit."""
    lengths = [3000, 10, 0, 700]
    cache, table, q = _attn_inputs(torch, okq, BF16, 128, 2, 4, 16, lengths)
    s = torch.cuda.Stream()
    td, ld = table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(4, 8, device="cuda")
    torch.cuda.synchronize()

    def step(stream):
        okq.call("okq_paged_attention", q.data_ptr(), 8 * 128, 4, 8, cache.ref(), td.data_ptr(), td.shape[1],
                 ld.data_ptr(), 3000, 0.09, 0.0, 0, out.data_ptr(), 8 * 128, lse.data_ptr(), stream)

    with torch.cuda.stream(s):
        step(s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        ld.copy_(torch.tensor([3000 - 700 * i, 10 + i, i, 700], dtype=torch.int32))
        torch.cuda.synchronize()
        out.fill_(math.nan)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        out.fill_(math.nan)
        torch.cuda.synchronize()
        step(None)
        torch.cuda.synchronize()
        # as bits: the second length's growth takes in rows of 0xFF bytes, NaN in both results
        for a, b in zip(got, (out, lse)):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32))
        assert got[0].isfinite().all(-1).all(-1).tolist() == [True, i == 0, True, True]


# ---- logits -------------------------------------------------------------------------

LOGITS = [  # rows, vocab, history, biases, mask, dtype of odd strides
    (1, 128256, 1200, 20, False, 0),
    (3, 1000, 0, 0, False, 0),
    (5, 1001, 33, 7, True, 3),
    (2, 1, 4, 1, True, 0),
    (4, 31, 5, 2, True, 1),
    (4, 32, 5, 0, True, 0),
    (2, 33, 100, 3, True, 2),
    (7, 4096, 500, 64, True, 0),
    (7, 4097, 500, 65, True, 0),
    (3, 8191, 4000, 300, False, 1),
    (2, 50257, 3000, 129, True, 0),
    (70, 20000, 700, 0, True, 4),
    (300, 2048, 64, 10, False, 0),
    (2, 262144, 900, 50, True, 0),
]


def _logits_inputs(torch, rows, vocab, hist, biases, mask, seed, duplicates=False):
    rng = np.random.default_rng(seed)
    d = {"x": (rng.standard_normal((rows, vocab)) * 3).astype(np.float32),
         "hist": (rng.random((rows, max(hist, 1))) ** 3 * vocab).astype(np.int32).clip(max=vocab - 1),
         "hist_len": rng.integers(0, hist + 1, rows).astype(np.int32),
         "rep": (1 + rng.random(rows) * 0.4).astype(np.float32), "freq": (rng.random(rows) * 0.5).astype(np.float32),
         "pres": (rng.random(rows) * 0.5).astype(np.float32)}
    d["hist_len"][0] = hist
    d["start"] = (d["hist_len"] * rng.random(rows)).astype(np.int32)
    b = max(biases, 1)
    d["bias_ids"] = np.stack([rng.permutation(vocab)[:b] if vocab >= b and not duplicates else rng.integers(0, min(vocab, 9), b)
                              for _ in range(rows)]).astype(np.int32)
    d["bias"] = (rng.standard_normal((rows, b)) * 4).astype(np.float32)
    d["bias_len"] = rng.integers(0, biases + 1, rows).astype(np.int32)
    d["bias_len"][-1] = biases
    share = np.array([0.01, 0.5, 0.98])[np.arange(rows) % 3]
    if rows > 2:
        share[rows // 2] = 0.0
    words = (vocab + 31) // 32
    bits = rng.random((rows, words * 32)) < share[:, None]
    d["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.uint32).reshape(rows, words)
    d["allowed"] = bits[:, :vocab]
    return d


def _logits_want(d, biased, masked, dtype):
    """The definition, each operation in `dtype`; and the bound's sizes in f64."""
    x = d["x"].astype(dtype)
    size = 2 * np.abs(x.astype(np.float64))
    for r in range(x.shape[0]):
        h, s = d["hist"][r, :d["hist_len"][r]], d["start"][r]
        h, new = h[(h >= 0) & (h < x.shape[1])], d["hist"][r, s:d["hist_len"][r]]
        new = new[(new >= 0) & (new < x.shape[1])]
        rep, freq, pres = (dtype(d[k][r]) for k in ("rep", "freq", "pres"))
        ids = np.unique(h)
        x[r, ids] = np.where(x[r, ids] > 0, x[r, ids] / rep, x[r, ids] * rep)
        size[r, ids] *= float(rep)
        ids, n = np.unique(new, return_counts=True)
        x[r, ids] = (x[r, ids] - freq * n.astype(dtype)) - pres
        size[r, ids] += float(freq) * n + float(pres)
        if biased:
            total = {}
            for i, b in zip(d["bias_ids"][r, :d["bias_len"][r]].tolist(), d["bias"][r]):
                if 0 <= i < x.shape[1]:
                    total[i] = dtype(total.get(i, dtype(0)) + dtype(b))
                    size[r, i] += abs(float(b))
            for i, b in total.items():
                x[r, i] = x[r, i] + b
        if masked:
            x[r, ~d["allowed"][r]] = -np.inf
    return x, size


def _logits(torch, okq, d, hist, biases, masked, pad=0, stream=None, inplace=False):
    rows, vocab = d["x"].shape
    dev = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in d.items()
           if k not in ("mask", "allowed")}
    dev["mask"] = torch.from_numpy(np.pad(d["mask"], ((0, 0), (0, pad))).view(np.int32)).cuda()
    x = torch.full((rows, vocab + pad), math.nan, device="cuda")
    x[:, :vocab] = dev["x"]
    out = x if inplace else torch.full((rows, vocab + pad), math.nan, device="cuda")
    best = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    p = {k: v.data_ptr() for k, v in dev.items()}
    h, b = hist > 0, biases > 0
    okq.call("okq_logits_process", x.data_ptr(), vocab + pad, rows, vocab, p["hist"] if h else None,
             d["hist"].shape[1] if h else 0, p["hist_len"] if h else None, p["start"] if h else None, p["rep"], p["freq"],
             p["pres"], p["bias_ids"] if b else None, p["bias"] if b else None, d["bias"].shape[1] if b else 0,
             p["bias_len"] if b else None, p["mask"] if masked else None, dev["mask"].shape[1] if masked else 0,
             out.data_ptr(), vocab + pad, best.data_ptr(), _stream(torch) if stream is None else stream)
    torch.cuda.synchronize()
    assert out[:, vocab:].isnan().all()
    return out[:, :vocab].cpu().numpy(), best.cpu().numpy()


def _logits_check(got, best, d, biased, masked):
    want, size = _logits_want(d, biased, masked, np.float64)
    single, _ = _logits_want(d, biased, masked, np.float32)
    fin = np.isfinite(want)
    assert (np.isfinite(got) == fin).all()
    assert (np.abs(got - want)[fin] <= 5 * U * size[fin]).all()
    assert (got == single).all()  # each operation rounded on its own
    expect = np.where((got > -np.inf).any(1), got.argmax(1), -1)
    assert (best == expect).all()


@pytest.mark.parametrize("case", LOGITS, ids=[f"{c[0]}x{c[1]}h{c[2]}b{c[3]}m{int(c[4])}" for c in LOGITS])
def test_logits(torch, okq, case):
    rows, vocab, hist, biases, masked, pad = case
    print(f"[gpu] logits {case}", flush=True)
    d = _logits_inputs(torch, rows, vocab, hist, biases, masked, 3 + vocab)
    got, best = _logits(torch, okq, d, hist, biases, masked, pad, inplace=rows % 2 == 1)
    _logits_check(got, best, d, biases > 0, masked)


def test_logits_of_ids_outside_the_vocabulary_and_of_repeated_biases(torch, okq):
    d = _logits_inputs(torch, 6, 5000, 200, 150, True, 9, duplicates=True)
    d["hist"][:, ::7] = np.array([-1, 5000, 2 ** 31 - 1, -2 ** 31, 123456, 4999])[:, None]
    d["bias_ids"][:, ::5] = np.array([-1, 5000, 2 ** 31 - 1, -2 ** 31, 123456, 4999])[:, None]
    for _ in range(2):
        got, best = _logits(torch, okq, d, 200, 150, True)
        _logits_check(got, best, d, True, True)


def test_logits_ties_infinities_and_nan(torch, okq):
    d = _logits_inputs(torch, 8, 9001, 0, 0, False, 2)
    x = d["x"]
    x[0, 17] = x[0, 8999] = x[0].max() + 1           # a tie across workgroups: the lowest index
    x[1] = -np.inf                                   # nothing left
    x[2] = -np.inf
    x[2, 9000] = np.finfo(np.float32).min            # the lowest finite value is a choice
    x[3, 4], x[3, 5000] = np.inf, np.inf
    x[4] = 0.0
    x[4, :40] = -0.0                                 # zeros of both signs are equal
    x[5, 8000] = np.nan
    x[6], x[6, 123] = -1e30, -5.0
    d["x"] = x
    got, best = _logits(torch, okq, d, 0, 0, False)
    assert (got.view(np.uint32) == x.view(np.uint32)).all()
    assert best[:7].tolist() == [17, -1, 9000, 4, 0, -1, 123]
    assert best[7] == x[7].argmax()


def test_logits_lengths_past_their_strides_and_absent_parts(torch, okq):
    d = _logits_inputs(torch, 3, 3000, 50, 8, False, 4)
    d["hist_len"][:] = [50, 2 ** 31 - 1, -3]
    d["start"][:] = [60, -5, 0]
    d["bias_len"][:] = [2 ** 31 - 1, -1, 8]
    got, best = _logits(torch, okq, d, 50, 8, False)
    d["hist_len"][:], d["start"][:], d["bias_len"][:] = [50, 50, 0], [50, 0, 0], [8, 0, 8]
    _logits_check(got, best, d, True, False)
    # history alone: no penalty is named, so nothing changes
    x, h, n = (torch.from_numpy(d[k]).cuda() for k in ("x", "hist", "hist_len"))
    out = torch.empty_like(x)
    okq.call("okq_logits_process", x.data_ptr(), 3000, 3, 3000, h.data_ptr(), 50, n.data_ptr(), None, None, None, None,
             None, None, 0, None, None, 0, out.data_ptr(), 3000, None, _stream(torch))
    torch.cuda.synchronize()
    assert torch.equal(out, x)


def test_logits_in_a_graph(torch, okq):
    d = _logits_inputs(torch, 5, 40000, 300, 30, True, 6)
    dev = {k: torch.from_numpy(np.ascontiguousarray(v.view(np.int32) if k == "mask" else v)).cuda() for k, v in d.items()}
    out, best = torch.empty(5, 40000, device="cuda"), torch.empty(5, dtype=torch.int32, device="cuda")
    p = {k: v.data_ptr() for k, v in dev.items()}

    def step(stream):
        okq.call("okq_logits_process", p["x"], 40000, 5, 40000, p["hist"], 300, p["hist_len"], p["start"], p["rep"],
                 p["freq"], p["pres"], p["bias_ids"], p["bias"], 30, p["bias_len"], p["mask"], 1250, out.data_ptr(),
                 40000, best.data_ptr(), stream)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(s.cuda_stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        d["x"] = np.roll(d["x"], 13, 1)
        dev["x"].copy_(torch.from_numpy(d["x"]))
        best.fill_(-9)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        _logits_check(out.cpu().numpy(), best.cpu().numpy(), d, True, True)
        step(None)
        torch.cuda.synchronize()
        _logits_check(out.cpu().numpy(), best.cpu().numpy(), d, True, True)


# ---- wider heads, larger groups, pages of one token, longer lists ---------------------

@pytest.mark.parametrize("tn", ["BF16", "F16", "F32", "Q8_0"])
@pytest.mark.parametrize("d", [160, 192, 320])
def test_attention_of_heads_between_the_common_sizes(torch, okq, tn, d):
    print(f"[gpu] attention {tn} head_dim {d}", flush=True)
    lengths = [700, 0, 33]
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, 2, 3, 16, lengths)
    got = _attention(torch, okq, cache, table, q, lengths, 700, d ** -0.5)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, 3))


@pytest.mark.parametrize("tn,kv,group,page", [("BF16", 520, 1, 1), ("F32", 520, 2, 1), ("F16", 130, 17, 2), ("Q8_0", 520, 1, 1)])
def test_attention_of_one_chunk_with_more_pages_than_are_held_at_once(torch, okq, tn, kv, group, page):
    """So many heads that nothing is split: one workgroup walks all pages, some of them hidden."""
    print(f"[gpu] attention pages {tn} {kv} {page}", flush=True)
    lengths = [1200 * page, 509 * page, 511 * page, 0]
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], 32, kv, group, page, lengths)
    table[0, 505:540], table[0, 1021], table[2, 510] = -1, cache.n_pages, -7
    got = _attention(torch, okq, cache, table, q, lengths, 1300 * page, 0.2)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, 0.2, 0.0, 0, group))


@pytest.mark.parametrize("tn,group", [("BF16", 17), ("F16", 40), ("F32", 33), ("Q8_0", 24)])
def test_attention_of_large_groups_split_over_a_long_cache(torch, okq, tn, group):
    print(f"[gpu] attention group {tn} {group}", flush=True)
    lengths = [9000, 5]
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], 64, 1, group, 32, lengths)
    got = [_attention(torch, okq, cache, table, q, lengths, 9000, 0.125, 40.0, 6001) for _ in range(2)]
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    _attn_check(torch, got[0], _attn_want(torch, cache, table, q, lengths, 0.125, 40.0, 6001, group))


@pytest.mark.parametrize("rows,vocab,hist,biases,masked,duplicates", [
    (3, 50001, 9000, 1025, True, False), (2, 6000, 5000, 3000, False, True), (40, 33000, 4500, 2000, True, True),
    (1, 70000, 4097, 1024, False, True), (3, 900, 6000, 1500, True, True)])
def test_logits_of_long_lists(torch, okq, rows, vocab, hist, biases, masked, duplicates):
    """Histories and biases longer than a workgroup reads at once."""
    print(f"[gpu] logits {rows}x{vocab} h{hist} b{biases}", flush=True)
    d = _logits_inputs(torch, rows, vocab, hist, biases, masked, 11 + vocab, duplicates)
    got, best = _logits(torch, okq, d, hist, biases, masked, inplace=rows == 2)
    _logits_check(got, best, d, True, masked)


@pytest.mark.parametrize("tn,d,kv,group,page,lengths,window,softcap", [
    ("BF16", 512, 1, 5, 16, [9001, 0, 40], 0, 0.0), ("F16", 100, 2, 1, 24, [12000], 5000, 30.0),
    ("F32", 33, 1, 3, 7, [7001, 1, 256, 257, 4000], 0, 0.0), ("Q8_0", 288, 2, 4, 32, [3000, 129], 0, 0.0),
    ("BF16", 260, 8, 9, 16, [300, 700], 0, 0.0), ("F32", 1, 1, 1, 64, [50000], 0, 0.0)])
def test_attention_of_odd_heads_over_long_caches(torch, okq, tn, d, kv, group, page, lengths, window, softcap):
    """Rows that are read one value at a time, split; two calls agree bit for bit."""
    print(f"[gpu] attention odd long {tn} {d} {lengths[:3]}", flush=True)
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, kv, group, page, lengths)
    table[0, 3] = -1
    got = [_attention(torch, okq, cache, table, q, lengths, max(lengths), d ** -0.5, softcap, window) for _ in range(2)]
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    _attn_check(torch, got[0], _attn_want(torch, cache, table, q, lengths, d ** -0.5, softcap, window, group))


@pytest.mark.parametrize("tn,d", [("BF16", 64), ("F32", 50)])
def test_attention_captured_after_a_call_of_other_sequences(torch, okq, tn, d):
    """Many short sequences, which nothing splits, then one long one in a graph
    on the same stream."""
    s = torch.cuda.Stream()
    short, st, sq = _attn_inputs(torch, okq, TYPES[tn], d, 2, 2, 16, [9] * 700)
    long, lt, lq = _attn_inputs(torch, okq, TYPES[tn], d, 2, 2, 16, [4000])
    td, ld = lt.cuda(), torch.tensor([4000], dtype=torch.int32, device="cuda")
    out, lse = torch.empty_like(lq), torch.empty(1, 4, device="cuda")
    torch.cuda.synchronize()
    got = _attention(torch, okq, short, st, sq, [9] * 700, 16, 0.125, stream=s.cuda_stream)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, short, st, sq, [9] * 700, 0.125, 0.0, 0, 2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        okq.call("okq_paged_attention", lq.data_ptr(), 4 * d, 1, 4, long.ref(), td.data_ptr(), td.shape[1],
                 ld.data_ptr(), 4000, 0.125, 0.0, 0, out.data_ptr(), 4 * d, lse.data_ptr(),
                 torch.cuda.current_stream().cuda_stream)
    want = _attn_want(torch, long, lt, lq, [4000], 0.125, 0.0, 0, 2)
    for _ in range(3):
        out.fill_(math.nan)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        _attn_check(torch, (out, lse), want)


# ---- weights, queries and scales of very different sizes --------------------------------

def _written_cache(torch, okq, tn, d, kv, page, K, V):
    """A cache whose sequences hold the rows of K and V: lists of f32 [tokens, kv, d]."""
    lengths = [k.shape[0] for k in K]
    cache, table, _ = _attn_inputs(torch, okq, TYPES[tn], d, kv, 1, page, lengths)
    for i, rows in enumerate(zip(K, V)):
        for t in range(0, lengths[i], page):
            p = int(table[i, t // page])
            for view, r in zip(cache.views, rows):
                r = r[t:t + page].transpose(0, 1).contiguous().cuda()
                view[p, :, :r.shape[1]] = _encode(torch, okq, TYPES[tn], r)
    return cache, table, lengths


def _parked(torch, d, kv, n, gap, seed):
    """n tokens of which the first is `gap` nats above all others (a query of
    8 in dim 0 and 1 in dim 1) and has a value of zeros."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.zeros(n, kv, d), torch.randn(n, kv, d, generator=g)
    k[:, :, 1] = torch.rand(n, kv, generator=g) - 0.5
    k[0, :, 0], k[0, :, 1], v[0] = gap / 8, 0.0, 0.0
    return k, v


@pytest.mark.parametrize("gap", [8, 13, 17, 22, 40])
@pytest.mark.parametrize("tn,d", [("F16", 128), ("F16", 256), ("F16", 80), ("Q8_0", 128), ("Q8_0", 256), ("Q8_0", 64),
                                  ("BF16", 128), ("F32", 128), ("F16", 100)])
def test_attention_keeps_the_weights_below_a_token_whose_value_is_zero(torch, okq, tn, d, gap):
    """The output is what the small weights make it, and each of them is off by
    2e + 8u of itself, however far below the largest: tokens of the heavy one's
    tile, of its wave's later tiles and of other chunks."""
    print(f"[gpu] parked {tn} {d} {gap}", flush=True)
    for kv, sizes in ((2, [20, 128, 2000]), (1, [5000]), (4, [400] * 70)):
        kvs = [_parked(torch, d, kv, n, gap, 3 + n + i) for i, n in enumerate(sizes)]
        cache, table, lengths = _written_cache(torch, okq, tn, d, kv, 16, [k for k, _ in kvs], [v for _, v in kvs])
        q = torch.zeros(len(sizes), kv, d, device="cuda")
        q[:, :, 0], q[:, :, 1] = 8.0, 1.0
        got = _attention(torch, okq, cache, table, q, lengths, max(lengths), 1.0)
        torch.cuda.synchronize()
        _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, 1.0, 0.0, 0, 1))


@pytest.mark.parametrize("tn,d", [("F16", 128), ("F16", 256), ("Q8_0", 128), ("Q8_0", 256), ("BF16", 128), ("F32", 128)])
def test_attention_keeps_the_small_elements_of_a_query(torch, okq, tn, d):
    """A query whose first element is 2^26 times the others, which meet large
    keys: scores of about 1 that the large element has no part in."""
    print(f"[gpu] small query elements {tn} {d}", flush=True)
    g = torch.Generator().manual_seed(17)
    K, V = [], []
    for n in (3, 50):
        k = torch.randn(n, 2, d, generator=g) * 2.0 ** 13
        k[:, :, 0:32] = 0.0
        K.append(k.clamp(-60000, 60000))
        V.append(torch.randn(n, 2, d, generator=g))
    cache, table, lengths = _written_cache(torch, okq, tn, d, 2, 16, K, V)
    q = torch.randn(2, 2, d, generator=g).cuda() * 2.0 ** -16
    q[:, :, 0] = 2.0 ** 10
    got = _attention(torch, okq, cache, table, q, lengths, 50, 1.0)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, 1.0, 0.0, 0, 1))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_of_q8_0_blocks_of_very_different_scales(torch, okq, d):
    """Each block's values keep their precision beside a block of 2^10 or 2^20
    times its scale, and beside a token of a tiny weight and a huge scale."""
    print(f"[gpu] q8_0 scales {d}", flush=True)
    g = torch.Generator().manual_seed(d)
    K, V = [], []
    for n in (30, 300, 3000):
        k, v = 0.3 * torch.randn(n, 2, d, generator=g), torch.randn(n, 2, d, generator=g)
        v[:, :, :32] *= 2.0 ** 10
        v[:, :, 32:64] *= torch.tensor([2.0 ** -10, 1.0])[torch.arange(n) % 2][:, None, None]
        k[n // 3] = 0.0
        k[n // 3, :, 0] = -4.0
        v[n // 3, :, :32] *= 2.0 ** 8  # 32 nats below the rest
        v[n // 3, :, 32:] = 0.0
        K.append(k)
        V.append(v)
    cache, table, lengths = _written_cache(torch, okq, "Q8_0", d, 2, 16, K, V)
    q = torch.randn(3, 4, d, generator=g).cuda() / d ** 0.5
    q[:, :, 0] = 8.0
    got = _attention(torch, okq, cache, table, q, lengths, 3000, 1.0)
    torch.cuda.synchronize()
    _attn_check(torch, got, _attn_want(torch, cache, table, q, lengths, 1.0, 0.0, 0, 2))


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("tn,d", [("BF16", 128), ("F16", 128), ("F16", 256), ("F32", 128), ("Q8_0", 128), ("BF16", 100),
                                  ("F32", 33), ("Q8_0", 320)])
def test_attention_of_an_infinite_key(torch, okq, tn, d, softcap):
    """One infinity of either sign among the keys of one sequence and head: no
    finite number in what reads it, whatever the queries' signs and bits are,
    and the results of all else as without it."""
    print(f"[gpu] infinite key {tn} {d} {softcap}", flush=True)
    lengths, group = [40, 600], 3
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, 2, group, 16, lengths)
    q[:, 0::3] = q[:, 0::3].to(torch.bfloat16).float()  # queries of few bits beside those of many
    q[:, 1::3, :] = q[:, 1::3, :].abs()
    plain = _attention(torch, okq, cache, table, q, lengths, 600, d ** -0.5, softcap)
    torch.cuda.synchronize()
    if tn == "Q8_0":
        bad = torch.tensor([0x00, 0xFC], dtype=torch.uint8, device="cuda")  # a block's scale: -inf
        at = slice(0, 2)
    else:
        bad = torch.tensor([-math.inf], device="cuda").to(_dtype(torch, TYPES[tn])).view(torch.uint8)
        at = slice(0, len(bad))
    key = cache.views[0][int(table[1, 20]), 1, 7]
    was = key[at].clone()
    for sign in (0x80, 0x00):
        bad[-1] = (int(bad[-1]) & 0x7F) | sign
        key[at] = bad
        out, lse = _attention(torch, okq, cache, table, q, lengths, 600, d ** -0.5, softcap)
        torch.cuda.synchronize()
        assert out[1, group:].isnan().all() and lse[1, group:].isnan().all()
        for a, b in zip((out, lse), plain):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1, :group], b[1, :group])
    key[at] = was


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_of_an_infinite_q8_0_scale_among_the_values(torch, okq, d):
    """It reaches its block's 32 columns in its head, and nothing else: not the
    columns of another block of its token, whose scale is far above all others."""
    print(f"[gpu] infinite scale {d}", flush=True)
    lengths = [33, 500]
    cache, table, q = _attn_inputs(torch, okq, Q8_0, d, 2, 2, 16, lengths)
    row = cache.views[1][int(table[1, 12]), 1, 3]
    if d > 96:
        row[102:104] = torch.tensor([0x00, 0x70], dtype=torch.uint8, device="cuda")  # 2^13
    want = _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, 2)
    row[34:36] = torch.tensor([0x00, 0x7C], dtype=torch.uint8, device="cuda")
    out, lse = _attention(torch, okq, cache, table, q, lengths, 500, d ** -0.5)
    torch.cuda.synchronize()
    assert not torch.isfinite(out[1, 2:, 32:64]).any()
    out[1, 2:, 32:64] = 0.0
    for w in (want[0], want[2]):
        w[1, 2:, 32:64] = 0.0
    _attn_check(torch, (out, lse), want)


@pytest.mark.parametrize("tn,d", [("BF16", 128), ("F16", 128), ("F16", 256), ("F32", 80), ("F16", 100), ("F32", 260)])
def test_attention_of_an_infinite_value(torch, okq, tn, d):
    """It reaches its column in its head, and nothing else, also where the
    token's weight is next to nothing."""
    print(f"[gpu] infinite value {tn} {d}", flush=True)
    t = TYPES[tn]
    lengths = [33, 500]
    cache, table, q = _attn_inputs(torch, okq, t, d, 2, 2, 16, lengths)
    for far in (False, True):
        view = cache.views[0][int(table[1, 12]), 1, 3]
        if far:  # the query points away from the key
            view[:] = (q[1, 2:].sum(0) * -5).to(_dtype(torch, t)).view(torch.uint8)
        want = _attn_want(torch, cache, table, q, lengths, d ** -0.5, 0.0, 0, 2)
        row = cache.views[1][int(table[1, 12]), 1, 3].view(_dtype(torch, t))
        was = row[5].item()
        row[5] = math.inf
        out, lse = _attention(torch, okq, cache, table, q, lengths, 500, d ** -0.5)
        torch.cuda.synchronize()
        row[5] = was
        assert not torch.isfinite(out[1, 2:, 5]).any()
        out[1, 2:, 5] = 0.0
        for w in (want[0], want[2]):
            w[1, 2:, 5] = 0.0
        _attn_check(torch, (out, lse), want)


@pytest.mark.parametrize("tn,d", [("BF16", 128), ("F16", 128), ("F16", 256), ("F32", 128), ("Q8_0", 128), ("BF16", 100)])
def test_attention_of_an_infinite_query(torch, okq, tn, d):
    """NaN in its head of its sequence, and all else as without it."""
    print(f"[gpu] infinite query {tn} {d}", flush=True)
    lengths = [40, 600]
    cache, table, q = _attn_inputs(torch, okq, TYPES[tn], d, 2, 3, 16, lengths)
    plain = _attention(torch, okq, cache, table, q, lengths, 600, d ** -0.5)
    torch.cuda.synchronize()
    for bad in (math.inf, -math.inf, math.nan):
        q[1, 4, 9] = bad
        out, lse = _attention(torch, okq, cache, table, q, lengths, 600, d ** -0.5)
        torch.cuda.synchronize()
        assert out[1, 4].isnan().all() and lse[1, 4].isnan()
        out[1, 4], lse[1, 4] = plain[0][1, 4], plain[1][1, 4]
        assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
