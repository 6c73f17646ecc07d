"""What okq_qk_norm_rope, okq_paged_attention and okq_logits_process refuse
(CPU only: everything here is decided before a device is looked for)."""
import ctypes

import pytest

from ocelotl_amd import okq

P = 1 << 12  # an aligned address that is never read
F32, F16, BF16, Q8_0, Q4_K = 0, 1, 30, 8, 12


def pages(**kw):
    d = dict(type=BF16, n_pages=4, page_tokens=16, kv_heads=2, head_dim=64, page_stride=2 * 16 * 128,
             head_stride=16 * 128, token_stride=128, k=P, v=P)
    d.update(kw)
    return okq.KvPages(**d)


def rope(**kw):
    d = dict(q=P, qs=512, k=P, ks=128, v=P, vs=128, tokens=3, hq=8, hkv=2, d=64, qn=None, kn=None, eps=1e-6, pos=P,
             freq=P, rotary=64, inter=0, qo=P, qos=512, ko=None, kos=0, cache=pages(), slots=P, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    if d["cache"] is not None:
        d["cache"] = ctypes.byref(d["cache"])
    return okq.lib().okq_qk_norm_rope(*d.values())


def attention(**kw):
    d = dict(q=P, qs=512, seqs=3, hq=8, cache=pages(), table=P, width=4, lengths=P, longest=64, scale=0.125, cap=0.0,
             window=0, out=P, outs=512, lse=None, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    if d["cache"] is not None:
        d["cache"] = ctypes.byref(d["cache"])
    return okq.lib().okq_paged_attention(*d.values())


def logits(**kw):
    d = dict(x=P, xs=1000, rows=2, vocab=1000, hist=P, hs=8, hlen=P, hstart=P, rep=P, freq=P, pres=P, bids=P, bias=P,
             bs=4, blen=P, mask=P, ms=32, out=P, os=1000, best=P, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    return okq.lib().okq_logits_process(*d.values())


CACHE_FAULTS = [
    (dict(type=Q4_K), okq.E_TYPE, "supported: F32, F16, BF16, Q8_0"),
    (dict(type=99), okq.E_TYPE, "(99)"),
    (dict(n_pages=0), okq.E_SHAPE, "at least 1"),
    (dict(page_tokens=0), okq.E_SHAPE, "at least 1"),
    (dict(n_pages=1 << 31), okq.E_SHAPE, "at least 1"),
    (dict(type=Q8_0, head_dim=48), okq.E_SHAPE, "multiple of 32"),
    (dict(token_stride=126), okq.E_SHAPE, "smaller than a row"),
    (dict(head_stride=64), okq.E_SHAPE, "smaller than a row"),
    (dict(page_stride=-128), okq.E_SHAPE, "smaller than a row"),
    (dict(token_stride=129), okq.E_ALIGN, "multiple of 2"),
    (dict(type=F32, token_stride=258, head_stride=1 << 13, page_stride=1 << 14), okq.E_ALIGN, "multiple of 4"),
    (dict(page_stride=(1 << 62) // 2 * 2), okq.E_SHAPE, "overflows"),
    (dict(k=None), okq.E_ARG, "null pointer"),
    (dict(v=None), okq.E_ARG, "null pointer"),
    (dict(k=P + 1), okq.E_ALIGN, "2-byte aligned"),
]


@pytest.mark.parametrize("call", [rope, attention], ids=["rope", "attention"])
@pytest.mark.parametrize("fault,status,text", CACHE_FAULTS, ids=[str(f[0]) for f in CACHE_FAULTS])
def test_a_bad_cache_is_refused(okqlib, call, fault, status, text):
    assert call(cache=pages(**fault)) == status
    assert text in okq.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(tokens=-1), okq.E_SHAPE, "tokens=-1"),
    (dict(hq=0), okq.E_SHAPE, "at least 1"),
    (dict(d=513), okq.E_SHAPE, "head_dim 1 to 512"),
    (dict(rotary=63), okq.E_SHAPE, "rotary=63"),
    (dict(rotary=66), okq.E_SHAPE, "rotary=66"),
    (dict(hkv=4, ks=256, vs=256), okq.E_SHAPE, "does not match"),
    (dict(eps=float("nan")), okq.E_ARG, "epsilon"),
    (dict(eps=-1.0), okq.E_ARG, "epsilon"),
    (dict(qs=511), okq.E_SHAPE, "q stride=511"),
    (dict(ks=1 << 61), okq.E_SHAPE, "overflows"),
    (dict(tokens=1 << 28, cache=None, ko=P, kos=128), okq.E_SHAPE, "launch limits"),
    (dict(q=None), okq.E_ARG, "q is null"),
    (dict(v=None), okq.E_ARG, "v is null"),
    (dict(qo=None), okq.E_ARG, "q_out is null"),
    (dict(pos=None), okq.E_ARG, "positions is null"),
    (dict(freq=None), okq.E_ARG, "inv_freq is null"),
    (dict(slots=None), okq.E_ARG, "slots is null"),
    (dict(cache=None), okq.E_ARG, "needs a cache or k_out"),
    (dict(k=P + 2), okq.E_ALIGN, "k must be 4-byte"),
    (dict(qn=P + 2), okq.E_ALIGN, "norm weights"),
    (dict(slots=P + 4), okq.E_ALIGN, "8-byte"),
])
def test_rope_refusals(okqlib, kw, status, text):
    assert rope(**kw) == status
    assert text in okq.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(cache=None), okq.E_ARG, "cache is null"),
    (dict(seqs=-1), okq.E_SHAPE, "seqs=-1"),
    (dict(hq=7), okq.E_SHAPE, "multiple of kv_heads"),
    (dict(hq=0), okq.E_SHAPE, "multiple of kv_heads"),
    (dict(seqs=1 << 29), okq.E_SHAPE, "launch limits"),
    (dict(width=-1), okq.E_SHAPE, "table_width=-1"),
    (dict(longest=-1), okq.E_SHAPE, "max_length=-1"),
    (dict(longest=1 << 31), okq.E_SHAPE, "max_length"),
    (dict(window=-1), okq.E_SHAPE, "window=-1"),
    (dict(scale=float("inf")), okq.E_ARG, "scale"),
    (dict(cap=-1.0), okq.E_ARG, "softcap"),
    (dict(cap=float("nan")), okq.E_ARG, "softcap"),
    (dict(qs=100), okq.E_SHAPE, "q stride=100"),
    (dict(outs=100), okq.E_SHAPE, "out stride=100"),
    (dict(q=None), okq.E_ARG, "q is null"),
    (dict(out=None), okq.E_ARG, "out is null"),
    (dict(lengths=None), okq.E_ARG, "lengths is null"),
    (dict(table=None), okq.E_ARG, "block_table is null"),
    (dict(lse=P + 2), okq.E_ALIGN, "lse"),
])
def test_attention_refusals(okqlib, kw, status, text):
    assert attention(**kw) == status
    assert text in okq.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(rows=-1), okq.E_SHAPE, "rows=-1"),
    (dict(vocab=0), okq.E_SHAPE, "vocab=0"),
    (dict(vocab=(1 << 31) - 1), okq.E_SHAPE, "vocab"),
    (dict(rows=1 << 31), okq.E_SHAPE, "launch limits"),
    (dict(hs=-1), okq.E_SHAPE, "history_stride=-1"),
    (dict(bs=-1), okq.E_SHAPE, "bias_stride=-1"),
    (dict(xs=999), okq.E_SHAPE, "logits stride=999"),
    (dict(os=999), okq.E_SHAPE, "out stride=999"),
    (dict(ms=31), okq.E_SHAPE, "mask stride=31"),
    (dict(x=None), okq.E_ARG, "logits is null"),
    (dict(out=None), okq.E_ARG, "out is null"),
    (dict(hlen=None), okq.E_ARG, "history_len is null"),
    (dict(bias=None), okq.E_ARG, "bias is null"),
    (dict(blen=None), okq.E_ARG, "bias_len is null"),
    (dict(mask=P + 2), okq.E_ALIGN, "mask"),
    (dict(best=P + 2), okq.E_ALIGN, "best"),
])
def test_logits_refusals(okqlib, kw, status, text):
    assert logits(**kw) == status
    assert text in okq.last_error()


def test_nothing_to_do_is_a_no_op(okqlib):
    assert rope(tokens=0, q=None, k=None, v=None, qo=None, pos=None, freq=None, slots=None) == okq.OK
    assert attention(seqs=0, q=None, out=None, table=None, lengths=None) == okq.OK
    assert logits(rows=0, x=None, out=None) == okq.OK


def test_valid_calls_without_a_device_are_refused_as_such(okqlib):
    n = ctypes.c_int()
    assert okqlib.okq_device_count(ctypes.byref(n)) == okq.OK
    if n.value > 0:
        pytest.skip("a GPU is present")
    assert rope() == okq.E_NODEV
    assert rope(cache=None, v=None, slots=None, ko=P, kos=128) == okq.E_NODEV
    assert rope(rotary=0, pos=None, freq=None) == okq.E_NODEV
    assert attention() == okq.E_NODEV
    assert attention(width=0, table=None) == okq.E_NODEV
    assert logits() == okq.E_NODEV
    assert logits(hist=None, hs=0, hlen=None, hstart=None, rep=None, freq=None, pres=None, bids=None, bias=None,
                  blen=None, mask=None, ms=0, best=None) == okq.E_NODEV


@pytest.mark.parametrize("call,kw,text", [
    (attention, dict(longest=(1 << 30) + 1), "max_length"),
    (logits, dict(hs=1 << 30), "history_stride"),
    (logits, dict(bs=1 << 30), "bias_stride"),
])
def test_sizes_past_what_the_kernels_index(okqlib, call, kw, text):
    assert call(**kw) == okq.E_SHAPE
    assert text in okq.last_error()


@pytest.mark.parametrize("vocab,rows", [(1, 1 << 22), (1000, 1 << 22), (2047, 1 << 22), (2048, 1 << 21), (4096, 1398102)])
def test_logits_rows_up_to_what_a_launch_counts(okqlib, vocab, rows):
    """2^32 threads are one too many for a launch's count: refused; a row less is not."""
    kw = dict(vocab=vocab, xs=vocab, os=vocab, hist=None, bids=None, mask=None)
    assert logits(rows=rows, **kw) == okq.E_SHAPE
    assert "launch limits" in okq.last_error()
    n = ctypes.c_int()
    assert okqlib.okq_device_count(ctypes.byref(n)) == okq.OK
    if n.value == 0:  # a valid call gets as far as looking for a device
        assert logits(rows=rows - 1, **kw) == okq.E_NODEV


def test_a_loose_max_length_is_bounded_by_the_table(okqlib):
    """A max_length of the type's range is as good as the table's own: what a
    launch counts is tokens that the table can name."""
    kw = dict(seqs=64, longest=1 << 30)
    assert attention(width=1 << 26, **kw) == okq.E_SHAPE
    assert "launch limits" in okq.last_error()
    n = ctypes.c_int()
    assert okqlib.okq_device_count(ctypes.byref(n)) == okq.OK
    if n.value == 0:  # a valid call gets as far as looking for a device
        assert attention(width=4, **kw) == okq.E_NODEV
        assert attention(width=0, table=None, **kw) == okq.E_NODEV
