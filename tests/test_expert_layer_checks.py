"""What okq_residual_norm, okq_moe_route and okq_moe_mlp_q refuse (CPU only:
everything here is decided before a device is looked for)."""
import pytest

from ocelotl_amd import okq

P = 1 << 12  # an aligned address that is never read
F32, F16, BF16, Q4_0, Q8_0, Q4_K, Q6_K = 0, 1, 30, 2, 8, 12, 14
NAN, INF = float("nan"), float("inf")


def norm(**kw):
    d = dict(x=P, xs=64, branch=2 * P, bs=64, rows=3, hidden=64, post=P, gate=P, gs=0, bscale=1.0, rscale=1.0, pre=P,
             eps=1e-6, sum=3 * P, ss=64, normed=4 * P, ntype=F32, ns=64, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    return okq.lib().okq_residual_norm(*d.values())


def route(**kw):
    d = dict(x=P, xs=64, rows=3, hidden=64, wtype=F32, w=P, experts=32, bias=P, score=0, choice=P, groups=4, top=2,
             best=2, k=8, renorm=1, scale=1.0, ids=P, weights=P, logits=P, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    return okq.lib().okq_moe_route(*d.values())


GU, DOWN = 6 * 512 * 144, 6 * 256 * 2 * 210


def moe(**kw):
    d = dict(x=P, xs=256, rows=3, hidden=256, inner=512, experts=6, k=2, ids=P, weights=P, gutype=Q4_K, gate=P, gbytes=GU,
             up=P, ubytes=GU, dtype=Q6_K, down=P, dbytes=DOWN, out=P, outs=256, stream=None)
    assert set(kw) <= set(d)
    d.update(kw)
    return okq.lib().okq_moe_mlp_q(*d.values())


NORM = [
    (dict(rows=-1), okq.E_SHAPE, "rows=-1"),
    (dict(rows=1 << 22), okq.E_SHAPE, "rows below 2^22"),
    (dict(hidden=0), okq.E_SHAPE, "hidden=0"),
    (dict(eps=-1.0), okq.E_ARG, "epsilon"),
    (dict(eps=NAN), okq.E_ARG, "epsilon"),
    (dict(bscale=INF), okq.E_ARG, "scales finite"),
    (dict(rscale=NAN), okq.E_ARG, "scales finite"),
    (dict(pre=None), okq.E_ARG, "come together"),
    (dict(normed=None), okq.E_ARG, "come together"),
    (dict(normed=None, pre=None, sum=None), okq.E_ARG, "sum or normed"),
    (dict(ntype=Q8_0), okq.E_TYPE, "supported: F32, F16, BF16"),
    (dict(x=None), okq.E_ARG, "x is null"),
    (dict(branch=None), okq.E_ARG, "branch is null"),
    (dict(xs=63), okq.E_SHAPE, "x stride=63"),
    (dict(bs=-64), okq.E_SHAPE, "branch stride"),
    (dict(gs=63), okq.E_SHAPE, "gate stride"),
    (dict(ss=1), okq.E_SHAPE, "sum stride"),
    (dict(ns=63), okq.E_SHAPE, "normed stride"),
    (dict(gate=P + 2), okq.E_ALIGN, "gate"),
    (dict(post=P + 1), okq.E_ALIGN, "post_norm"),
    (dict(sum=P, ss=128), okq.E_SHAPE, "in place"),
    (dict(sum=2 * P, ss=128), okq.E_SHAPE, "in place"),
    (dict(xs=1 << 62), okq.E_SHAPE, "overflows"),
]
ROUTE = [
    (dict(wtype=Q8_0), okq.E_TYPE, "supported: F32, F16, BF16"),
    (dict(rows=-1), okq.E_SHAPE, "rows=-1"),
    (dict(rows=(1 << 26) + 1), okq.E_SHAPE, "at most 2^26"),
    (dict(hidden=0), okq.E_SHAPE, "hidden=0"),
    (dict(experts=0), okq.E_SHAPE, "experts=0"),
    (dict(experts=513, groups=1, top=1), okq.E_SHAPE, "1 to 512"),
    (dict(groups=5), okq.E_SHAPE, "groups=5"),
    (dict(groups=0), okq.E_SHAPE, "groups=0"),
    (dict(experts=390, groups=65), okq.E_SHAPE, "groups=65"),
    (dict(top=0), okq.E_SHAPE, "top_groups=0"),
    (dict(top=5), okq.E_SHAPE, "top_groups=5"),
    (dict(k=0), okq.E_SHAPE, "top_k=0"),
    (dict(k=17), okq.E_SHAPE, "top_k=17"),
    (dict(experts=512, groups=1, top=1, k=65), okq.E_SHAPE, "top_k=65"),
    (dict(score=2), okq.E_ARG, "score=2"),
    (dict(best=3), okq.E_ARG, "group_best=3"),
    (dict(best=0), okq.E_ARG, "group_best=0"),
    (dict(scale=INF), okq.E_ARG, "scale"),
    (dict(x=None), okq.E_ARG, "x is null"),
    (dict(w=None), okq.E_ARG, "w is null"),
    (dict(ids=None), okq.E_ARG, "ids is null"),
    (dict(weights=None), okq.E_ARG, "weights is null"),
    (dict(w=P + 2), okq.E_ALIGN, "aligned to its elements"),
    (dict(w=P + 1, wtype=BF16), okq.E_ALIGN, "aligned to its elements"),
    (dict(choice=P + 2), okq.E_ALIGN, "choice_bias"),
    (dict(xs=63), okq.E_SHAPE, "x stride=63"),
]
MOE = [
    (dict(rows=-1), okq.E_SHAPE, "rows=-1"),
    (dict(experts=0), okq.E_SHAPE, "experts=0"),
    (dict(experts=4097), okq.E_SHAPE, "1 to 4096"),
    (dict(k=0), okq.E_SHAPE, "top_k=0"),
    (dict(k=65), okq.E_SHAPE, "top_k=65"),
    (dict(gutype=F32), okq.E_TYPE, "Q8_0, Q4K, Q5K, Q6K"),
    (dict(gutype=Q4_0), okq.E_TYPE, "Q4_0"),
    (dict(dtype=BF16), okq.E_TYPE, "BF16"),
    (dict(hidden=255), okq.E_SHAPE, "block size 256"),
    (dict(inner=500, gbytes=6 * 500 * 144, ubytes=6 * 500 * 144), okq.E_SHAPE, "down rows of 500"),
    (dict(hidden=0), okq.E_SHAPE, "gate rows of 0"),
    (dict(inner=0), okq.E_SHAPE, "0 outputs"),
    (dict(gbytes=GU - 1), okq.E_SHAPE, "gate bytes"),
    (dict(ubytes=GU + 144), okq.E_SHAPE, "up bytes"),
    (dict(dbytes=0), okq.E_SHAPE, "down bytes"),
    (dict(hidden=1 << 20, inner=1 << 20, xs=1 << 20, outs=1 << 20), okq.E_SHAPE, "4 GiB"),
    (dict(inner=1 << 24), okq.E_SHAPE, "above 2^23"),
    (dict(x=None), okq.E_ARG, "x is null"),
    (dict(ids=None), okq.E_ARG, "ids is null"),
    (dict(weights=None), okq.E_ARG, "weights is null"),
    (dict(out=None), okq.E_ARG, "out is null"),
    (dict(gate=None), okq.E_ARG, "gate weight is null"),
    (dict(down=None), okq.E_ARG, "down weight is null"),
    (dict(up=P + 2), okq.E_ALIGN, "up weight"),
    (dict(x=P + 8), okq.E_ALIGN, "16-byte"),
    (dict(xs=258), okq.E_ALIGN, "x_stride=258"),
    (dict(xs=255), okq.E_SHAPE, "x stride=255"),
    (dict(outs=255), okq.E_SHAPE, "out stride=255"),
]


@pytest.mark.parametrize("call,kw,status,text",
                         [(c, *f) for c, fs in ((norm, NORM), (route, ROUTE), (moe, MOE)) for f in fs],
                         ids=lambda v: v.__name__ if callable(v) else None)
def test_refused_before_a_launch(okqlib, call, kw, status, text):
    assert call(**kw) == status
    assert text in okq.last_error()


@pytest.mark.parametrize("call", [norm, route, moe])
def test_no_rows_is_no_work(okqlib, call):
    assert call(rows=0) == okq.OK


@pytest.mark.parametrize("call", [norm, route, moe])
def test_good_arguments_get_as_far_as_the_device(okqlib, call):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses here are not real ones")
    assert call() == okq.E_NODEV
