"""Refusals of the head norms, the mixture-of-experts layer and the logit rules,
on the host before the context is touched (no GPU)."""
import pytest

import cw
from test_paged_args import CTX, NULL, P, batch, pages, refused, spec


def rows_call(s=None, ctx=CTX, x=4096, xs=384, qg=64, kg=64, eps=1e-6, pos=P, rows=3, heads=4, kvh=2,
              hd=64, y=1 << 20, ys=384):
    return cw.lib().cw_qk_norm_rope_rows(ctx, s or spec(), x, xs, qg, kg, eps, pos, rows, heads, kvh,
                                         hd, y, ys)


def kv_call(s=None, ctx=CTX, kv=None, qkv=4096, stride=512, qg=64, kg=64, eps=1e-6, pos=P, slots=P,
            rows=3, heads=4, q=1 << 20, qs=256):
    return cw.lib().cw_qk_norm_rope_kv_rows(ctx, s or spec(), kv or pages(), qkv, stride, qg, kg, eps,
                                            pos, slots, rows, heads, q, qs)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=NULL), "null"), (dict(x=None), "null"), (dict(pos=None), "null"), (dict(y=None), "null"),
    (dict(rows=0), "rows=0"), (dict(rows=(1 << 23) + 1), "2^23"), (dict(heads=-1), "n_heads=-1"),
    (dict(heads=4097, xs=1 << 20, ys=1 << 20), "n_heads=4097"), (dict(kvh=-1), "n_kv_heads=-1"),
    (dict(heads=0, kvh=0), "n_heads=0"), (dict(hd=258, xs=2000, ys=2000), "head_dim=258"),
    (dict(qg=None), "null gain"), (dict(kg=None), "null gain"), (dict(eps=-1e-6), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(xs=383), "strides"),
    (dict(ys=383), "strides"), (dict(y=4096 + 4 * 384), "overlap"), (dict(y=4096, ys=388), "overlap"),
    (dict(s=spec(rot_dim=66)), "at most head_dim"), (dict(s=spec(layout=2)), "layout=2"),
])
def test_qk_norm_rope_rows(kw, text):
    refused(rows_call(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=NULL), "null"), (dict(qkv=None), "null"), (dict(slots=None), "null"),
    (dict(pos=None), "null"), (dict(rows=0), "rows=0"), (dict(heads=-1), "n_heads=-1"),
    (dict(heads=0), "q_out"), (dict(q=None), "q_out"), (dict(stride=511), "stride 511"),
    (dict(qs=255), "q_stride 255"), (dict(q=4096 + 64, qs=512), "overlap"),
    (dict(q=4096, qs=256), "overlap"), (dict(qg=None), "null gain"), (dict(kg=None), "null gain"),
    (dict(eps=-1.0), "eps"), (dict(kv=pages(k=None)), "null cache"), (dict(kv=pages(v=8200)), "aligned"),
    (dict(kv=pages(head_dim=96)), "head_dim=96"), (dict(kv=pages(kv_dtype=3)), "kv_dtype=3"),
    (dict(s=spec(theta=0.5)), "theta"),
])
def test_qk_norm_rope_kv_rows(kw, text):
    refused(kv_call(**kw), text)


def moe_call(ctx=CTX, x=1 << 20, rows=3, pos=None, res=None, y=1 << 24, ids=None, p=None, **kw):
    d = dict(dim=64, hidden=96, n_experts=8, top_k=2, normalise=1, router=4096, gate_scales=4096,
             up_scales=4096, down_scales=4096, gate_quants=4096, up_quants=4096, down_quants=4096)
    return cw.lib().cw_moe_rows(ctx, cw.Moe(**{**d, **kw}), x, rows, pos, res, y, ids, p)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=NULL), "null"), (dict(x=None), "null"), (dict(y=None), "null"),
    *[(dict([(k, None)]), "null weights") for k in ("router", "gate_scales", "up_scales", "down_scales",
                                                    "gate_quants", "up_quants", "down_quants")],
    (dict(rows=0), "rows=0"), (dict(rows=65537), "rows=65537"), (dict(dim=0), "dim=0"),
    (dict(dim=48), "dim=48"), (dict(dim=32800), "dim=32800"), (dict(hidden=-32), "hidden=-32"),
    (dict(hidden=33), "hidden=33"), (dict(n_experts=0), "n_experts=0"),
    (dict(n_experts=513), "n_experts=513"), (dict(top_k=0), "top_k=0"), (dict(top_k=9), "top_k=9"),
    (dict(n_experts=64, top_k=33), "top_k=33"), (dict(normalise=2), "normalise=2"),
    (dict(x=(1 << 20) + 4), "aligned"), (dict(router=4100), "aligned"), (dict(up_quants=4104), "aligned"),
    (dict(y=1 << 20), "overlap"), (dict(y=(1 << 20) + 767), "overlap"), (dict(y=(1 << 20) - 764), "overlap"),
    (dict(res=(1 << 24) + 4), "residual and y"), (dict(res=(1 << 24) - 764), "residual and y"),
])
def test_moe_rows(kw, text):
    refused(moe_call(**kw), text)


def test_moe_rows_without_a_layer():
    refused(cw.lib().cw_moe_rows(CTX, None, P, 1, None, None, 1 << 20, None, None), "null")


def logits_call(rules=None, b=None, ctx=CTX, x=1 << 20, stride=100, rows=3, vocab=100, out=1 << 24,
                os=100, token=None, logprob=None):
    return cw.lib().cw_logits_rows(ctx, cw.LogitRules(**(rules or {})), b or batch(), None, x, stride,
                                   rows, vocab, out, os, token, logprob)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=NULL), "null"), (dict(x=None), "null"), (dict(out=None), "no output"),
    (dict(rows=0), "rows=0"), (dict(rows=65536), "rows=65536"), (dict(vocab=0), "vocab=0"),
    (dict(vocab=(1 << 24) + 1, stride=1 << 25, os=1 << 25), "2^24"), (dict(stride=99), "stride 99"),
    (dict(os=99), "out_stride 99"), (dict(out=(1 << 20) + 400), "overlap"),
    (dict(out=1 << 20, os=104), "overlap"), (dict(b=batch(first_row=None)), "first_row"),
    (dict(b=batch(n_seq=0)), "n_seq=0"), (dict(b=batch(rows=0)), "rows=0"),
    (dict(b=batch(mask=4096)), "mask_words=0"), (dict(rules=dict(tokens=4096)), "length"),
    (dict(rules=dict(tokens=4096, length=4096)), "max_len=0"),
    (dict(rules=dict(bias=4096, n_bias=3)), "bias_first"),
    (dict(rules=dict(bias=4096, bias_first=4096, bias_token=4096)), "n_bias=0"),
    (dict(rules=dict(allowed=4096, allowed_words=4)), "n_allowed=0"),
    (dict(rules=dict(allowed=4096, allowed_words=3, n_allowed=2)), "allowed_words=3"),
])
def test_logits_rows(kw, text):
    refused(logits_call(**kw), text)


def test_logits_rows_without_rules_or_batch():
    lib, r, b = cw.lib(), cw.LogitRules(), batch()
    refused(lib.cw_logits_rows(CTX, None, b, None, P, 100, 3, 100, 1 << 24, 100, None, None), "null")
    refused(lib.cw_logits_rows(CTX, r, None, None, P, 100, 3, 100, 1 << 24, 100, None, None), "null")
