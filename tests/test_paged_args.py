"""Refusals of the paged cache's entry points, on the host before the context
is touched (no GPU)."""
import ctypes as C

import pytest

import cw

CTX, P = C.c_void_p(64), C.c_void_p(4096)
NULL = None


def refused(rc, text):
    assert rc == cw.CW_ERR_ARG
    assert text in cw.lib().cw_last_error().decode()


def spec(**kw):
    return cw.rope_spec(**{**dict(rot_dim=64, theta=1e4), **kw})


def pages(**kw):
    d = dict(k=4096, v=8192, kv_dtype=cw.CW_F16, n_kv_heads=2, head_dim=64, page=16, n_blocks=8)
    return cw.KvPages(**{**d, **kw})


def batch(**kw):
    d = dict(cached=4096, n_seq=3, rows=9, first_row=4096, tables=4096, max_blocks=4, mask=None,
             mask_words=0)
    return cw.Batch(**{**d, **kw})


def rope(s=None, ctx=CTX, x=4096, xs=256, rows=3, heads=4, hd=64, y=1 << 20, ys=256):
    return cw.lib().cw_rope_rows(ctx, s or spec(), x, xs, P, rows, heads, hd, y, ys)


@pytest.mark.parametrize("kw,text", [
    (dict(rot_dim=63), "even"), (dict(rot_dim=0), "even"), (dict(rot_dim=66), "at most head_dim"),
    (dict(layout=2), "layout=2"), (dict(scaling=4), "scaling=4"), (dict(theta=1.0), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(scaling=1, factor=0.5), "factor"),
    (dict(scaling=1, factor=float("inf")), "factor"), (dict(scaling=2, factor=2.0), "trained=0"),
    (dict(scaling=2, factor=2.0, trained=64, beta_fast=0.5), "beta_fast"),
    (dict(scaling=2, factor=2.0, trained=64, beta_slow=0.0), "beta_slow"),
    (dict(scaling=2, factor=2.0, trained=64, gain=-1.0), "gain"),
    (dict(scaling=3, factor=2.0, trained=64, low_turns=4.0), "low_turns"),
    (dict(scaling=3, factor=2.0, trained=64, low_turns=0.0), "low_turns"),
])
def test_rope_specs(kw, text):
    refused(rope(spec(**kw)), text)
    refused(cw.lib().cw_rope_kv_rows(CTX, spec(**kw), pages(), P, 512, P, P, 3, 4, 1 << 20, 256), text)


def test_rope_rows():
    refused(rope(ctx=NULL), "null")
    refused(rope(x=None), "null")
    refused(rope(rows=0), "rows=0")
    refused(rope(rows=(1 << 23) + 1), "2^23")
    refused(rope(heads=0), "heads=0")
    refused(rope(heads=4097, xs=1 << 20, ys=1 << 20), "heads=4097")
    refused(rope(hd=258, xs=2000, ys=2000), "head_dim=258")
    refused(rope(xs=255), "strides")
    refused(rope(ys=255), "strides")
    # overlaps: shifted by a row, by a part of one, other strides on the same rows
    refused(rope(y=4096 + 4 * 256), "overlap")
    refused(rope(y=4096 + 16), "overlap")
    refused(rope(y=4096, ys=260), "overlap")
    refused(rope(xs=600, ys=600, y=4096 + 4 * 255), "overlap")
    refused(rope(xs=600, ys=600, y=4096 + 4 * 400), "overlap")


def test_kv_pages():
    lib = cw.lib()
    for kw, text in ((dict(k=None), "null cache"), (dict(v=None), "null cache"),
                     (dict(k=4100), "aligned"), (dict(kv_dtype=2), "kv_dtype=2"),
                     (dict(n_kv_heads=0), "n_kv_heads=0"), (dict(head_dim=96), "head_dim=96"),
                     (dict(page=0), "page=0"), (dict(n_blocks=0), "n_blocks=0"),
                     (dict(page=1 << 16, n_blocks=1 << 15), "2^31 - 1")):
        kv = pages(**kw)
        refused(lib.cw_rope_kv_rows(CTX, spec(rot_dim=16), kv, P, 4096, P, P, 3, 4, 1 << 20, 4096), text)
        refused(lib.cw_attention_tree(CTX, kv, batch(), P, 4096, 4, 1 << 20, 4096), text)
        refused(lib.cw_kv_accept(CTX, kv, batch(), P, 4, P, None), text)
    for page in (8, 24):
        refused(lib.cw_attention_tree(CTX, pages(page=page), batch(), P, 256, 4, 1 << 20, 256),
                "power of two")
        refused(lib.cw_kv_accept(CTX, pages(page=page), batch(), P, 4, P, None), "power of two")
        refused(lib.cw_block_tables(CTX, pages(page=page), batch(), *[P] * 9), "power of two")


def test_rope_kv_rows():
    def call(kv=None, stride=512, rows=3, heads=4, q=1 << 20, qs=256, slots=P):
        return cw.lib().cw_rope_kv_rows(CTX, spec(), kv or pages(), P, stride, P, slots, rows, heads,
                                        q, qs)
    refused(call(slots=None), "null")
    refused(call(rows=0), "rows=0")
    refused(call(heads=-1), "n_heads=-1")
    refused(call(heads=0), "q_out")
    refused(call(q=None), "q_out")
    refused(call(stride=511), "stride 511")
    refused(call(qs=255), "q_stride 255")
    refused(call(q=4096 + 64, qs=512), "overlap")
    refused(call(q=4096, qs=256), "overlap")


def test_batches():
    lib = cw.lib()
    for kw, text in ((dict(cached=None), "cached"), (dict(n_seq=0), "n_seq=0"),
                     (dict(n_seq=65536), "n_seq=65536"), (dict(max_blocks=0), "max_blocks=0"),
                     (dict(tables=None, n_seq=9), "9 requests"), (dict(rows=0), "rows=0"),
                     (dict(rows=(1 << 23) + 1), "2^23"), (dict(first_row=None), "first_row"),
                     (dict(mask=4096), "mask_words=0")):
        b = batch(**kw)
        refused(lib.cw_attention_tree(CTX, pages(), b, P, 256, 4, 1 << 20, 256), text)
        if "tables" not in kw:
            refused(lib.cw_block_tables(CTX, pages(), b, *[P] * 9), text)
        if not {"rows", "first_row", "mask"} & set(kw):
            refused(lib.cw_kv_accept(CTX, pages(), b, P, 4, P, None), text)
    refused(lib.cw_block_tables(CTX, pages(), batch(tables=None), *[P] * 9), "tables")
    for i in range(9):
        refused(lib.cw_block_tables(CTX, pages(), batch(), *[None if j == i else P for j in range(9)]),
                "null")


def test_attention_tree():
    def call(kv=None, q=4096, qs=256, heads=4, out=1 << 20, os=256):
        return cw.lib().cw_attention_tree(CTX, kv or pages(), batch(), q, qs, heads, out, os)
    refused(call(q=None), "null")
    refused(call(heads=0), "n_heads=0")
    refused(call(heads=3), "multiple")
    refused(call(qs=252), "strides")
    refused(call(os=252), "strides")
    refused(call(qs=258), "multiples of 4")
    refused(call(q=4100), "aligned")
    refused(call(out=(1 << 20) + 8), "aligned")
    refused(call(out=4096), "overlap")
    refused(call(out=4096 + 1024), "overlap")


def test_attention_tree_rows_of_many_heads():
    """Rows are counted per kv head, 16 to a workgroup of the join."""
    refused(cw.lib().cw_attention_tree(CTX, pages(n_kv_heads=1), batch(rows=1 << 23), P, 1 << 20, 4096,
                                       1 << 50, 1 << 20), "2^27")
    refused(cw.lib().cw_attention_tree(CTX, pages(n_kv_heads=1024), batch(rows=1 << 23), P, 1 << 20, 4096,
                                       1 << 50, 1 << 20), "2^33")


def test_kv_accept():
    lib = cw.lib()
    refused(lib.cw_kv_accept(CTX, pages(), batch(), None, 4, P, None), "null")
    refused(lib.cw_kv_accept(CTX, pages(), batch(), P, 0, P, None), "max_path=0")
    refused(lib.cw_kv_accept(CTX, pages(), batch(), P, 4, P, 4096), "cached_out")
