"""The paged-cache entry points without a GPU: the C ABI's struct layout and what the library refuses by itself."""
import ctypes as C

import pytest
import torch

from lowlat_gemm import _native as N, tp as TP


def paged(cls, **kw):
    """Arguments of a call that is right but for what a test changes; no pointer is followed before the checks."""
    a = cls()
    c = a.kv
    c.k, c.v = 4096, 8192
    c.k_stride = c.v_stride = (C.c_int64 * 3)(2 * 16 * 128, 16 * 128, 128)
    c.page_table, c.table_stride, c.kv_lens = 4096, 8, 4096
    c.dtype, c.pages, c.kv_heads, c.page_size, c.head_dim, c.table_width, c.batch, c.tokens = 1, 64, 2, 16, 128, 8, 3, 3
    for name, value in kw.items():
        setattr(c, name, value)
    return a


def refused(fn, a, text):
    assert fn(C.byref(a), None) == -1
    msg = N.lib.llg_last_error().decode()
    assert msg.startswith("lowlat_gemm: ") and text in msg, msg


def append(**kw):
    a = paged(N.KvAppendArgs, **kw)
    a.k_in, a.v_in, a.in_dtype = 4096, 4096, 1
    a.k_in_stride = a.v_in_stride = (C.c_int64 * 2)(256, 128)
    return a


def attention(**kw):
    a = paged(N.AttnArgs, **kw)
    a.q, a.out, a.q_dtype, a.heads, a.scale, a.causal = 4096, 4096, 1, 16, 0.1, 1
    a.q_stride = a.out_stride = (C.c_int64 * 2)(2048, 128)
    return a


def test_struct_layout_matches_library():
    sizes = (C.c_int32 * 4)()
    N.lib.llg_attn_struct_sizes(C.byref(sizes))
    assert tuple(sizes) == (C.sizeof(N.PagedKV), C.sizeof(N.KvAppendArgs), C.sizeof(N.KvReadArgs), C.sizeof(N.AttnArgs))


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "must be bf16, f16 or e4m3"), (dict(head_dim=24), "multiple of 16"), (dict(head_dim=272), "multiple of 16"),
    (dict(page_size=0), "out of range"), (dict(kv_heads=0), "out of range"), (dict(batch=-1), "out of range"),
    (dict(tokens=4), "multiple of the 3 sequences"), (dict(table_width=1 << 28), "more than"), (dict(dtype=4), "needs k_scale and v_scale"),
    (dict(k_scale=4096, v_scale=4096), "takes none"), (dict(k=4100), "16-byte aligned"), (dict(kv_lens=None), "device pointers")])
def test_cache_refusals(change, text):
    refused(N.lib.llg_kv_append, append(**change), text)
    refused(N.lib.llg_paged_attention, attention(**change), text)
    if "tokens" not in change:
        r = paged(N.KvReadArgs, **change)
        r.k_out, r.v_out, r.max_len, r.out_dtype = 4096, 4096, 5, 1
        refused(N.lib.llg_kv_read, r, text)


def test_cache_rows_must_be_aligned():
    a = append()
    a.kv.k_stride = (C.c_int64 * 3)(4096, 2048, 132)
    refused(N.lib.llg_kv_append, a, "16-byte aligned")
    a = append()
    a.k_in_stride = (C.c_int64 * 2)(260, 132)
    refused(N.lib.llg_kv_append, a, "rows of k and v must be 16-byte aligned")


def test_append_and_read_refusals():
    a = append()
    a.in_dtype = 4
    refused(N.lib.llg_kv_append, a, "bf16, f16 or f32")
    a.in_dtype = 2
    refused(N.lib.llg_kv_append, a, "of its own type")
    r = paged(N.KvReadArgs)
    r.k_out, r.v_out, r.max_len, r.out_dtype = 4096, 4096, 5, 2
    refused(N.lib.llg_kv_read, r, "16-bit cache's type")
    r.out_dtype, r.max_len = 1, -1
    refused(N.lib.llg_kv_read, r, "max_len")
    r.max_len, r.k_out = 5, 4100
    refused(N.lib.llg_kv_read, r, "outputs must be 16-byte aligned")


def test_attention_refusals():
    refused(N.lib.llg_paged_attention, attention(head_dim=96), "head_dim must be 64 or 128")
    a = attention()
    a.q_dtype = 3
    refused(N.lib.llg_paged_attention, a, "q must be bf16 or f16")
    a.q_dtype = 2
    refused(N.lib.llg_paged_attention, a, "must have q's type")
    for heads in (0, 3, 66):
        a = attention()
        a.heads = heads
        refused(N.lib.llg_paged_attention, a, "1 to 32 times")
    a = attention()
    a.window = -1
    refused(N.lib.llg_paged_attention, a, "window")
    a = attention()
    a.q_stride = (C.c_int64 * 2)(2048, 132)
    refused(N.lib.llg_paged_attention, a, "rows of q and out")
    a = attention()
    refused(N.lib.llg_paged_attention, a, "bytes of 16-byte aligned workspace")  # none given
    # more key tiles than the kernels count in 32 bits
    a = attention(batch=1 << 16, tokens=1 << 16, table_width=1 << 20, kv_heads=16)
    a.heads = 16
    assert N.lib.llg_paged_attention_ws(C.byref(a)) == -1 and b"too many key tiles" in N.lib.llg_last_error()


def test_empty_calls_do_nothing():
    for a, fn in ((append(batch=0, tokens=0), N.lib.llg_kv_append), (attention(batch=0, tokens=0), N.lib.llg_paged_attention),
                  (append(pages=0), N.lib.llg_kv_append)):
        assert fn(C.byref(a), None) == 0


def test_null_arguments():
    for fn in (N.lib.llg_kv_append, N.lib.llg_kv_read, N.lib.llg_paged_attention):
        assert fn(None, None) == -1 and b"null arguments" in N.lib.llg_last_error()


def test_decode_cache_arguments():
    c = TP.DecodeCache(2, 3, 100, 2, "cpu", head_dim=64, page_size=16)
    assert c.page_table.shape == (3, 7) and c.page_table.flatten().tolist() == list(range(21)) and c.kv_lens.tolist() == [0, 0, 0]
    (k, v, table, lens), scales = c.layers[1]
    assert k.shape == v.shape == (21, 2, 16, 64) and k.dtype == torch.float8_e4m3fn and scales["k_scale"].shape == (21, 2, 16)
    assert TP.DecodeCache(1, 1, 1, 1, "cpu", dtype=torch.bfloat16).layers[0][1] == {}
    for bad in (dict(dtype=torch.float32), dict(page_size=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            TP.DecodeCache(**{**dict(layers=1, batch=1, max_len=8, kv_heads=1, device="cpu"), **bad})
    with pytest.raises(ValueError, match="own entry points"):
        TP.DecodeStep("bf16", 1, 1, 0, torch.device("cpu"), TP.LayerShape(hidden=256, qkv=512, inter=256), gemm_fn=lambda *a, **k: None,
                      cache=TP.DecodeCache(1, 1, 8, 1, "cpu"))


def test_decode_cache_holds_whole_pages():
    """max_len is what a sequence's pages hold, not less than was asked for."""
    for asked, page, held in ((100, 16, 112), (64, 64, 64), (1, 64, 64), (65, 64, 128)):
        c = TP.DecodeCache(1, 2, asked, 1, "cpu", page_size=page)
        assert c.max_len == held == c.page_table.shape[1] * c.layers[0][0][0].shape[2]


@pytest.mark.parametrize("hidden,kv_heads,cache,kind,text", [
    (10 * 128, 4, {}, "bf16", "10 query heads"), (66 * 64, 2, dict(head_dim=64), "bf16", "66 query heads"),
    (512, 2, dict(head_dim=32), "bf16", "64 or 128"), (1024, 2, dict(dtype=torch.bfloat16), "f16", "bfloat16"),
    (1024, 2, dict(dtype=torch.float16), "w8a16_bf16", "float16")])
def test_a_step_refuses_caches_that_it_cannot_attend_over(hidden, kv_heads, cache, kind, text):
    """Before any step, so that lengths never run ahead of what is stored."""
    c = TP.DecodeCache(1, 1, 8, kv_heads, "cpu", **cache)
    shape = TP.LayerShape(hidden=hidden, qkv=hidden + 2 * kv_heads * c.head_dim, inter=256)
    with pytest.raises(ValueError, match=text):
        TP.DecodeStep(kind, 1, 1, 0, torch.device("cpu"), shape, cache=c)
