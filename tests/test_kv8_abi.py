"""The batched-serving entry points on the CPU: arguments that they refuse, before anything is launched."""
import ctypes

import pytest

OK = 1 << 12  # an aligned address that a refused call never reads


@pytest.fixture
def args(fb):
    c = fb.KV8Cache(k=OK, v=OK, k_scale=OK, v_scale=OK, n_pages=10, n_kv_heads=2, page_tokens=16, head_dim=128, format=0)
    b = fb.PagedBatch(n_req=2, n_tokens=4, page_tokens=16, max_pages=5, n_pages=10, n_touch=4, ctx_len=OK, new_len=2 * OK, block_table=OK,
                      free_pages=OK, n_free=OK, n_free_out=3 * OK, ctx_out=4 * OK, kv_len=5 * OK, new_start=OK, slot=OK, pos=OK, touch=OK)
    a = fb.KV8Attn(q=OK, out=OK, lse=None, q_stride=1024, out_stride=1024, type=0, n_q_heads=8, max_new=2, window=0, scale=0.1,
                   workspace=OK, workspace_bytes=1 << 40)
    return c, b, a


def refused(fb, code, text, name, *a):
    a = [ctypes.byref(x) if isinstance(x, ctypes.Structure) else x for x in a]
    assert getattr(fb.lib(), name)(*a) == code, fb.last_error()
    assert text in fb.last_error()


@pytest.mark.parametrize("field,value,code,text", [
    ("n_req", 0, -1, "n_req"), ("n_req", 4097, -4, "at most 4096"), ("n_tokens", -1, -1, "n_tokens"), ("page_tokens", 48, -4, "page_tokens"),
    ("max_pages", 0, -1, "max_pages"), ("n_pages", 0, -1, "n_pages"), ("ctx_len", None, -1, "null"), ("touch", None, -1, "null"),
    ("touch", OK + 4, -2, "16-byte"), ("n_touch", 3, -1, "n_touch"), ("ctx_out", OK, -1, "also an input"),
    ("n_free_out", OK, -1, "also an input"), ("max_pages", 1 << 27, -4, "31 bits")])
def test_plan_refuses(fb, args, field, value, code, text):
    _, b, _ = args
    setattr(b, field, value)
    refused(fb, code, text, "fence_paged_plan", b, None)


def test_null_structs(fb, args):
    c, b, a = args
    for name, x in (("fence_paged_plan", (None, None)), ("fence_kv8_store", (None, b, OK, OK, 0, 256, 256, None)),
                    ("fence_kv8_store", (c, None, OK, OK, 0, 256, 256, None)), ("fence_kv8_load", (None, OK, 1, OK, OK, 0, 256, 256, None)),
                    ("fence_kv8_attention", (None, b, a, None)), ("fence_kv8_attention", (c, None, a, None)),
                    ("fence_kv8_attention", (c, b, None, None))):
        refused(fb, -1, "null", name, *x)
    assert fb.lib().fence_kv8_attention_workspace_bytes(None, None, None) == 0


@pytest.mark.parametrize("field,value,code,text", [
    ("k", None, -1, "null"), ("k", OK + 8, -2, "16-byte"), ("n_pages", 0, -1, "n_pages"), ("n_pages", 11, -1, "differ"),
    ("page_tokens", 8, -4, "page_tokens"), ("page_tokens", 32, -1, "differ"), ("head_dim", 96, -4, "head_dim"), ("format", 2, -4, "format"),
    ("n_kv_heads", 0, -1, "n_kv_heads"), ("n_kv_heads", 1 << 28, -4, "2^31")])
def test_caches_refused(fb, args, field, value, code, text):
    c, b, a = args
    setattr(c, field, value)
    if field == "n_kv_heads" and value:
        a.n_q_heads = value
    refused(fb, code, text, "fence_kv8_attention", c, b, a, None)
    refused(fb, code, text, "fence_kv8_store", c, b, OK, OK, 0, 256, 256, None)
    if "differ" not in text:
        refused(fb, code, text, "fence_kv8_load", c, OK, 1, OK, OK, 0, 256, 256, None)


def test_store_and_load_refuse(fb, args):
    c, b, _ = args
    refused(fb, -1, "null", "fence_kv8_store", c, b, None, OK, 0, 256, 256, None)
    refused(fb, -4, "type", "fence_kv8_store", c, b, OK, OK, 3, 256, 256, None)
    refused(fb, -1, "strides", "fence_kv8_store", c, b, OK, OK, 0, 255, 256, None)
    refused(fb, -2, "aligned", "fence_kv8_store", c, b, OK + 2, OK, 0, 256, 256, None)
    refused(fb, -1, "bad arguments", "fence_kv8_load", c, None, 1, OK, OK, 0, 256, 256, None)
    refused(fb, -1, "bad arguments", "fence_kv8_load", c, OK, 1, None, None, 0, 256, 256, None)
    refused(fb, -1, "strides", "fence_kv8_load", c, OK, 1, None, OK, 0, 0, 255, None)
    refused(fb, -2, "aligned", "fence_kv8_load", c, OK, 1, None, OK + 1, 1, 0, 256, None)
    b.n_tokens = 0
    assert fb.lib().fence_kv8_store(c, b, None, None, 0, 0, 0, None) == 0  # nothing to do
    assert fb.lib().fence_kv8_load(c, None, 0, None, None, 0, 0, 0, None) == 0


@pytest.mark.parametrize("field,value,code,text", [
    ("q", None, -1, "null"), ("workspace", None, -1, "null"), ("workspace", OK + 16, -2, "256-byte"), ("workspace_bytes", 8, -8, "needs"),
    ("n_q_heads", 7, -1, "query heads"), ("type", 5, -4, "type"), ("q_stride", 1023, -1, "strides"), ("out_stride", 1000, -1, "strides"),
    ("max_new", 0, -1, "max_new"), ("scale", -0.5, -1, "scale"),
    ("scale", float("nan"), -1, "scale"), ("scale", float("inf"), -1, "scale"), ("q", OK + 2, -2, "aligned")])
def test_attention_refuses(fb, args, field, value, code, text):
    c, b, a = args
    setattr(a, field, value)
    refused(fb, code, text, "fence_kv8_attention", c, b, a, None)


def test_attention_of_no_tokens(fb, args):
    c, b, a = args
    b.n_tokens = 0
    assert fb.lib().fence_kv8_attention(c, b, a, None) == 0
