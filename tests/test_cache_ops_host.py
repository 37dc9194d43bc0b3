"""What the entry points of the 8-bit cache and of attention in windows refuse, before anything is launched (no GPU needed)."""
import ctypes as C

import pytest

from tensorrt_amd import capi

A = 0x10000  # an aligned address


@pytest.fixture(scope="module")
def api():
    return capi.api()


def refused(api, status, *words):
    assert status != 0
    text = api.last_error_str()
    for w in words:
        assert w in text, text


def cache(**change):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, page_table=A, lengths=A, cu_seqlens=A, data_type=2, pages=9, page_tokens=16, kv_heads=2, d=64,
             B=3, max_pages=4, max_tokens=5, T=7)
    f.update({n: v for n, v in change.items() if n in f})
    return capi.KvCache(**f)


def copied(kind, **change):
    f = dict(k=A, v=A, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
    f.update({n[5:]: v for n, v in change.items() if n.startswith("rows_")})
    return C.byref(kind(cache=cache(**change), **f))


def attention(**change):
    f = dict(q=A, out=A, q_token_stride=256, q_head_stride=64, out_token_stride=256, out_head_stride=64, q_heads=4, scale=0.125, window=0,
             sinks=0, max_length=40, workspace=A, workspace_bytes=1 << 30)
    f.update({n: v for n, v in change.items() if n in f})
    return C.byref(capi.KvCacheAttentionParams(cache=cache(**change), **f))


CACHE = [
    (dict(data_type=1), "data_type 1"), (dict(data_type=0), "data_type 0"), (dict(page_tokens=8), "page_tokens=8"),
    (dict(page_tokens=48), "page_tokens=48"), (dict(page_tokens=256), "page_tokens=256"), (dict(page_tokens=0), "page_tokens=0"),
    (dict(d=0), "d=0"), (dict(d=72), "d=72"), (dict(d=272), "d=272"), (dict(d=-16), "d=-16"), (dict(kv_heads=0), "kv_heads=0"),
    (dict(B=-1), "B=-1"), (dict(T=-1), "T=-1"), (dict(max_tokens=-1), "max_tokens=-1"), (dict(max_pages=-1), "max_pages=-1"),
    (dict(max_pages=0), "max_pages=0"), (dict(pages=0), "pages=0"), (dict(B=65536), "65535"),
    (dict(max_pages=(1 << 26) + 1), "2^30"), (dict(pages=1 << 30), "2^31"), (dict(k_scale=0), "null"), (dict(v_scale=0), "null"), (dict(page_table=0), "null"), (dict(lengths=0), "null"),
    (dict(cu_seqlens=0), "null"), (dict(k_scale=A + 2), "aligned"), (dict(page_table=A + 1), "aligned"), (dict(lengths=A + 2), "aligned")]


@pytest.mark.parametrize("change,word", CACHE)
def test_cache_refused_everywhere(api, change, word):
    refused(api, api.kv_cache_write(None, copied(capi.KvCacheWriteParams, **change)), word, "kv_cache_write")
    refused(api, api.kv_cache_read(None, copied(capi.KvCacheReadParams, **change)), word, "kv_cache_read")
    refused(api, api.kv_cache_attention(None, attention(**change)), word, "kv_cache_attention")


@pytest.mark.parametrize("change,word", [
    (dict(rows_k=0), "null"), (dict(rows_v=0), "null"), (dict(rows_k=A + 2), "aligned"), (dict(rows_v=A + 8), "aligned"),
    (dict(rows_k_token_stride=100), "strides"), (dict(rows_v_head_stride=-8), "strides"), (dict(kv_heads=16384), "16383"), (dict(pages=1 << 30), "2^31")])
def test_copies_refuse(api, change, word):
    refused(api, api.kv_cache_write(None, copied(capi.KvCacheWriteParams, **change)), word)
    refused(api, api.kv_cache_read(None, copied(capi.KvCacheReadParams, **change)), word)


@pytest.mark.parametrize("change,word", [
    (dict(q_heads=0), "q_heads=0"), (dict(q_heads=3), "q_heads=3"), (dict(q_heads=-2), "q_heads=-2"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(window=-1), "window=-1"), (dict(sinks=-1), "sinks=-1"),
    (dict(max_length=-1), "max_length=-1"), (dict(q=0), "null"), (dict(out=0), "null"), (dict(q=A + 8), "aligned"),
    (dict(out=A + 2), "aligned"), (dict(q_token_stride=250), "strides"), (dict(out_head_stride=-64), "strides"),
    (dict(T=1 << 28, q_heads=4), "2^30"),
    (dict(max_pages=1 << 12, max_length=0, workspace=0), "workspace"), (dict(max_pages=1 << 12, max_length=0, workspace=A + 8), "workspace"),
    (dict(max_pages=1 << 12, max_length=0, workspace_bytes=64), "workspace")])
def test_attention_refuses(api, change, word):
    refused(api, api.kv_cache_attention(None, attention(**change)), word)


def window(**change):
    f = dict(q=A, k=A, v=A, out=A, cu_seqlens=A, B=2, T=9, max_tokens=5, q_heads=4, kv_heads=2, d=64, scale=0.125, left=3, right=3, sinks=1)
    f.update({f"{n}_{s}_stride": 64 for n in ("q", "k", "v", "out") for s in ("token", "head")})
    f.update(change)
    return C.byref(capi.WindowAttentionParams(**f))


@pytest.mark.parametrize("change,word", [
    (dict(B=-1), "B=-1"), (dict(T=-1), "T=-1"), (dict(max_tokens=-1), "max_tokens=-1"), (dict(q_heads=0), "q_heads=0"),
    (dict(q_heads=3), "q_heads=3"), (dict(kv_heads=0), "kv_heads=0"), (dict(d=0), "d=0"), (dict(d=60), "d=60"), (dict(d=264), "d=264"),
    (dict(scale=-0.5), "scale"), (dict(scale=float("nan")), "scale"), (dict(left=-2), "left=-2"), (dict(right=-2), "right=-2"),
    (dict(sinks=-1), "sinks=-1"), (dict(q=0), "null"), (dict(k=0), "null"), (dict(v=0), "null"), (dict(out=0), "null"),
    (dict(cu_seqlens=0), "null"), (dict(q=A + 8), "aligned"), (dict(out=A + 2), "aligned"), (dict(cu_seqlens=A + 2), "aligned"),
    (dict(k_token_stride=68), "strides"), (dict(v_head_stride=-64), "strides"), (dict(B=65536), "65535"),
    (dict(T=1 << 29, max_tokens=1 << 29), "2^30"), (dict(q_heads=65536, kv_heads=65536, T=1), "65535")])
def test_window_refuses(api, change, word):
    refused(api, api.window_attention(None, window(**change)), word, "window_attention")


def test_null_parameters(api):
    for f in (api.kv_cache_write, api.kv_cache_read, api.kv_cache_attention, api.window_attention):
        refused(api, f(None, None), "null params")
    assert api.kv_cache_attention_workspace_size(None) == 0


@pytest.mark.parametrize("change", [dict(B=0), dict(T=0), dict(max_tokens=0)])
def test_nothing_to_do(api, change):
    gone = dict(k=0, v=0, k_scale=0, v_scale=0, page_table=0, lengths=0, cu_seqlens=0)
    assert api.kv_cache_write(None, copied(capi.KvCacheWriteParams, rows_k=0, rows_v=0, **change, **gone)) == 0
    assert api.kv_cache_read(None, copied(capi.KvCacheReadParams, rows_k=0, rows_v=0, **change, **gone)) == 0
    assert api.kv_cache_attention(None, attention(q=0, out=0, workspace=0, **change, **gone)) == 0
    assert api.kv_cache_attention_workspace_size(attention(**change)) == 0
    assert api.window_attention(None, window(q=0, k=0, v=0, out=0, cu_seqlens=0, **change)) == 0


def test_workspace_follows_sizes_alone(api):
    size = api.kv_cache_attention_workspace_size(attention(max_pages=1 << 12, max_length=0))
    assert size > 0
    gone = dict(k=0, v=0, k_scale=0, v_scale=0, page_table=0, lengths=0, cu_seqlens=0, q=0, out=0, workspace=0, workspace_bytes=0)
    assert api.kv_cache_attention_workspace_size(attention(max_pages=1 << 12, max_length=0, **gone)) == size
    assert api.kv_cache_attention_workspace_size(attention(q_heads=3)) == 0


SIZES = [(change, word) for change, word in CACHE if word not in ("null", "aligned")] + [
    (dict(kv_heads=16384, q_heads=16384), "16383"), (dict(d=300), "d=300"), (dict(d=24), "d=24"), (dict(d=2 ** 31 - 1), "d="), (dict(q_heads=0), "q_heads=0"),
    (dict(q_heads=3), "q_heads=3"), (dict(q_heads=-2), "q_heads=-2"), (dict(window=-1), "window=-1"), (dict(sinks=-1), "sinks=-1"),
    (dict(max_length=-1), "max_length=-1"), (dict(T=1 << 28), "2^30")]


@pytest.mark.parametrize("change,word", SIZES)
def test_no_workspace_for_sizes_that_are_refused(api, change, word):
    """0 where the call refuses the sizes, and the error says which, with pages enough to need a workspace; no pointer is looked at."""
    gone = dict(k=0, v=0, k_scale=0, v_scale=0, page_table=0, lengths=0, cu_seqlens=0, q=0, out=0, workspace=0)
    more = {**dict(max_pages=1 << 12, max_length=0), **gone, **change}
    refused(api, api.kv_cache_attention(None, attention(**more)), word, "kv_cache_attention")
    assert api.kv_cache_attention_workspace_size(attention(**more)) == 0
    assert word in api.last_error_str() and "workspace_size" in api.last_error_str()
    assert api.test_kv_cache_attention_route(attention(**more)) == -1
