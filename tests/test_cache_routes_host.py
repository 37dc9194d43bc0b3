"""Which kernels attention over the cache takes at which sizes (no GPU needed): the rules by their sizes, and that the parts' number and
the workspace stay within what the launches and callers rely on."""
import ctypes as C

import pytest

from tensorrt_amd import capi


@pytest.fixture(scope="module")
def api():
    return capi.api()


def params(B=1, n=1, length=1000, H=8, heads=32, d=128, P=64, window=0, sinks=0, T=None, max_pages=None):
    c = capi.KvCache(data_type=2, pages=1000, page_tokens=P, kv_heads=H, d=d, B=B, max_pages=max_pages or -(-length // P), max_tokens=n,
                     T=T or B * n)
    return C.byref(capi.KvCacheAttentionParams(cache=c, q_heads=heads, scale=1.0, window=window, sinks=sinks, max_length=length))


def route(api, **k):
    r = api.test_kv_cache_attention_route(params(**k))
    return dict(waves=r & 15, stretches=bool(r & 16), aligned=bool(r & 32), tiles=bool(r & 64), parts=r >> 8)


@pytest.mark.parametrize("k,want", [
    # short contexts: one launch, more wavefronts where there are few heads; up to 128 KB of keys and values a head
    (dict(length=300), dict(waves=8, stretches=False)), (dict(length=512), dict(waves=8, stretches=False)),
    (dict(length=513), dict(waves=0, stretches=True)), (dict(length=1024, d=64), dict(waves=8, stretches=False)),
    (dict(length=1025, d=64), dict(stretches=True)), (dict(B=64, length=500), dict(waves=4, stretches=False)),
    (dict(length=300, d=256), dict(stretches=True)), (dict(length=200, d=256), dict(waves=4)),
    # few heads: stretches of one head each; many: across them; very many: one workgroup each
    (dict(length=100000), dict(stretches=True, aligned=True)), (dict(B=16, length=4000), dict(stretches=True, aligned=True)),
    (dict(B=17, length=4000), dict(stretches=True, aligned=False)), (dict(B=64, length=8000), dict(stretches=True, aligned=False)),
    (dict(B=511, length=8000), dict(stretches=True)), (dict(B=512, length=8000), dict(waves=4, stretches=False)),
    (dict(B=1024, H=1, heads=4, length=8000), dict(stretches=True)), (dict(B=1025, H=1, heads=4, length=8000), dict(waves=4, stretches=False)),
    # a window bounds what there is to share
    (dict(length=100000, window=300), dict(waves=8, stretches=False)), (dict(length=100000, window=3000), dict(stretches=True)),
    # rows of a key head: 16 and more
    (dict(n=4), dict(tiles=False)), (dict(n=5), dict(tiles=True, waves=0, stretches=False)), (dict(B=2, n=5, T=9), dict(tiles=True, stretches=True)),
    (dict(B=2, n=5), dict(tiles=True, stretches=False, waves=0)), (dict(B=8, n=512, T=4096), dict(tiles=True, stretches=False, waves=0)),
    (dict(B=8, n=512, T=3000), dict(tiles=True, stretches=True)),
    (dict(n=1, heads=136), dict(tiles=True, waves=0)), (dict(B=3, n=1, heads=136), dict(tiles=True, waves=0, stretches=False)),
    # tiles enough for the chip: whole keys; otherwise parts
    (dict(B=4, n=1024, length=9000), dict(tiles=True, parts=1)), (dict(n=64, length=100000), dict(tiles=True)), (dict(n=8192, length=8192), dict(parts=1))])
def test_rules(api, k, want):
    got = route(api, **k)
    assert {n: got[n] for n in want} == want, got


def test_parts_of_few_tiles(api):
    assert route(api, n=64, length=100000)["parts"] > 10
    assert route(api, n=64, length=500)["parts"] <= 2


@pytest.mark.parametrize("k", [dict(length=131072), dict(B=64, length=131072), dict(B=64, n=512, length=131072), dict(B=1, n=40, length=1 << 27, P=128),
                               dict(B=1024, length=1 << 20), dict(B=65535, n=1, length=100), dict(B=2, n=5, length=1 << 27, P=16),
                               dict(n=100, length=500, max_pages=1 << 20), dict(n=20, H=1, heads=1, length=1, max_pages=1 << 20),
                               dict(B=3, n=6, H=1, heads=8, length=1000, max_pages=1 << 16)])
def test_workspace_is_bounded(api, k):
    """Sums of a fixed number of stretches, and of no more parts than fill the chip four times over, whatever the pages allow."""
    r, size = route(api, **k), api.kv_cache_attention_workspace_size(params(**k))
    assert r["parts"] < 65536
    assert size < 240 << 20


def test_refused_sizes(api):
    assert api.test_kv_cache_attention_route(None) == -1
    assert api.test_kv_cache_attention_route(params(heads=12)) == -1
    assert api.test_kv_cache_attention_route(params(B=0, T=1)) == -1
