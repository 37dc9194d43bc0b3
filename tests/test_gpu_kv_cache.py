"""The 8-bit cache: bytes and scales against the definition operation by operation, what comes back exactly, attention over it against
binary64 with the tolerance of cache_helpers.attention_reference."""
import ctypes as C

import numpy as np
import pytest

from cache_helpers import Cache, assert_within, attention_reference, round_codes, values, visible_keys
from helpers import dev, dev_empty, host, ptr, rng, stream, sync
from tensorrt_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    return capi.api()


def new_rows(r, T, H, d):
    """Keys and values as a projection leaves them, [token][head][k|v][d], some tokens louder than others."""
    kv = r.standard_normal((T, H, 2, d)) * np.exp(r.standard_normal((T, H, 1, 1)))
    return kv.astype(np.float16)


def write(api, cache, kv, cu, s=None, **more):
    t = dev(kv)
    c, keep = cache.described(cu, **more)
    H, d = kv.shape[1], kv.shape[3]
    p = capi.KvCacheWriteParams(cache=c, k=ptr(t), v=ptr(t) + 2 * d, k_token_stride=H * 2 * d, k_head_stride=2 * d,
                                v_token_stride=H * 2 * d, v_head_stride=2 * d)
    api.check(api.kv_cache_write(stream() if s is None else s, C.byref(p)))
    sync()
    cache.write(kv[:, :, 0], kv[:, :, 1], cu, **more)


def read(api, cache, cu, T=None, **more):
    rows = int(cu[-1]) if T is None else T
    k, v = (dev_empty((rows + 1, cache.H, cache.d), np.float16, fill=-7) for _ in range(2))
    c, keep = cache.described(cu, T=T, **more)
    p = capi.KvCacheReadParams(cache=c, k=ptr(k), v=ptr(v), k_token_stride=cache.H * cache.d, k_head_stride=cache.d,
                               v_token_stride=cache.H * cache.d, v_head_stride=cache.d)
    api.check(api.kv_cache_read(stream(), C.byref(p)))
    sync()
    return host(k), host(v)


def attention_params(cache, cu, q, out, scale, window=0, sinks=0, max_length=0, ws=None, api=None, **more):
    c, keep = cache.described(cu, **more)
    heads, d = q.shape[1], q.shape[2]
    p = capi.KvCacheAttentionParams(cache=c, q=ptr(q), out=ptr(out), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                                    out_token_stride=out.stride(0), out_head_stride=out.stride(1), q_heads=heads, scale=scale, window=window,
                                    sinks=sinks, max_length=max_length)
    size = api.kv_cache_attention_workspace_size(C.byref(p))
    ws = dev_empty((max(size, 16),), np.uint8, fill=0xFF) if ws is None else ws  # NaN everywhere
    p.workspace, p.workspace_bytes = ptr(ws), size
    return p, (keep, ws)


def attend(api, cache, cu, q, scale, **more):
    dq, out = dev(q), dev_empty(q.shape, np.float16, fill=-7)
    p, keep = attention_params(cache, cu, dq, out, scale, api=api, **more)
    api.check(api.kv_cache_attention(stream(), C.byref(p)))
    sync()
    return host(out)


def check_attention(cache, cu, q, got, scale, window=0, sinks=0, sample=None, T=None, max_tokens=None):
    """Rows of every sequence, head by head; sample: only so many of them."""
    group = q.shape[1] // cache.H
    r = rng(5)
    T = len(q) if T is None else T
    for b in range(cache.B):
        k, sk, there = cache.codes_of(b, "k")
        v, sv, _ = cache.codes_of(b, "v")
        n = int(cu[b + 1] - cu[b])
        rows = np.arange(n)
        if sample and n * q.shape[1] > sample:
            rows = np.unique(np.concatenate([[0, n - 1], r.integers(0, n, max(sample // q.shape[1], 1))]))
        for i in rows:
            t = int(cu[b]) + i
            if t >= T or (max_tokens is not None and i >= max_tokens):
                assert (got[t] == -7).all()
                continue
            at = int(cache.lengths[b]) - n + i
            ok = visible_keys(at, len(k), window - 1 if window else None, 0, sinks) & there
            for h in range(q.shape[1]):
                want, tol = attention_reference(q[t, h], k[:, h // group], sk[:, h // group], v[:, h // group], sv[:, h // group], ok, scale)
                assert_within(got[t, h], want, tol, f"sequence {b} row {i} head {h}")


def filled(api, dtype, P, H, d, lens, seed=0, spare=2, max_pages=None):
    """A cache whose sequences have `lens` tokens, written by the kernel and followed by the model."""
    pages = sum(-(-n // P) for n in lens) + spare
    cache = Cache(dtype, P, H, d, pages, len(lens), max_pages or max(-(-max(lens) // P), 1) + 1, seed)
    cache.grow(lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    write(api, cache, new_rows(cache.r, int(cu[-1]), H, d), cu)
    return cache


WRITES = [("int8", 16, 1, 16, [1]), ("fp8", 16, 1, 16, [1]), ("int8", 16, 3, 64, [5, 16, 33]), ("fp8", 32, 2, 80, [31, 1, 70]),
          ("int8", 64, 2, 128, [64, 65, 130]), ("fp8", 64, 4, 128, [1, 100]), ("int8", 128, 1, 256, [300, 7]), ("fp8", 128, 2, 96, [129, 2]),
          ("int8", 32, 5, 48, [40, 3, 1, 9]), ("fp8", 16, 2, 256, [17, 16])]


@pytest.mark.parametrize("dtype,P,H,d,lens", WRITES)
def test_write(api, dtype, P, H, d, lens):
    """Prompts, then tokens one by one and a few at a time, across the ends of pages; every byte of the pool after each call."""
    B = len(lens)
    cache = Cache(dtype, P, H, d, sum(-(-(n + 40) // P) for n in lens) + 3, B, -(-(max(lens) + 40) // P) + 1, seed=len(lens) + d)
    r = cache.r
    for new in [lens, [1] * B, [3] * B, [1] * B, [0] + [2] * (B - 1), list(r.integers(0, 12, B)), [17] * B]:
        cu = np.concatenate([[0], np.cumsum(new)])
        if cu[-1] == 0:
            continue
        cache.grow(new)
        write(api, cache, new_rows(r, int(cu[-1]), H, d), cu)
        cache.check()


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
def test_write_extremes(api, dtype):
    """Zeros, subnormals and the largest values, a page that grows from each to each, ties, and what is not a number."""
    H, d, P = 2, 32, 16
    cache = Cache(dtype, P, H, d, 12, 1, 10, seed=3)
    r = cache.r
    one = lambda f: np.broadcast_to(np.float16(f), (1, H, 2, d)).copy()
    ties = (np.arange(d) - 15.5).astype(np.float16)[None, None, None] * np.ones((1, H, 2, 1), np.float16)
    steps = [one(0), one(2.0 ** -24), one(0), one(1e-3), ties, one(65504), one(-65504), one(0), new_rows(r, 1, H, d)]
    steps += [new_rows(r, 5, H, d) * np.float16(2.0 ** -14), new_rows(r, 9, H, d) * np.float16(100), one(2.0 ** -24), one(3e-8)]
    for x in steps:
        cache.grow([len(x)])
        write(api, cache, x, [0, len(x)])
        cache.check()
    bad = new_rows(r, 3, H, d)
    bad[1, 0, 0, 3], bad[1, 1, 1, 0] = np.nan, np.inf
    for x in (bad, new_rows(r, 2, H, d), new_rows(r, 20, H, d)):  # the page stays without a number; the next ones are sound
        cache.grow([len(x)])
        write(api, cache, x, [0, len(x)])
        cache.check()
    assert np.isnan(cache.ks).sum() == 1 and np.isnan(cache.vs).sum() == 1


def test_drift_is_bounded(api):
    """A page whose tokens get louder one by one: each token is within a step of the last scale."""
    H, d, P = 1, 64, 64
    cache = Cache("int8", P, H, d, 2, 1, 1, seed=4)
    x = (cache.r.uniform(-1, 1, (P, H, 2, d)) * 1.07 ** np.arange(P)[:, None, None, None]).astype(np.float16)
    for t in range(P):
        cache.grow([1])
        write(api, cache, x[t:t + 1], [0, 1])
    cache.check()
    page = cache.table[0, 0]
    back = values(cache.k[page, 0], "int8") * cache.ks[page, 0]
    assert np.abs(back - x[:, 0, 0]).max() <= cache.ks[page, 0] * (1 + 1e-5)


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
def test_what_does_not_fit_is_left_out(api, dtype):
    """Rows behind T and max_tokens, tokens before a sequence's first and behind its pages, pages that are none."""
    H, d, P = 2, 64, 16
    cache = Cache(dtype, P, H, d, 9, 4, 2, seed=6)
    cache.lengths = np.array([20, 40, 5, 30], np.int32)
    cache.table = np.array([[0, 1], [2, 3], [4, -1], [9, 5]], np.int32)  # 9: behind the pool
    cache.dtable.copy_(dev(cache.table))
    cache.dlengths.copy_(dev(cache.lengths))
    for new, more in (([20, 40, 5, 30], {}), ([3, 12, 9, 20], {}), ([20, 17, 3, 9], dict(T=45)), ([20, 17, 3, 9], dict(max_tokens=10))):
        cu = np.concatenate([[0], np.cumsum(new)])
        kv = new_rows(cache.r, int(cu[-1]), H, d)
        write(api, cache, kv, cu, **more)
        cache.check()
        k, v = read(api, cache, cu, **more)
        want_k, want_v = np.full(k.shape, -7, np.float16), np.full(v.shape, -7, np.float16)
        for b in range(4):
            ck, sk, there = cache.codes_of(b, "k")
            cv, sv, _ = cache.codes_of(b, "v")
            for i in range(new[b]):
                t, at = int(cu[b]) + i, int(cache.lengths[b]) - new[b] + i
                if t >= more.get("T", 1 << 30) or i >= more.get("max_tokens", 1 << 30):
                    continue
                seen = 0 <= at < len(there) and there[at]
                want_k[t] = ck[at] * sk[at][:, None] if seen else 0
                want_v[t] = cv[at] * sv[at][:, None] if seen else 0
        assert np.array_equal(k, want_k) and np.array_equal(v, want_v)


@pytest.mark.parametrize("dtype,P,H,d,lens", WRITES)
def test_read(api, dtype, P, H, d, lens):
    """Whole sequences and their last tokens, bit for bit."""
    cache = filled(api, dtype, P, H, d, lens)
    for new in (lens, [1] * len(lens), [max(n // 2, 1) for n in lens]):
        cu = np.concatenate([[0], np.cumsum(new)])
        got = read(api, cache, cu)
        for x, which in zip(got, "kv"):
            assert (x[-1] == -7).all()
            for b, n in enumerate(new):
                codes, scales, _ = cache.codes_of(b, which)
                want = (codes * scales[..., None]).astype(np.float16)[len(codes) - n:]
                assert np.array_equal(x[cu[b]:cu[b + 1]], want)


# dtype, page, key heads, query heads, d, lengths, rows of the call, window, sinks
ATTENTION = [
    ("int8", 16, 1, 1, 16, [1], [1], 0, 0), ("fp8", 16, 1, 1, 64, [2], [1], 0, 0), ("int8", 64, 2, 8, 128, [63, 64, 65], [1, 1, 1], 0, 0),
    ("fp8", 16, 4, 4, 64, [300, 1, 17, 129], [1, 1, 1, 1], 0, 0), ("int8", 32, 2, 6, 80, [200, 31], [2, 3], 0, 0),
    ("fp8", 128, 1, 16, 96, [500], [1], 0, 0), ("int8", 16, 2, 2, 256, [700, 64], [1, 4], 0, 0), ("fp8", 64, 1, 2, 256, [90], [90], 0, 0),
    ("int8", 16, 2, 8, 128, [1000, 40], [3, 3], 100, 4), ("fp8", 32, 2, 8, 64, [1000, 40, 512], [1, 2, 1], 64, 70),
    ("int8", 64, 1, 4, 48, [257], [1], 1, 0), ("fp8", 64, 1, 4, 48, [257], [1], 1, 1),
    ("int8", 64, 2, 4, 128, [40, 300, 128], [40, 300, 128], 0, 0), ("fp8", 16, 1, 7, 80, [333], [100], 0, 0),
    ("int8", 32, 2, 2, 64, [600, 129], [257, 129], 50, 0), ("fp8", 128, 2, 8, 128, [777, 200], [130, 33], 150, 5),
    ("int8", 16, 1, 8, 128, [513, 90, 7, 300], [1, 40, 7, 2], 0, 0), ("fp8", 64, 2, 16, 96, [300, 301], [5, 1], 40, 17)]


@pytest.mark.parametrize("dtype,P,H,heads,d,lens,new,window,sinks", ATTENTION)
def test_attention(api, dtype, P, H, heads, d, lens, new, window, sinks):
    cache = filled(api, dtype, P, H, d, lens, seed=d + len(lens))
    cu = np.concatenate([[0], np.cumsum(new)])
    q = (2 * cache.r.standard_normal((int(cu[-1]), heads, d))).astype(np.float16)
    for max_length in (0, max(lens), 1):  # other ways to share the work out
        got = attend(api, cache, cu, q, 1 / np.sqrt(d), window=window, sinks=sinks, max_length=max_length)
        check_attention(cache, cu, q, got, 1 / np.sqrt(d), window, sinks, sample=60)


@pytest.mark.parametrize("dtype,heads,lens,new,window", [("int8", 8, [9000], [1], 0), ("fp8", 16, [5000, 20], [1, 1], 0),
                                                         ("int8", 4, [7000], [200], 0), ("fp8", 8, [12000], [3], 3000)])
def test_long_contexts(api, dtype, heads, lens, new, window):
    """Keys shared between many workgroups."""
    cache = filled(api, dtype, 64, 2, 128, lens, max_pages=200)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = cache.r.standard_normal((int(cu[-1]), heads, 128)).astype(np.float16)
    for max_length in (0, max(lens)):
        got = attend(api, cache, cu, q, 0.1, window=window, sinks=4 if window else 0, max_length=max_length)
        check_attention(cache, cu, q, got, 0.1, window, 4 if window else 0, sample=16)


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
@pytest.mark.parametrize("few", [True, False])
def test_rows_that_see_nothing_and_pages_that_are_gone(api, dtype, few):
    """Pages given back from under a window, rows before a sequence's first token, a sequence of no tokens; a page without a number
    touches nobody who does not see it."""
    H, heads, d, P = 2, 4, 64, 16
    lens = [200, 3, 64, 40]
    cache = filled(api, dtype, P, H, d, lens, max_pages=13)
    cache.table[0, 2:7] = -1
    cache.table[0, 8] = cache.pages + 5
    cache.table[2, 0] = -1
    cache.lengths[3] = 0
    cache.ks[cache.table[0, 1], 0] = np.nan
    cache.vs[cache.table[2, 1], 1] = np.nan
    cache.upload()
    new = [3, 5, 4, 2] if few else [50, 40, 33, 20]  # sequence 1: rows before its first token
    cu = np.concatenate([[0], np.cumsum(new)])
    q = cache.r.standard_normal((int(cu[-1]), heads, d)).astype(np.float16)
    for window, sinks in ((0, 0), (20, 0), (60, 3), (20, 40)):
        got = attend(api, cache, cu, q, 0.125, window=window, sinks=sinks)
        check_attention(cache, cu, q, got, 0.125, window, sinks)
    assert (got[cu[3]:] == 0).all() and (got[cu[1]:cu[1] + new[1] - 3] == 0).all()


@pytest.mark.parametrize("more", [dict(T=20), dict(max_tokens=6), dict(T=31, max_tokens=25)])
def test_rows_left_out_stay(api, more):
    cache = filled(api, "int8", 16, 2, 64, [100, 50, 30])
    new = [30, 6, 9]
    cu = np.concatenate([[0], np.cumsum(new)])
    q = cache.r.standard_normal((int(cu[-1]), 4, 64)).astype(np.float16)
    got = attend(api, cache, cu, q, 0.125, **more)
    check_attention(cache, cu, q, got, 0.125, **more)


@pytest.mark.parametrize("lengths,cu,T", [
    ([2 ** 31 - 1, 100, -5], [0, 2, 4, 6], 6), ([64, 64, 64], [3, 1, 6, 2], 6), ([64, 64, 64], [-7, 2, 2 ** 31 - 1, 5], 6),
    ([2 ** 31 - 1] * 3, [0, 20, 40, 60], 60), ([64, 2 ** 30, 33], [50, 10, 45, 60], 60)])
def test_tables_of_no_sense(api, lengths, cu, T):
    """Lengths and rows that no cache has: everything stays within the call's tensors and the pool, and what is out of them stays."""
    cache = filled(api, "int8", 16, 2, 64, [64, 64, 64])
    cache.lengths = np.array(lengths, np.int32)
    cache.dlengths.copy_(dev(cache.lengths))
    kv, q = new_rows(cache.r, T, 2, 64), cache.r.standard_normal((T, 4, 64)).astype(np.float16)
    n = max(1, min(T, 40))
    for window in (0, 10):
        out = attend(api, cache, np.array(cu), q, 0.125, window=window, T=T, max_tokens=n)
        assert np.isfinite(out).all()
    k, v = read(api, cache, np.array(cu), T=T, max_tokens=n)
    assert (k[T] == -7).all() and (v[T] == -7).all()
    c, keep = cache.described(cu, T=T, max_tokens=n)
    t = dev(kv)
    s = dict(k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128)
    api.check(api.kv_cache_write(stream(), C.byref(capi.KvCacheWriteParams(cache=c, k=ptr(t), v=ptr(t) + 128, **s))))
    sync()


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
def test_scales_far_apart(api, dtype):
    """Pages whose values are 2^20 times others': the weights keep their digits whatever the scales are; a page of zeros counts too."""
    H, d, P = 1, 64, 16
    cache = filled(api, dtype, P, H, d, [160, 160])
    cache.ks[:] = 1.0 / (100 if dtype == "int8" else 400)
    for i in range(10):
        cache.vs[cache.table[0, i], 0] = 2.0 ** (2 * i - 12)
        cache.vs[cache.table[1, i], 0] = 2.0 ** (8 - 2 * i)
    cache.v[cache.table[0, 3]] = 0
    cache.vs[cache.table[0, 3]] = 0
    cache.upload()
    for new in ([1, 1], [30, 30]):
        cu = np.concatenate([[0], np.cumsum(new)])
        q = cache.r.standard_normal((int(cu[-1]), 2, d)).astype(np.float16)
        for window in (0, 17):
            check_attention(cache, cu, q, attend(api, cache, cu, q, 0.125, window=window), 0.125, window)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 30.0])
def test_scales_of_the_scores(api, scale):
    """All weights alike, and all but one nothing."""
    cache = filled(api, "int8", 16, 1, 64, [100, 7])
    cu = np.array([0, 2, 4])
    q = cache.r.standard_normal((4, 2, 64)).astype(np.float16)
    check_attention(cache, cu, q, attend(api, cache, cu, q, scale), np.float32(scale))


def test_strides_and_in_place(api):
    """Queries in the packing of the projection, results over them."""
    H, heads, d = 2, 4, 64
    cache = filled(api, "fp8", 32, H, d, [100, 30])
    for new in ([2, 3], [60, 30]):
        cu = np.concatenate([[0], np.cumsum(new)])
        T = int(cu[-1])
        q = cache.r.standard_normal((T, heads + 2 * H, d)).astype(np.float16)
        t = dev(q)
        p, keep = attention_params(cache, cu, t[:, :heads], t[:, :heads], 0.125, api=api)
        api.check(api.kv_cache_attention(stream(), C.byref(p)))
        sync()
        got = host(t)
        assert np.array_equal(got[:, heads:], q[:, heads:])
        check_attention(cache, cu, q[:, :heads], got[:, :heads], 0.125)


def test_pool_past_4_gib(api):
    """Pages whose offsets pass 32 bits, written, read and attended to."""
    import torch
    P, H, d = 128, 8, 128
    pages = (1 << 32) // (P * H * d) + 40
    k, v = (torch.empty(pages * P * H * d, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, H), device="cuda") for _ in range(2))
    small = Cache("int8", P, H, d, 4, 1, 4, seed=2)
    small.grow([300])
    cu = np.array([0, 300])
    kv = new_rows(small.r, 300, H, d)
    small.write(kv[:, :, 0], kv[:, :, 1], cu)
    far = small.table[0] + pages - 5  # the same, at the pool's end
    table = dev(np.where(small.table[0] < 0, -1, far).astype(np.int32))

    def described(cu):
        c, keep = small.described(cu)
        c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.pages = ptr(k), ptr(v), ptr(ks), ptr(vs), ptr(table), pages
        return c, keep
    t = dev(kv)
    c, keep = described(cu)
    s = dict(k_token_stride=2 * H * d, k_head_stride=2 * d, v_token_stride=2 * H * d, v_head_stride=2 * d)
    api.check(api.kv_cache_write(stream(), C.byref(capi.KvCacheWriteParams(cache=c, k=ptr(t), v=ptr(t) + 2 * d, **s))))
    back = dev_empty((300, H, 2, d), np.float16, fill=0)
    api.check(api.kv_cache_read(stream(), C.byref(capi.KvCacheReadParams(cache=c, k=ptr(back), v=ptr(back) + 2 * d, **s))))
    sync()
    for i, which in enumerate("kv"):
        codes, scales, _ = small.codes_of(0, which)
        assert np.array_equal(host(back)[:, :, i], (codes * scales[..., None]).astype(np.float16))
    for n in (1, 20):
        cu = np.array([0, n])
        q = small.r.standard_normal((n, H, d)).astype(np.float16)
        dq, out = dev(q), dev_empty(q.shape, np.float16, fill=-7)
        p, keep2 = attention_params(small, cu, dq, out, 0.1, api=api)
        p.cache, keep3 = described(cu)
        api.check(api.kv_cache_attention(stream(), C.byref(p)))
        sync()
        check_attention(small, cu, q, host(out), 0.1, sample=16)


def test_tensors_longer_than_their_sequences(api):
    """As many rows as if all sequences had the most, though two have one: nobody is left out."""
    cache = filled(api, "int8", 32, 2, 64, [300, 200, 90])
    cu = np.array([0, 50, 51, 52])
    q = cache.r.standard_normal((150, 8, 64)).astype(np.float16)
    got = attend(api, cache, cu, q, 0.125, T=150)
    check_attention(cache, cu, q, got, 0.125, sample=40)
    assert (got[52:] == -7).all()


def test_calls_again_give_the_same_bits(api):
    cache = filled(api, "fp8", 16, 2, 128, [3000, 700])
    for new in ([1, 1], [200, 100]):
        cu = np.concatenate([[0], np.cumsum(new)])
        q = cache.r.standard_normal((int(cu[-1]), 8, 128)).astype(np.float16)
        first = attend(api, cache, cu, q, 0.1)
        for _ in range(3):
            assert np.array_equal(first, attend(api, cache, cu, q, 0.1))


@pytest.mark.parametrize("dtype,P,d", [("int8", 16, 64), ("fp8", 64, 128), ("int8", 128, 256), ("fp8", 128, 256)])
@pytest.mark.parametrize("behind", [False, True])
def test_sequences_without_rows_write_nothing(api, dtype, P, d, behind):
    """Idle sequences, of no rows or with all of theirs behind T, whose last page, partly filled, is a page that another sequence of the call
    appends to, loud enough to double its scale; and idle ones whose table names pages with scales that no write leaves. One
    wavefront a page and head, and four (128 x 256)."""
    H, writers = 2, 12
    old = [P // 2 + 1 + b % (P // 2 - 4) for b in range(writers)]
    cache = Cache(dtype, P, H, d, 3 * writers, 3 * writers, 2, seed=P + d)
    cache.grow(old + [0] * (2 * writers))
    cu = np.concatenate([[0], np.cumsum(cache.lengths)])
    write(api, cache, new_rows(cache.r, int(cu[-1]), H, d), cu)
    idle, odd = np.arange(writers, 2 * writers), np.arange(2 * writers, 3 * writers)
    cache.table[idle] = cache.table[:writers]
    cache.lengths[idle] = np.array(old) - np.arange(writers) % 3
    cache.table[odd, 0] = cache.free[:writers]
    cache.lengths[odd] = P // 2
    for x in (cache.ks, cache.vs):
        x[cache.table[odd, 0]] = np.array([-1.0, -0.0, np.inf, 1e-40], np.float32)[np.arange(writers) % 4, None]
    cache.upload()
    for new in (1, 2):
        cache.grow([new] * writers + [0] * (2 * writers))
        cu = np.concatenate([[0], np.cumsum([new] * writers + [2 if behind else 0] * (2 * writers))])
        kv = new_rows(cache.r, int(cu[-1]), H, d) * np.float16(8 ** new)
        write(api, cache, kv, cu, T=new * writers)
        cache.check()
        for which in ("ks", "vs"):
            assert np.array_equal(host(getattr(cache, "d" + which)).view(np.uint32), getattr(cache, which).view(np.uint32))


@pytest.mark.parametrize("dtype,P", [("int8", 16), ("fp8", 32)])
@pytest.mark.parametrize("what", [1e-40, np.nan, np.inf, -1.0, 0.0])
def test_scales_of_pages_that_no_row_sees(api, dtype, P, what):
    """Pages behind a sequence's end that the table names already, and page 0, which stands in for pages that are gone: whatever their
    scales are, subnormal numbers included, no row is touched by them."""
    H, heads, d = 2, 4, 64
    lens = [40, 70, 150, 1]
    cache = Cache(dtype, P, H, d, 40, len(lens), 16, seed=P)
    cache.free.remove(0)
    cache.grow(lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    write(api, cache, new_rows(cache.r, int(cu[-1]), H, d), cu)
    for b, n in enumerate(lens):
        behind = -(-n // P)
        cache.table[b, behind:behind + 3] = cache.free[3 * b:3 * b + 3]
    cache.table[2, 1:3] = -1
    unwritten = np.setdiff1d(np.arange(40), [cache.table[b, i] for b, n in enumerate(lens) for i in range(-(-n // P))])
    assert 0 in unwritten and cache.table[0, -(-40 // P)] in unwritten
    cache.ks[unwritten], cache.vs[unwritten] = what, what
    cache.upload()
    for new in ([2, 1, 4, 1], [20, 40, 30, 1]):
        cu = np.concatenate([[0], np.cumsum(new)])
        q = cache.r.standard_normal((int(cu[-1]), heads, d)).astype(np.float16)
        for window, max_length in ((0, 0), (0, 2), (30, 0)):
            got = attend(api, cache, cu, q, 0.125, window=window, max_length=max_length)
            check_attention(cache, cu, q, got, 0.125, window, sample=40)


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
@pytest.mark.parametrize("lengths,cu,T", [
    ([2 ** 31 - 1, 100, -5], [0, 2, 4, 6], 6), ([64, 64, 64], [3, 1, 6, 2], 6), ([64, 64, 64], [-7, 2, 2 ** 31 - 1, 5], 6),
    ([2 ** 31 - 1] * 3, [0, 20, 40, 60], 60), ([64, 2 ** 30, 33], [50, 10, 45, 60], 60), ([-2 ** 31, 70, 2 ** 31 - 1], [0, 2 ** 31 - 1, 1, 30], 60)])
def test_writes_of_no_sense_stay_in_their_pages(api, dtype, lengths, cu, T):
    """Lengths and rows that no cache has: pages that no table entry names, and what lies behind the pool and the scales, stay as they were."""
    import torch
    cache = filled(api, dtype, 16, 2, 64, [64, 64, 64], spare=5)
    cache.lengths = np.array(lengths, np.int32)
    cache.dlengths.copy_(dev(cache.lengths))
    pool = [cache.dk, cache.dv, cache.dks, cache.dvs]
    guarded = [torch.cat([x.flatten().view(torch.uint8), torch.full((4096,), 0x5A, dtype=torch.uint8, device="cuda")]) for x in pool]
    before = [host(x) for x in guarded]
    kv = new_rows(cache.r, T, 2, 64)
    c, keep = cache.described(np.array(cu), T=T, max_tokens=min(T, 40))
    c.k, c.v, c.k_scale, c.v_scale = (ptr(x) for x in guarded)
    t = dev(kv)
    s = dict(k_token_stride=256, k_head_stride=128, v_token_stride=256, v_head_stride=128)
    api.check(api.kv_cache_write(stream(), C.byref(capi.KvCacheWriteParams(cache=c, k=ptr(t), v=ptr(t) + 128, **s))))
    sync()
    others = np.setdiff1d(np.arange(cache.pages), cache.table)
    assert len(others) == 5
    for x, was, shape in zip(guarded, before, (cache.k.shape, cache.v.shape, cache.ks.shape, cache.vs.shape)):
        now = host(x)
        assert np.array_equal(now[-4096:], was[-4096:])
        pages = [y[:-4096].reshape(shape[0], -1)[others] for y in (now, was)]
        assert np.array_equal(*pages)
