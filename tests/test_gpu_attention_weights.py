"""Weights far below the largest one: a loud first token that the rows look at for want of anything else, with a value of zero, and
thousands of quiet keys whose weights only add up to something. Attention over the cache and in windows, against binary64. And scales of the
scores near the largest binary32, and scores of minus infinity."""
import numpy as np
import pytest

from cache_helpers import Cache, assert_within, attention_reference, round_codes, values, visible_keys
from tensorrt_amd import capi
from test_gpu_kv_cache import attend, check_attention, filled
from test_gpu_window_attention import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    return capi.api()


N, D = 8192, 64
# powers of 2 between the first token and the others, a row each
DEPTHS = np.array([8.0, 12.03, 14.6, 16.03, 18.7, 20.03, 21.97, 23.4, 24.03, 25.6, 26.0, 27.3])


def expected(depths, v):
    """(result, tolerance) of rows whose first key has the weight 1 and a value of zero, the others 2^-depth and the values v [keys][d].

    Tolerance. A score is a product of one element (exact), scaled: within 8 * 2^-24 of itself, of at most 32 powers of 2, so a weight is
    off by ln(2) * 8 * 2^-24 * 32 = 2^-16.5 of itself, all of a row alike, and its exponential by 2^-22. The largest weight is held at 2^7 or more, so
    a weight that is rounded to binary16 is off by 2^-11 of itself, or by 2^-25 / 2^7 = 2^-32 of the largest where that is more. The
    sums add 2^-23 for each of the terms, and the result is rounded to binary16."""
    w = 2.0 ** -depths[:, None]
    total = 1 + w * len(v)
    size = w * np.abs(v).sum(0) / total
    want = w * v.sum(0) / total
    each = 2.0 ** -16 + 2.0 ** -11 + 2 * (len(v) + 16) * 2.0 ** -23
    return want, size * each + 2.0 ** -32 * np.abs(v).sum(0) / total + 2.0 ** -11 * np.abs(want) + 2.0 ** -25


@pytest.mark.parametrize("dtype", ["int8", "fp8"])
@pytest.mark.parametrize("rows", [1, 12, 40])
@pytest.mark.parametrize("max_length", [0, 64])
def test_over_the_cache(api, dtype, rows, max_length):
    """A row a query head of one token each: one, a few, and tiles of 40."""
    P = 64
    depths = np.resize(DEPTHS[::-1], rows)
    cache = Cache(dtype, P, 1, D, N // P + 1, 1, N // P, seed=rows, junk=False)
    cache.grow([N])
    cache.ks[:], cache.vs[:] = 1.0, 2.0 ** -6
    v = round_codes(cache.r.uniform(20, 60, (N, D)).astype(np.float32), dtype)
    v[0] = 0
    k = np.zeros((N, D), np.uint8)
    k[0, 0] = round_codes(np.float32([32.0]), dtype)[0]
    page = cache.table[0]
    cache.k[page, 0] = k.reshape(-1, P, D)
    cache.v[page, 0] = v.reshape(-1, P, D).transpose(0, 2, 1)
    cache.upload()
    q = np.zeros((1, rows, D), np.float16)
    scale = np.float32(1 / 32)
    q[0, :, 0] = depths / np.log2(np.e)
    depths = q[0, :, 0].astype(np.float64) * np.log2(np.e)
    want, tol = expected(depths, values(v, dtype).astype(np.float64)[1:] * 2.0 ** -6)
    got = attend(api, cache, np.array([0, 1]), q, scale, max_length=max_length)
    assert_within(got[0], want, tol)


@pytest.mark.parametrize("heads", [1, 3])
def test_in_windows(api, heads):
    """The last rows of a sequence, which see all of it."""
    p = Problem([N], heads, 1, D, seed=heads)
    p.q[:], p.k[:], p.scale = 0, 0, 1.0 / 32
    p.k[0, 0, 0] = 32
    p.v[:] = p.r.uniform(0.3, 0.9, p.v.shape).astype(np.float16)
    p.v[0] = 0
    p.q[-len(DEPTHS):, :, 0] = (DEPTHS / np.log2(np.e))[:, None]
    depths = p.q[-len(DEPTHS):, 0, 0].astype(np.float64) * np.log2(np.e)
    got = p.run(api, -1, -1, 0)
    want, tol = expected(depths, p.v[1:, 0].astype(np.float64))
    for h in range(heads):
        assert_within(got[-len(DEPTHS):, h], want, tol, f"head {h}")


@pytest.mark.parametrize("scale", [1e37, 3.4e38])
def test_scales_near_the_largest(api, scale):
    """Scores of zero stay zero whatever they are scaled by, times a page's scale too: rows whose query is zero weigh all keys alike."""
    cache = filled(api, "int8", 16, 1, D, [100, 7])
    cache.ks[cache.table[0, 2:4]], cache.ks[cache.table[0, 4]] = 100, 0
    cache.upload()
    for new in ([2, 2], [40, 7]):
        cu = np.concatenate([[0], np.cumsum(new)])
        q = np.zeros((int(cu[-1]), 2, D), np.float16)
        check_attention(cache, cu, q, attend(api, cache, cu, q, scale), np.float32(1))
    p = Problem([70, 5], 2, 1, D, seed=6)
    p.q[:], p.scale = 0, scale
    got = p.run(api, 20, 3, 1)
    p.scale = 1.0
    p.check(got, 20, 3, 1)


def test_scores_of_minus_infinity(api):
    """They weigh nothing: keys that a window sees are as if it did not, and a row that has no other is zeros."""
    p = Problem([150, 20], 4, 2, D, seed=3)
    p.q[:, :, 5] = np.abs(p.q[:, :, 5]) + np.float16(0.5)
    gone = np.zeros(170, bool)
    gone[[3, 40, 41, 64, 149, 155]] = True
    gone[90:120] = True
    p.k[gone, :, 5] = -np.inf
    got = p.run(api, 10, 10, 0)
    assert (got[100:110] == 0).all()
    for lo, hi in zip(p.cu[:-1], p.cu[1:]):
        n = int(hi - lo)
        k = np.where(gone[lo:hi, None, None], 0, p.k[lo:hi])
        for i in range(n):
            ok = visible_keys(i, n, 10, 10, 0) & ~gone[lo:hi]
            for h in range(4):
                want, tol = attention_reference(p.q[lo + i, h], k[:, h // 2], np.ones(n), p.v[lo:hi, h // 2], np.ones(n), ok, p.scale)
                assert_within(got[lo + i, h], want, tol, f"row {lo + i} head {h}")
    cache = filled(api, "int8", 16, 1, D, [100])
    cache.k[:] = 5
    cache.upload()
    for rows in (1, 40):
        q = np.zeros((rows, 2, D), np.float16)
        q[:, 1, 5] = -np.inf
        q[:, 1] += 1
        got = attend(api, cache, np.array([0, rows]), q, 0.125)
        assert (got[:, 1] == 0).all()
        check_attention(cache, np.array([0, rows]), q[:, :1], got[:, :1], 0.125)
