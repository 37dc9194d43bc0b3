"""Attention in windows over packed FP16 sequences, against binary64. The tolerance is that of the attention over the cache
(cache_helpers.attention_reference), with scales of 1: the same products, sums and roundings."""
import ctypes as C

import numpy as np
import pytest

from cache_helpers import assert_within, attention_reference, visible_keys
from helpers import dev, dev_empty, host, ptr, rng, stream, sync
from tensorrt_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    return capi.api()


def params(q, k, v, out, dcu, B, longest, scale, left, right, sinks, T=None):
    p = capi.WindowAttentionParams(cu_seqlens=ptr(dcu), B=B, T=q.shape[0] if T is None else T, max_tokens=longest, q_heads=q.shape[1],
                                   kv_heads=k.shape[1], d=q.shape[2], scale=scale, left=left, right=right, sinks=sinks)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        setattr(p, name, ptr(t))
        setattr(p, name + "_token_stride", t.stride(0))
        setattr(p, name + "_head_stride", t.stride(1))
    return p


class Problem:
    def __init__(self, lens, heads, kv_heads, d, packed=False, seed=0):
        r = self.r = rng(seed)
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        T = int(self.cu[-1])
        shapes = [(T, heads, d), (T, kv_heads, d), (T, kv_heads, d)]
        self.q, self.k, self.v = (r.standard_normal(s).astype(np.float16) for s in shapes)
        self.packed = packed
        self.lens, self.scale = lens, float(np.float32(1 / np.sqrt(d)))

    def run(self, api, left, right, sinks, **more):
        if self.packed:  # [token][head][q|k|v][d]
            t = dev(np.stack([self.q, self.k, self.v], 2))
            q, k, v = t[:, :, 0], t[:, :, 1], t[:, :, 2]
        else:
            q, k, v = dev(self.q), dev(self.k), dev(self.v)
        T = len(self.q)
        out = dev_empty((T + 1,) + self.q.shape[1:], np.float16, fill=-7)
        dcu = dev(self.cu)
        longest = more.pop("longest", max(self.lens))
        p = params(q, k, v, out, dcu, len(self.lens), longest, self.scale, left, right, sinks, **more)
        api.check(api.window_attention(stream(), C.byref(p)))
        sync()
        got = host(out)
        assert (got[T:] == -7).all()
        return got[:T]

    def check(self, got, left, right, sinks, sample=None, heads=None):
        group = self.q.shape[1] // self.k.shape[1]
        for lo, hi in zip(self.cu[:-1], self.cu[1:]):
            n = int(hi - lo)
            rows = np.arange(n)
            if sample and n > sample:
                rows = np.unique(np.concatenate([[0, n - 1], self.r.integers(0, n, sample)]))
            ones = np.ones(n)
            for i in rows:
                ok = visible_keys(i, n, None if left < 0 else left, None if right < 0 else right, sinks)
                for h in heads or range(self.q.shape[1]):
                    want, tol = attention_reference(self.q[lo + i, h], self.k[lo:hi, h // group], ones, self.v[lo:hi, h // group], ones, ok, self.scale)
                    assert_within(got[lo + i, h], want, tol, f"row {lo + i} head {h}")


CASES = [([1], 1, 1, 64), ([2, 1, 3], 2, 2, 8), ([63, 64, 65], 2, 1, 64), ([127, 128, 129, 5], 3, 3, 64), ([200, 0, 33], 4, 2, 128),
         ([90], 7, 1, 80), ([150, 31], 2, 2, 96), ([77, 130], 2, 1, 256), ([140], 4, 4, 72), ([66], 1, 1, 200), ([300, 7], 16, 4, 32)]


@pytest.mark.parametrize("lens,heads,kv_heads,d", CASES)
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (-1, 0, 0), (0, 0, 0), (10, 10, 0), (64, 0, 3), (5, 40, 70), (0, -1, 2), (-1, 63, 0)])
def test_window(api, lens, heads, kv_heads, d, left, right, sinks):
    p = Problem(lens, heads, kv_heads, d, packed=heads == kv_heads, seed=d)
    p.check(p.run(api, left, right, sinks), left, right, sinks, sample=12)


@pytest.mark.parametrize("left,right,sinks", [(1000, 0, 4), (200, 200, 0), (-1, -1, 0), (70, 0, 300)])
def test_long_sequences(api, left, right, sinks):
    p = Problem([3001, 900], 4, 2, 128, seed=9)
    p.check(p.run(api, left, right, sinks), left, right, sinks, sample=10)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_what_is_not_seen_does_not_matter(api, what, d):
    """Infinities and NaNs in keys and values of some tokens: rows that do not see them are as if they were not there."""
    p = Problem([150, 90], 4, 2, d, seed=11)
    spots = {3: "k", 40: "v", 149: "v", 150 + 64: "v", 150 + 20: "k"}
    for t, name in spots.items():
        getattr(p, name)[t, 0, 5] = what
    for left, right, sinks in ((10, 10, 0), (20, 0, 2), (0, 0, 0)):
        got = p.run(api, left, right, sinks).astype(np.float64)
        group = 2
        for lo, hi in zip(p.cu[:-1], p.cu[1:]):
            n = int(hi - lo)
            for i in range(n):
                ok = visible_keys(i, n, left, right, sinks)
                for h in range(4):
                    k, v = p.k[lo:hi, h // group], p.v[lo:hi, h // group]
                    if np.isfinite(k[ok]).all() and np.isfinite(v[ok]).all():
                        want, tol = attention_reference(p.q[lo + i, h], np.where(ok[:, None], k, 0), np.ones(n), np.where(ok[:, None], v, 0), np.ones(n), ok, p.scale)
                        assert_within(got[lo + i, h], want, tol, f"row {lo + i} head {h}")
                    elif np.isfinite(k[ok]).all():  # a value that is seen: its element is it, or no number; the others are sound
                        v = v.astype(np.float64)
                        s = (k[ok].astype(np.float64) @ p.q[lo + i, h].astype(np.float64)) * p.scale
                        w = np.exp(s - s.max())
                        with np.errstate(invalid="ignore"):
                            want = (w / w.sum()) @ v[ok]
                        odd = ~np.isfinite(want)
                        assert np.array_equal(np.isnan(got[lo + i, h][odd]), np.isnan(want[odd]))
                        assert np.allclose(got[lo + i, h][~odd], want[~odd], atol=4e-3, rtol=4e-3)


def test_rows_left_out_stay(api):
    p = Problem([100, 40, 9], 2, 2, 64, seed=4)
    want = p.run(api, 10, 10, 0)
    got = p.run(api, 10, 10, 0, longest=30)
    assert (got[30:100] == -7).all() and (got[130:140] == -7).all()
    short = Problem([30, 30, 9], 2, 2, 64)
    for name in "qkv":
        x = getattr(p, name)
        setattr(short, name, np.concatenate([x[:30], x[100:130], x[140:]]))
    assert np.array_equal(np.concatenate([got[:30], got[100:130], got[140:]]), short.run(api, 10, 10, 0))
    got = p.run(api, 10, 10, 0, T=120)
    assert np.array_equal(got[:100], want[:100]) and (got[120:] == -7).all()


def test_all_of_a_scale(api):
    """Scores of any size, a scale of 0 too."""
    for scale in (0.0, 1e-30, 30.0):
        p = Problem([70, 5], 2, 1, 64, seed=6)
        p.scale = float(np.float32(scale))
        p.check(p.run(api, 20, 3, 1), 20, 3, 1)


def test_agrees_with_the_fused_attention(api):
    """Windows that are as long as the sequences: what the fused attention computes, to the roundings of both."""
    from helpers import assert_fp_close, half2_bits
    p = Problem([100, 384, 17], 4, 4, 64, packed=True, seed=8)
    got = p.run(api, -1, -1, 0)
    t = dev(np.stack([p.q, p.k, p.v], 2))
    out, dcu = dev_empty(p.q.shape, np.float16, fill=-7), dev(p.cu)
    f = capi.FmhaParams(qkv_ptr=ptr(t), o_ptr=ptr(out), qkv_stride_in_bytes=6 * 256, o_stride_in_bytes=512, b=3, h=4, s=384, d=64,
                        scale_bmm1=half2_bits(0.125), scale_softmax=half2_bits(1.0), scale_bmm2=half2_bits(1.0), cu_seqlens=ptr(dcu))
    api.check(api.fused_mha_run(stream(), 1, C.byref(f)))
    sync()
    assert_fp_close(got, host(out), what="the two attentions")


def test_captured(api):
    """A graph follows the lengths, between eager calls of another problem; rows behind the last sequence stay."""
    import torch
    p, other = (Problem([150, 90, 40], 4, 2, 96, seed=s) for s in (1, 2))
    T = len(p.q)
    q, k, v, out, dcu = dev(p.q), dev(p.k), dev(p.v), dev_empty(p.q.shape, np.float16, fill=-7), dev(p.cu)
    a = params(q, k, v, out, dcu, 3, T, p.scale, 20, 5, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.check(api.window_attention(stream(), C.byref(a)))
    for lens in ([150, 90, 40], [1, 0, 200], [100, 100, 80], [0, 0, 0]):
        p.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        dcu.copy_(dev(p.cu))
        out.fill_(-7)
        graph.replay()
        sync()
        got = host(out)
        assert (got[p.cu[-1]:] == -7).all()
        p.check(got, 20, 5, 3, sample=10)
        other.check(other.run(api, 20, 5, 3), 20, 5, 3, sample=5)


def test_two_streams(api):
    import torch
    problems = [Problem([700, 300], 4, 4, 64, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in problems]
    held = []
    for p in problems:
        q, k, v, out, dcu = dev(p.q), dev(p.k), dev(p.v), dev_empty(p.q.shape, np.float16, fill=-7), dev(p.cu)
        held.append((q, k, v, out, dcu, params(q, k, v, out, dcu, 2, 700, p.scale, 100, 100, 0)))
    sync()
    for _ in range(3):
        for h, s in zip(held, streams):
            api.check(api.window_attention(s.cuda_stream, C.byref(h[5])))
    sync()
    for p, h in zip(problems, held):
        p.check(host(h[3]), 100, 100, 0, sample=20)


@pytest.mark.parametrize("strides", [(1 << 25) + 64, 1 << 20])
def test_far_rows(api, strides):
    """Rows so far apart that a chunk passes 32-bit offsets, or does not."""
    import torch
    d, n = 64, 70
    r = rng(3)
    x = r.standard_normal((3, n, 1, d)).astype(np.float16)
    far = torch.empty((n * strides,), dtype=torch.float16, device="cuda")
    rows = [torch.as_strided(far, (n, 1, d), (strides, d, 1), i * d) for i in range(3)]
    for t, y in zip(rows, x):
        t.copy_(dev(y))
    out, dcu = dev_empty((n, 1, d), np.float16, fill=-7), dev(np.array([0, n], np.int32))
    p = Problem([n], 1, 1, d)
    p.q, p.k, p.v = x
    api.check(api.window_attention(stream(), C.byref(params(*rows, out, dcu, 1, n, p.scale, 9, 9, 2))))
    sync()
    p.check(host(out), 9, 9, 2)


@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_infinities_that_are_seen(api, what, d):
    """A value that a row sees and that is infinite: its element is that infinity, of its sign, in every row that sees it, and no other
    element is touched; two of opposite signs are no number."""
    p = Problem([150, 90], 4, 2, d, seed=12)
    for t, h, e, x in ((30, 0, 5, what), (64, 1, 0, what), (150 + 70, 0, d - 1, what), (100, 0, 7, what), (103, 0, 7, -what)):
        p.v[t, h, e] = x
    for left, right, sinks in ((10, 10, 0), (20, 0, 40), (-1, -1, 0)):
        got = p.run(api, left, right, sinks).astype(np.float64)
        for lo, hi in zip(p.cu[:-1], p.cu[1:]):
            n = int(hi - lo)
            for i in range(n):
                ok = visible_keys(i, n, None if left < 0 else left, None if right < 0 else right, sinks)
                for h in range(4):
                    k, v = p.k[lo:hi, h // 2], p.v[lo:hi, h // 2].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        odd = np.where(ok[:, None] & ~np.isfinite(v), v, 0).sum(0)
                    sound = odd == 0
                    want, tol = attention_reference(p.q[lo + i, h], k, np.ones(n), np.where(np.isfinite(v), v, 0), np.ones(n), ok, p.scale)
                    assert np.array_equal(got[lo + i, h][~sound], odd[~sound], equal_nan=True), (lo + i, h)
                    assert_within(got[lo + i, h][sound], want[sound], tol[sound], f"row {lo + i} head {h}")
