"""Quantisation with a scale for each token and the INT8 linear layers on it, against the definitions in binary64.

Tolerances. The quantised values are exact, and so is the scale (one binary32 division). A layer's result is formed in
binary32: the accumulator's conversion, its products with the two scales and the addition of the bias round at most
four times, each to 2^-24 of the product p or of the sum (which is no more than |p| + |bias|); GELU's slope is at most
1.13, and its polynomial is within 8.5e-5 of the value where that is a normal binary16 and 5.2e-9 below
(test_gelu_polynomial evaluates it). One rounding to binary16 follows: half a step, 2^-11 of the value or 2^-25,
whichever is more."""
import ctypes as C

import numpy as np
import pytest
from scipy.special import ndtr

from helpers import dev, dev_empty, host, ptr, rng, stream, sync
from tensorrt_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    return capi.api()


def activations(r, T, K):
    x = r.standard_normal((T, K)) * np.exp(0.5 * r.standard_normal((T, 1)))
    x[:, r.random(K) < 0.02] *= 10
    return x.astype(np.float16)


def quantised(x):
    """(values, scales) of the definition; rows that are not finite become zeros with scale NaN."""
    wide = x.astype(np.float64)
    amax = np.abs(wide).max(1)
    finite = np.isfinite(amax)
    safe = np.where(finite & (amax > 0), amax, 1.0)
    q = np.rint(np.where(finite[:, None], wide, 0.0) * 127 / safe[:, None]).astype(np.int8)
    return q, np.where(finite, amax.astype(np.float32) / np.float32(127), np.float32(np.nan))


def run_quantise(api, x, view=None, s=None):
    T, K = x.shape
    d = dev(x) if view is None else view
    q, scales = dev_empty((T + 1, K), np.int8, fill=77), dev_empty((T + 1,), np.float32, fill=-7)
    api.check(api.quantize_fp16_per_token(s or stream(), T, K, ptr(d), d.stride(0), ptr(q), ptr(scales)))
    sync()
    q, scales = host(q), host(scales)
    assert (q[T] == 77).all() and scales[T] == -7, "something behind the last token was written"
    return q[:T], scales[:T]


def reference(q, scales, w, channel, bias, gelu):
    """(result, tolerance)."""
    p = (q.astype(np.float64) @ w.astype(np.float64).T) * scales.astype(np.float64)[:, None] * channel.astype(np.float64)
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(np.float64)
    y = p + b
    off = 4 * 2.0 ** -24 * (np.abs(p) + np.abs(b))
    if gelu:
        y, off = y * ndtr(y), 1.13 * off
        off += 8.5e-5 * np.abs(y) + 5.2e-9
    return y, off + np.maximum(2.0 ** -11 * (np.abs(y) + off), 2.0 ** -25)


def assert_within(got, want, tol, what=""):
    got = got.astype(np.float64)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0]}: "
                           f"{got[bad][0]} for {want[bad][0]} +- {tol[bad][0]}")


def weights(r, N, K):
    w = r.integers(-127, 128, (N, K)).astype(np.int8)
    channel = (r.uniform(0.5, 1.5, N) / (73 * np.sqrt(K))).astype(np.float32)
    return w, channel, (0.3 * r.standard_normal(N)).astype(np.float32)


def params(cls, T, K, N, gelu, w, channel, bias, out, **more):
    p = cls(w=ptr(w), channel_scale=ptr(channel), bias=ptr(bias), out=ptr(out), T=T, K=K, N=N,
            epilogue=capi.LINEAR_GELU if gelu else capi.LINEAR_AFFINE)
    for k, v in more.items():
        setattr(p, k, v)
    return p


class Layer:
    """Device operands of one layer; the output has a row behind its last one that must stay as it is."""

    def __init__(self, api, T, K, N, gelu=False, bias=True, seed=0, x=None):
        r = rng([T, K, N, seed])
        self.api, self.sizes, self.gelu = api, (T, K, N), gelu
        self.x = activations(r, T, K) if x is None else x
        self.w, self.channel, b = weights(r, N, K)
        self.bias = b if bias else None
        self.dx, self.dw, self.dc = dev(self.x), dev(self.w), dev(self.channel)
        self.db = dev(self.bias) if bias else None

    def want(self):
        q, scales = quantised(self.x)
        return reference(q, scales, self.w, self.channel, self.bias, self.gelu)

    def out(self):
        return dev_empty((self.sizes[0] + 1, self.sizes[2]), np.float16, fill=-7)

    def token(self, out, s=None):
        q, scales = quantised(self.x)
        self.dq, self.ds = dev(q), dev(scales)
        p = params(capi.Int8TokenLinearParams, *self.sizes, self.gelu, self.dw, self.dc, self.db, out, a=ptr(self.dq),
                   token_scale=ptr(self.ds))
        self.api.check(self.api.int8_token_linear(s or stream(), C.byref(p)))

    def workspace(self):
        return dev_empty((self.api.int8_dynamic_linear_workspace_size(*self.sizes),), np.uint8, fill=0xAB)

    def dynamic(self, out, ws, s=None, view=None):
        x = self.dx if view is None else view
        p = params(capi.Int8DynamicLinearParams, *self.sizes, self.gelu, self.dw, self.dc, self.db, out, a=ptr(x),
                   a_stride=x.stride(0), workspace=ptr(ws), workspace_bytes=ws.numel())
        self.api.check(self.api.int8_dynamic_linear(s or stream(), C.byref(p)))


def bits(t):
    return host(t).view(np.uint16)


# ---- the quantiser -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("C_", [32, 64, 96, 256, 480, 512, 544, 768, 1024, 1056, 2048, 2080, 4096, 4128, 8192, 8224, 16384, 33024])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 37])
def test_quantiser(api, T, C_):
    x = activations(rng(T * 100000 + C_), T, C_)
    got, want = run_quantise(api, x), quantised(x)
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1])


@pytest.mark.parametrize("T,C_", [(4099, 96), (1000, 1024), (777, 4096), (20011, 64)])
def test_quantiser_many_tokens(api, T, C_):
    x = activations(rng(T + C_), T, C_)
    got, want = run_quantise(api, x), quantised(x)
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1])


def test_quantiser_ties_and_every_pair_of_maximum_and_value(api):
    """Half-way quotients are those of the definition: for many maxima, every finite binary16 value up to the maximum."""
    r = rng(5)
    values = np.arange(0x7c00, dtype=np.uint16).view(np.float16)
    maxima = np.concatenate([values[r.integers(1, 0x7c00, 60)], values[[1, 2, 3, 1023, 1024, 0x7bff]],
                             np.float16([127, 254, 127 / 1024, 1, 0.5, 63.5, 95.25])])
    for top in maxima:
        x = values[values <= top]
        x = np.concatenate([x, -x, np.zeros(-2 * len(x) % 32, np.float16)])
        x = np.stack([x, x[::-1]])
        got, want = run_quantise(api, x), quantised(x)
        assert np.array_equal(got[0], want[0]), top
        assert np.array_equal(got[1], want[1]), top


@pytest.mark.parametrize("C_", [64, 768, 4096, 20000])
def test_quantiser_zeros_and_values_that_are_not_finite(api, C_):
    x = activations(rng(C_), 11, C_)
    x[1] = 0
    x[3, C_ - 1] = np.nan
    x[4, 0] = np.inf
    x[6, C_ // 2] = -np.inf
    x[7] = -0.0
    x[8] = 0
    x[8, 5] = 2.0 ** -24
    x[9] = np.nan
    x[10] = 65504
    q, s = run_quantise(api, x)
    wq, ws = quantised(x)
    assert np.array_equal(q, wq)
    assert np.array_equal(s.view(np.uint32)[np.isfinite(ws)], ws.view(np.uint32)[np.isfinite(ws)])
    assert np.isnan(s[[3, 4, 6, 9]]).all() and s[1] == s[7] == 0


def test_quantiser_of_strided_rows(api):
    """Rows that lie between others: the middle of a wider tensor, and every second row."""
    wide = activations(rng(3), 54, 1600)
    d = dev(wide)
    for view, x in ((d[:, 512:512 + 1024], wide[:, 512:512 + 1024]), (d[::2, 8:8 + 96], wide[::2, 8:8 + 96])):
        got, want = run_quantise(api, np.ascontiguousarray(x), view), quantised(x)
        assert np.array_equal(got[0], want[0])
        assert np.array_equal(got[1], want[1])


def test_quantiser_beyond_32_bits(api):
    """More than 2^32 bytes of input and 2^31 of output."""
    import torch
    T, C_ = 70001, 32768
    x = torch.zeros((T, C_), dtype=torch.float16, device="cuda")
    tail = activations(rng(9), 3, C_)
    x[-3:] = dev(tail)
    q = torch.full((T, C_), 77, dtype=torch.int8, device="cuda")
    scales = torch.empty((T,), dtype=torch.float32, device="cuda")
    api.check(api.quantize_fp16_per_token(stream(), T, C_, ptr(x), C_, ptr(q), ptr(scales)))
    sync()
    want = quantised(tail)
    assert np.array_equal(host(q[-3:]), want[0]) and np.array_equal(host(scales[-3:]), want[1])
    assert not q[:-3].any() and not scales[:-3].any()


# ---- the layers --------------------------------------------------------------------------------------------------

SHAPES = [(1, 64, 32), (1, 1024, 1024), (2, 768, 2304), (3, 4096, 1024), (4, 128, 4096), (5, 192, 96),
          (7, 1088, 544), (8, 1024, 4096), (9, 512, 512), (16, 4096, 1024), (17, 64, 4128), (31, 128, 64),
          (33, 320, 160), (40, 4096, 1024), (64, 768, 768), (100, 1024, 288), (129, 192, 32), (257, 1024, 1024),
          (777, 768, 2304), (1000, 4096, 1024), (2049, 384, 1536), (4099, 1024, 4096), (5003, 960, 4096),
          (2600, 832, 2304)]


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("gelu,bias", [(False, True), (False, False), (True, True), (True, False)])
def test_layers(api, T, K, N, gelu, bias):
    layer = Layer(api, T, K, N, gelu, bias)
    want, tol = layer.want()
    one, two = layer.out(), layer.out()
    layer.token(one)
    layer.dynamic(two, layer.workspace())
    sync()
    assert_within(host(one)[:T], want, tol, f"token {T} {K} {N}")
    assert (host(one)[T] == -7).all() and (host(two)[T] == -7).all(), "something behind the last token was written"
    assert np.array_equal(bits(one), bits(two)), "the two entry points differ"


@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 47, 64, 65])
@pytest.mark.parametrize("K", [64, 128, 192, 576, 960, 1024, 1088, 1152, 2048, 2112, 4032, 4096, 4160, 8192])
@pytest.mark.parametrize("N", [32, 224])
def test_few_tokens(api, T, K, N):
    """Both sides of every length up to which few tokens go in one launch."""
    layer = Layer(api, T, K, N, gelu=N == 32, bias=K % 128 == 0)
    want, tol = layer.want()
    one, two, ws = layer.out(), layer.out(), layer.workspace()
    layer.token(one)
    layer.dynamic(two, ws)
    sync()
    assert_within(host(one)[:T], want, tol)
    assert np.array_equal(bits(one), bits(two))


def test_few_tokens_of_many_channels(api):
    for T, N in ((1, 8160), (1, 8192), (3, 8224), (16, 16384), (5, 30528)):
        layer = Layer(api, T, 128, N)
        want, tol = layer.want()
        out = layer.out()
        layer.dynamic(out, layer.workspace())
        sync()
        assert_within(host(out)[:T], want, tol, f"{T} {N}")
        assert (host(out)[T] == -7).all()


PLANS = range(1, 15)


@pytest.mark.parametrize("T,K,N", [(300, 256, 288), (300, 192, 320), (130, 192, 160), (61, 128, 96), (520, 64, 544)])
@pytest.mark.parametrize("gelu", [False, True])
def test_every_plan_gives_the_same_bits(api, T, K, N, gelu):
    layer = Layer(api, T, K, N, gelu)
    want, tol = layer.want()
    first = layer.out()
    layer.token(first)
    sync()
    assert_within(host(first)[:T], want, tol)
    try:
        for plan in PLANS:
            api.check(api.test_set_tuning(b"TRTAMD_LINEAR_PLAN", plan))
            out = layer.out()
            layer.token(out)
            sync()
            assert np.array_equal(bits(out), bits(first)), f"plan {plan}"
        api.check(api.test_reset_tuning(b"TRTAMD_LINEAR_PLAN"))
        for switch in (b"TRTAMD_LINEAR_DIRECT", b"TRTAMD_LINEAR_PERSISTENT"):
            api.check(api.test_set_tuning(switch, 0))
            out = layer.out()
            layer.token(out)
            sync()
            assert np.array_equal(bits(out), bits(first)), switch
            api.check(api.test_reset_tuning(switch))
    finally:
        for switch in (b"TRTAMD_LINEAR_PLAN", b"TRTAMD_LINEAR_DIRECT", b"TRTAMD_LINEAR_PERSISTENT"):
            api.test_reset_tuning(switch)


def test_choices_of_other_layers_are_kept_apart(api):
    """Plans are remembered by sizes, and token-scaled layers have some that the other INT8 layers lack: the two in turn at the same sizes."""
    T, K, N = 5003, 960, 1056
    layer = Layer(api, T, K, N, bias=False)
    want, tol = layer.want()
    q, scales = quantised(layer.x)
    dq, ones, zeros = dev(q), dev(np.full(N, 2.0 ** -13, np.float32)), dev(np.zeros(N, np.float32))
    first = None
    for _ in range(2):
        out, out8 = layer.out(), dev_empty((T, N), np.int8, fill=99)
        layer.token(out)
        p = capi.Int8LinearParams(a=ptr(dq), w=ptr(layer.dw), alpha=ptr(ones), beta=ptr(zeros), out=ptr(out8), T=T, K=K, N=N)
        api.check(api.int8_linear(stream(), C.byref(p)))
        sync()
        assert_within(host(out)[:T], want, tol)
        acc = q.astype(np.float64) @ layer.w.astype(np.float64).T
        assert np.array_equal(host(out8), np.clip(np.rint(acc * 2.0 ** -13), -128, 127))
        assert first is None or np.array_equal(first, bits(out))
        first = bits(out)


@pytest.mark.parametrize("T,K,N", [(6, 1024, 1024), (70, 256, 96), (700, 1024, 1024)])
@pytest.mark.parametrize("gelu", [False, True])
def test_tokens_that_are_not_finite_stay_by_themselves(api, T, K, N, gelu):
    x = activations(rng(T), T, K)
    x[1, 3], x[T - 1, K - 1], x[2] = np.nan, -np.inf, 0
    layer = Layer(api, T, K, N, gelu, x=x)
    want, tol = layer.want()
    one, two = layer.out(), layer.out()
    layer.token(one)
    layer.dynamic(two, layer.workspace())
    sync()
    for out in (host(one)[:T], host(two)[:T]):
        assert np.isnan(out[[1, T - 1]]).all()
        rows = [t for t in range(T) if t not in (1, T - 1)]
        assert_within(out[rows], want[rows], tol[rows])


@pytest.mark.parametrize("T,K,N", [(33333, 64, 1056), (33000, 128, 1024), (9001, 192, 4128)])
@pytest.mark.parametrize("gelu", [False, True])
def test_results_past_the_cache(api, T, K, N, gelu):
    """Results of more than 64 MiB, in whole tiles and with ends in either direction."""
    layer = Layer(api, T, K, N, gelu)
    want, tol = layer.want()
    out = layer.out()
    layer.dynamic(out, layer.workspace())
    sync()
    assert_within(host(out)[:T], want, tol)
    assert (host(out)[T] == -7).all()


def test_large_accumulators(api):
    """Sums beyond 2^24, which a binary32 no longer holds exactly, and the largest in either direction."""
    T, K, N = 3, 8192, 64
    x = np.full((T, K), 3, np.float16)
    x[1] = -3
    x[2, ::2] = -1
    layer = Layer(api, T, K, N, x=x)
    layer.w = np.full((N, K), 127, np.int8)
    layer.w[1::2] = -127
    layer.w[5, :77] = 1
    layer.channel = np.full(N, 2e-5, np.float32)
    layer.dw, layer.dc = dev(layer.w), dev(layer.channel)
    want, tol = layer.want()
    out = layer.out()
    layer.dynamic(out, layer.workspace())
    sync()
    assert_within(host(out)[:T], want, tol)


def test_results_beyond_binary16_are_infinities(api):
    layer = Layer(api, 4, 128, 64)
    layer.channel = np.full(64, 1e4, np.float32)
    layer.dc = dev(layer.channel)
    want, _ = layer.want()
    out = layer.out()
    layer.dynamic(out, layer.workspace())
    sync()
    got = host(out)[:4]
    large = np.abs(want) > 70000
    assert large.any() and np.array_equal(got[large], np.sign(want[large]) * np.inf)


@pytest.mark.parametrize("T,K,N", [(1, 1024, 512), (90, 256, 288), (1500, 512, 256)])
def test_strided_tokens(api, T, K, N):
    import torch
    layer = Layer(api, T, K, N)
    wide = torch.full((T, 2 * K + 8), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 8:8 + K] = layer.dx
    one, two = layer.out(), layer.out()
    layer.dynamic(one, layer.workspace())
    layer.dynamic(two, layer.workspace(), view=wide[:, 8:8 + K])
    sync()
    assert np.array_equal(bits(one), bits(two))


@pytest.mark.parametrize("T,K,N", [(33, 1024, 2048), (3, 768, 512)])
def test_a_token_does_not_depend_on_its_neighbours(api, T, K, N):
    """Each token by itself, through the kernels of single tokens, gives the bits it has in the batch."""
    layer = Layer(api, T, K, N, gelu=True)
    out = layer.out()
    layer.dynamic(out, layer.workspace())
    for t in (0, 1, T - 1):
        single = Layer(api, 1, K, N, gelu=True, x=layer.x[t:t + 1])
        single.w, single.dw, single.dc, single.db = layer.w, layer.dw, layer.dc, layer.db
        alone = single.out()
        single.dynamic(alone, single.workspace())
        sync()
        assert np.array_equal(bits(alone)[0], bits(out)[t]), t


def test_two_calls_at_once_on_streams_of_their_own(api):
    import torch
    layers = [Layer(api, 600, 1024, 1024, seed=1), Layer(api, 2, 2048, 1024, gelu=True, seed=2)]
    want = [l.out() for l in layers]
    for l, o in zip(layers, want):
        l.dynamic(o, l.workspace())
    sync()
    streams, outs, spaces = [torch.cuda.Stream() for _ in layers], [l.out() for l in layers], [l.workspace() for l in layers]
    sync()
    for _ in range(10):
        for l, o, ws, s in zip(layers, outs, spaces, streams):
            l.dynamic(o, ws, s.cuda_stream)
    sync()
    for o, w in zip(outs, want):
        assert np.array_equal(bits(o), bits(w))


@pytest.mark.parametrize("T,K,N", [(1, 1024, 1024), (12, 1024, 1024), (500, 768, 768)])
def test_captured_and_replayed(api, T, K, N):
    """A captured call follows what its input holds at each replay, with eager calls on the same operands between the replays."""
    import torch
    layer = Layer(api, T, K, N, gelu=True)
    out, eager, ws, other = layer.out(), layer.out(), layer.workspace(), layer.workspace()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    sync()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer.dynamic(out, ws, side.cuda_stream)
    for replay in range(3):
        layer.x = activations(rng(replay + 50), T, K)
        layer.dx.copy_(dev(layer.x))
        out.fill_(-7)
        layer.dynamic(eager, other)
        graph.replay()
        sync()
        assert np.array_equal(bits(out), bits(eager)), replay
        want, tol = layer.want()
        assert_within(host(out)[:T], want, tol)
    del graph


@pytest.mark.parametrize("T,K,N", [(1, 12352, 96), (33, 16384, 64), (300, 20480, 288), (70, 33344, 160), (2, 131008, 32)])
def test_long_rows(api, T, K, N):
    layer = Layer(api, T, K, N)
    want, tol = layer.want()
    one, two = layer.out(), layer.out()
    layer.token(one)
    layer.dynamic(two, layer.workspace())
    sync()
    assert_within(host(one)[:T], want, tol)
    assert np.array_equal(bits(one), bits(two))


@pytest.mark.parametrize("T", [1, 40, 300])
def test_the_largest_sums(api, T):
    """Rows of the greatest length whose values and weights are all at the ends of their range: sums up to 2146435072 of the 2147483647
    that INT32 holds."""
    K, N = 131008, 64
    x = np.full((T, K), 5, np.float16)
    x[1::2] = -5
    layer = Layer(api, T, K, N, x=x)
    layer.w = np.full((N, K), 127, np.int8)
    layer.w[1::2] = -128
    layer.channel = np.full(N, 1e-6, np.float32)
    layer.dw, layer.dc = dev(layer.w), dev(layer.channel)
    out = layer.out()
    layer.dynamic(out, layer.workspace())
    sync()
    assert_within(host(out)[:T], *layer.want())
    q, scales = np.full((T, K), -128, np.int8), np.full(T, 0.0125, np.float32)
    q[1::2] = 127
    dq, ds, one = dev(q), dev(scales), layer.out()
    p = params(capi.Int8TokenLinearParams, T, K, N, False, layer.dw, layer.dc, layer.db, one, a=ptr(dq), token_scale=ptr(ds))
    api.check(api.int8_token_linear(stream(), C.byref(p)))
    sync()
    assert_within(host(one)[:T], *reference(q, scales, layer.w, layer.channel, layer.bias, False))


@pytest.mark.parametrize("T,K,N", [(1, 1024, 64), (20, 128, 64), (4, 4160, 64), (300, 256, 288), (1500, 192, 320), (2600, 1024, 1024)])
def test_gelu_beyond_binary32(api, T, K, N):
    """Products past the end of binary32, either way: infinity and zero, as for every large result; the other channels as ever."""
    layer = Layer(api, T, K, N, gelu=True, bias=False)
    layer.channel[::2] = 3e38
    layer.dc = dev(layer.channel)
    one, two = layer.out(), layer.out()
    layer.token(one)
    layer.dynamic(two, layer.workspace())
    sync()
    assert np.array_equal(bits(one), bits(two))
    q, scales = quantised(layer.x)
    acc = q.astype(np.float64) @ layer.w.astype(np.float64).T
    got, up, down = host(one)[:T], acc[:, ::2] > 1000, acc[:, ::2] < -1000  # scales of 0.005 and more: beyond 1.5e39
    assert up.any() and down.any() and (scales > 0.005).all()
    assert (got[:, ::2][up] == np.inf).all() and (got[:, ::2][down] == 0).all()
    want, tol = layer.want()
    assert_within(got[:, 1::2], want[:, 1::2], tol[:, 1::2])


@pytest.mark.parametrize("T,K,N", [(33333, 64, 2208), (33000, 128, 2304), (17001, 192, 4512), (40001, 256, 1952), (19000, 64, 4160)])
@pytest.mark.parametrize("gelu", [False, True])
def test_results_past_the_last_level_cache(api, T, K, N, gelu):
    """The bits of the same tokens in calls whose results stay in the caches, and the definition on some of them."""
    import torch
    assert api.test_token_linear_streams(T, K, N) and not api.test_token_linear_streams(4000, K, N)
    layer = Layer(api, T, K, N, gelu)
    out, ws = layer.out(), layer.workspace()
    layer.dynamic(out, ws)
    for t in range(0, T, 4000):
        n = min(4000, T - t)
        part, space = dev_empty((n, N), np.float16, fill=-7), dev_empty((api.int8_dynamic_linear_workspace_size(n, K, N),), np.uint8)
        p = params(capi.Int8DynamicLinearParams, n, K, N, gelu, layer.dw, layer.dc, layer.db, part, a=ptr(layer.dx[t:]), a_stride=K,
                   workspace=ptr(space), workspace_bytes=space.numel())
        api.check(api.int8_dynamic_linear(stream(), C.byref(p)))
        assert torch.equal(part.view(torch.int16), out[t:t + n].view(torch.int16)), t
    sync()
    assert (host(out[T]) == -7).all()
    some = np.r_[0:40, T - 300:T]
    want, tol = reference(*quantised(layer.x[some]), layer.w, layer.channel, layer.bias, gelu)
    assert_within(host(out[:T])[some], want, tol)


def test_two_threads_at_once(api):
    """Calls of two threads, each with layers and a stream of its own: plans are remembered by each thread for itself."""
    import threading

    import torch
    work = [[Layer(api, T, K, N, gelu, seed=s) for T, K, N, gelu in sizes]
            for s, sizes in enumerate([[(600, 960, 1056, False), (5003, 960, 1056, False), (1, 1024, 512, True)],
                                       [(600, 960, 1056, True), (3, 4096, 224, False), (2049, 384, 1536, True)]])]
    want = []
    for layers in work:
        for layer in layers:
            want.append(layer.out())
            layer.dynamic(want[-1], layer.workspace())
    outs = [[layer.out() for layer in layers] for layers in work]
    spaces = [[layer.workspace() for layer in layers] for layers in work]
    streams = [torch.cuda.Stream() for _ in work]
    sync()
    failed = []

    def calls(i):
        try:
            for _ in range(20):
                for layer, out, ws in zip(work[i], outs[i], spaces[i]):
                    layer.dynamic(out, ws, streams[i].cuda_stream)
        except Exception as e:  # an assertion of a thread is not seen by itself
            failed.append(e)

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    sync()
    assert not failed
    for got, ref in zip(outs[0] + outs[1], want):
        assert np.array_equal(bits(got), bits(ref))
