"""The operators of a layer that generates, run together as a serving loop runs them: norms and rotation of the projection's queries and
keys in place, keys and values into the cache, attention over it; prompts first, then tokens one by one and a few at a time; as graphs,
on two streams, from two threads. And attention's ways to share work out, each at sizes that take it."""
import ctypes as C
import threading

import numpy as np
import pytest

from cache_helpers import Cache
from helpers import dev, dev_empty, host, ptr, rng, stream, sync
from tensorrt_amd import capi
from test_gpu_kv_cache import attend, attention_params, check_attention, filled, new_rows, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def api():
    return capi.api()


class Layer:
    """B sequences of one attention layer, at most `rows` rows a step; its calls' parameters are made once, as a captured step needs."""

    def __init__(self, api, dtype, B, heads, H, d, P, capacity, rows, window=0, sinks=0, seed=0):
        self.api, self.heads, self.H, self.d, self.rows, self.window, self.sinks = api, heads, H, d, rows, window, sinks
        self.cache = Cache(dtype, P, H, d, B * -(-capacity // P) + 2, B, -(-capacity // P), seed)
        self.r = self.cache.r
        N = heads + 2 * H
        self.qkv, self.out = dev_empty((rows, N, d), np.float16, fill=0), dev_empty((rows, heads, d), np.float16, fill=-7)
        self.dcu, self.positions = dev_empty((B + 1,), np.int32, fill=0), dev_empty((rows,), np.int32, fill=0)
        self.weights = [dev(self.r.uniform(0.5, 1.5, d).astype(np.float32)) for _ in range(2)]
        self.frequencies = dev((10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32))
        c, keep = self.cache.described([0] * (B + 1), T=rows, max_tokens=rows)
        c.cu_seqlens = ptr(self.dcu)
        s = dict(token_stride=N * d, head_stride=d)
        at = lambda x, n: ptr(x) + 2 * n * d
        strides = lambda *names: {f"{n}_{k}": v for n in names for k, v in s.items()}
        self.rotary = capi.QkNormRotaryParams(q=ptr(self.qkv), k=at(self.qkv, heads), q_out=ptr(self.qkv), k_out=at(self.qkv, heads), T=rows, q_heads=heads,
                                              k_heads=H, d=d, norm=capi.QK_NORM_RMS, eps=1e-6, q_weight=ptr(self.weights[0]), k_weight=ptr(self.weights[1]),
                                              rotary_dim=d, frequencies=ptr(self.frequencies), positions=ptr(self.positions), axes=1,
                                              **strides("q", "k", "q_out", "k_out"))
        self.write = capi.KvCacheWriteParams(cache=c, k=at(self.qkv, heads), v=at(self.qkv, heads + H), **strides("k", "v"))
        self.attention = capi.KvCacheAttentionParams(cache=c, q=ptr(self.qkv), out=ptr(self.out), q_token_stride=N * d, q_head_stride=d,
                                                     out_token_stride=heads * d, out_head_stride=d, q_heads=heads, scale=float(np.float32(d ** -0.5)),
                                                     window=window, sinks=sinks)
        self.size = api.kv_cache_attention_workspace_size(C.byref(self.attention))
        self.use(dev_empty((max(self.size, 16),), np.uint8, fill=0xFF))

    def use(self, workspace):
        self.ws = workspace
        self.attention.workspace, self.attention.workspace_bytes = ptr(workspace), workspace.numel()

    def feed(self, new):
        """The projection's result for `new` rows of each sequence, and the tables that go with it, on the current stream."""
        self.cache.grow(new)
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        T = int(self.cu[-1])
        x = self.r.standard_normal((self.rows, self.heads + 2 * self.H, self.d)).astype(np.float16)
        at = np.zeros(self.rows, np.int32)
        for b, n in enumerate(new):
            at[self.cu[b]:self.cu[b + 1]] = self.cache.lengths[b] - n + np.arange(n)
        self.qkv.copy_(dev(x))
        self.dcu.copy_(dev(self.cu))
        self.positions.copy_(dev(at))
        self.out.fill_(-7)
        return T

    def run(self, s=None):
        s = stream() if s is None else s
        self.api.check(self.api.qk_norm_rotary(s, 1, C.byref(self.rotary)))
        self.api.check(self.api.kv_cache_write(s, C.byref(self.write)))
        self.api.check(self.api.kv_cache_attention(s, C.byref(self.attention)))

    def check(self, sample=24):
        """The cache byte by byte, and the attention, on what the rotation left."""
        sync()
        T, x, got = int(self.cu[-1]), host(self.qkv), host(self.out)
        self.cache.write(x[:, self.heads:self.heads + self.H], x[:, self.heads + self.H:], self.cu)
        self.cache.check()
        check_attention(self.cache, self.cu, x[:T, :self.heads], got[:T], self.attention.scale, self.window, self.sinks, sample=sample)
        assert (got[T:] == -7).all()


LAYERS = [("int8", 3, 4, 4, 64, 16, 0, 0), ("fp8", 2, 8, 2, 128, 64, 0, 0), ("int8", 5, 6, 2, 80, 32, 60, 3), ("fp8", 1, 4, 1, 256, 128, 0, 0)]
STEPS = [[97, 5, 64, 31, 12], [1, 1, 1, 1, 1], [3, 1, 2, 0, 3], [1, 1, 1, 1, 1], [30, 1, 1, 50, 2], [1, 1, 1, 1, 1]]


@pytest.mark.parametrize("dtype,B,heads,H,d,P,window,sinks", LAYERS)
def test_generating(api, dtype, B, heads, H, d, P, window, sinks):
    layer = Layer(api, dtype, B, heads, H, d, P, 256, 300, window, sinks, seed=d)
    for new in STEPS:
        layer.feed(new[:B])
        layer.run()
        layer.check()


def captured(layer):
    """A warmed step as a graph; what it wrote is of a step that has been fed."""
    import torch
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    return graph


@pytest.mark.parametrize("dtype,B,heads,H,d,P,window,sinks", LAYERS)
def test_captured_steps(api, dtype, B, heads, H, d, P, window, sinks):
    """One graph for steps of any rows and lengths: each replay follows what the tables hold; eager steps of another layer between them. The
    graph is captured before any eager call of its layer."""
    layer, other = (Layer(api, dtype, B, heads, H, d, P, 256, 300, window, sinks, seed=s) for s in (1, 2))
    graph = captured(layer)
    for new in STEPS:
        layer.feed(new[:B])
        graph.replay()
        layer.check()
        other.feed(new[:B])
        other.run()
        other.check()


def test_two_graphs_share_a_workspace(api):
    """Replayed in turn, on contexts long enough to need it."""
    layers = [Layer(api, t, 2, 8, 2, 128, 64, 4000, 4000, seed=s) for s, t in enumerate(("int8", "fp8"))]
    ws = dev_empty((max(l.size for l in layers),), np.uint8, fill=0xFF)
    assert layers[0].size > 0
    for l in layers:
        l.use(ws)
    graphs = [captured(l) for l in layers]
    for new in ([3000, 900], [1, 1], [2, 1], [1, 1]):
        for l, g in zip(layers, graphs):
            l.feed(new)
            g.replay()
        for l in layers:
            l.check(sample=8)


@pytest.mark.parametrize("threads", [False, True])
def test_two_streams(api, threads):
    """Two layers at once, each on a stream, with a workspace and from a thread of its own."""
    import torch
    layers = [Layer(api, t, 3, 8, 2, 128, 16, 700, 700, seed=s) for s, t in enumerate(("int8", "fp8"))]
    streams = [torch.cuda.Stream() for _ in layers]
    for new in ([400, 100, 30], [1, 1, 1], [1, 2, 3], [1, 1, 1]):
        for l in layers:
            l.feed(new)
        sync()
        calls = [lambda l=l, s=s: l.run(s.cuda_stream) for l, s in zip(layers, streams)]
        if threads:
            started = [threading.Thread(target=c) for c in calls]
            [t.start() for t in started]
            [t.join() for t in started]
        else:
            [c() for c in calls]
        for l in layers:
            l.check(sample=8)


def lengths_of(B, top, seed):
    r = rng(seed)
    lens = np.maximum(1, (top * r.uniform(0, 1, B) ** 3).astype(int))
    lens[r.integers(0, B)] = top
    return lens


# dtype, sequences, key heads, d, longest, page, window; and the route: wavefronts, stretches, of one head each, tiles
ROUTES = [
    ("int8", 9, 1, 64, 300, 16, 0, (8, False, False)), ("fp8", 70, 8, 64, 200, 32, 0, (4, False, False)),
    ("int8", 3, 2, 128, 3000, 64, 0, (0, True, True)), ("fp8", 70, 1, 64, 3000, 16, 0, (0, True, True)),
    ("int8", 40, 4, 128, 1500, 16, 0, (0, True, False)), ("fp8", 70, 4, 96, 1500, 64, 700, (0, True, False)),
    ("fp8", 200, 5, 64, 1200, 128, 0, (0, True, False)), ("int8", 35, 4, 256, 700, 32, 0, (0, True, False))]


@pytest.mark.parametrize("dtype,B,H,d,top,P,window,want", ROUTES)
@pytest.mark.parametrize("mixed", [False, True])
def test_routes(api, dtype, B, H, d, top, P, window, want, mixed):
    """Sequences of very different lengths, of one chunk and of none; mixed: some of no rows, and some of more than the few rows' kernels take."""
    lens = lengths_of(B, top, seed=B)
    cache = filled(api, dtype, P, H, d, list(lens), seed=B + d, max_pages=-(-top // P))
    r = cache.r
    new = np.minimum(lens, r.integers(1, 3, B))
    if mixed:
        new[r.integers(0, B, 3)] = 0
        new[-1] = 0
        some = r.integers(0, B - 1, 4)
        new[some] = np.minimum(lens[some], 40)
    cache.lengths[r.integers(0, B, 2)] = 0  # rows that see nothing
    cache.upload()
    cu = np.concatenate([[0], np.cumsum(new)])
    q = r.standard_normal((int(cu[-1]), 2 * H, d)).astype(np.float16)
    p, keep = attention_params(cache, cu, dev(q), dev(q), 0.1, window=window, max_length=top, api=api)
    route = api.test_kv_cache_attention_route(C.byref(p))
    assert (route & 15, bool(route & 16), bool(route & 32)) == want and bool(route & 64) == mixed
    got = attend(api, cache, cu, q, 0.1, window=window, max_length=top)
    check_attention(cache, cu, q, got, 0.1, window, sample=4)
