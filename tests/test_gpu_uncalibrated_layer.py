"""One encoder layer without calibrated activations and with rotary positions, put together as a caller would: the QKV
projection on FP16 tokens, norms and rotation of queries and keys in place in the packed tensor, fused attention,
projection, SkipLayerNorm, and the feed-forward layers, the first from tokens that are quantised once. Every stage is
checked against the binary64 definition on what the stage before it left on the GPU; the attention and the norms with
the tolerances of their own tests, the rest with theirs."""
import ctypes as C

import numpy as np
import pytest

from helpers import assert_fp_close, attention_f64, dev, dev_empty, half2_bits, host, layer_norm_f64, ptr, rng, stream, sync
from tensorrt_amd import capi
from test_gpu_qk_norm_rotary import Problem, case_of, definition
from test_gpu_token_linear import activations, assert_within, quantised, reference, weights

pytestmark = pytest.mark.gpu
D = 64


@pytest.fixture(scope="module")
def api():
    return capi.api()


class EncoderLayer:
    def __init__(self, api, lens, heads, ffn, axes, seed):
        r = self.r = rng(seed)
        self.api, self.heads, self.ffn = api, heads, ffn
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        T, H = int(self.cu[-1]), heads * D
        self.T, self.H, self.S = T, H, int(max(lens))
        # name: (in, out, gelu)
        self.shapes = dict(qkv=(H, 3 * H, False), proj=(H, H, False), up=(H, ffn, True), down=(ffn, H, False))
        self.w = {n: weights(r, N, K) for n, (K, N, _) in self.shapes.items()}
        self.dw = {n: tuple(dev(t) for t in w) for n, w in self.w.items()}
        self.gamma, self.beta = (r.uniform(0.5, 1.5, H).astype(np.float16), (0.1 * r.standard_normal(H)).astype(np.float16))
        self.dgamma, self.dbeta, self.dcu = dev(self.gamma), dev(self.beta), dev(self.cu)
        sections = [32] if axes == 1 else [12, 10, 10]
        self.rotary = Problem(api, case_of(T=T, hq=heads, hk=heads, sections=sections), seed)
        if axes == 1:
            self.rotary.positions[0] = np.concatenate([np.arange(n) for n in lens])
            self.rotary.fixed[5].copy_(dev(self.rotary.positions))
        half = lambda *s: dev_empty(s, np.float16, fill=-7)
        self.x = dev(activations(r, T, H))
        self.qkv_in, self.qkv, self.ctx, self.ao, self.mid = half(T, 3 * H), half(T, 3 * H), half(T, H), half(T, H), half(T, H)
        self.up, self.down, self.out = half(T, ffn), half(T, H), half(T, H)
        self.q8, self.scales = dev_empty((T, H), np.int8, fill=0), dev_empty((T,), np.float32, fill=0)
        size = max(api.int8_dynamic_linear_workspace_size(T, K, N) for K, N, _ in self.shapes.values())
        self.ws = dev_empty((size,), np.uint8, fill=0)

    def dynamic(self, s, name, x, out):
        (K, N, gelu), (w, channel, bias) = self.shapes[name], self.dw[name]
        p = capi.Int8DynamicLinearParams(a=ptr(x), a_stride=K, w=ptr(w), channel_scale=ptr(channel), bias=ptr(bias), out=ptr(out),
                                         workspace=ptr(self.ws), workspace_bytes=self.ws.numel(), T=self.T, K=K, N=N, epilogue=int(gelu))
        self.api.check(self.api.int8_dynamic_linear(s, C.byref(p)))

    def norm(self, s, x, skip, out):
        self.api.check(self.api.skip_layer_norm_fp16(s, self.H, self.T * self.H, ptr(x), ptr(skip), ptr(self.dbeta), ptr(self.dgamma),
                                                     ptr(out), None))

    def run(self, s=None):
        s, T, H, api = s or stream(), self.T, self.H, self.api
        self.dynamic(s, "qkv", self.x, self.qkv)
        self.qkv_in.copy_(self.qkv)  # what the rotation overwrites, for the check
        packed = self.qkv.view(T, self.heads, 3, D)
        p = self.rotary.params(packed[:, :, 0], packed[:, :, 1], packed[:, :, 0], packed[:, :, 1])
        api.check(api.qk_norm_rotary(s, 1, C.byref(p)))
        f = capi.FmhaParams(qkv_ptr=ptr(self.qkv), o_ptr=ptr(self.ctx), qkv_stride_in_bytes=6 * H, o_stride_in_bytes=2 * H,
                            b=len(self.cu) - 1, h=self.heads, s=self.S, d=D, scale_bmm1=half2_bits(0.125), scale_softmax=half2_bits(1.0),
                            scale_bmm2=half2_bits(1.0), cu_seqlens=ptr(self.dcu))
        api.check(api.fused_mha_run(s, 1, C.byref(f)))
        self.dynamic(s, "proj", self.ctx, self.ao)
        self.norm(s, self.ao, self.x, self.mid)
        api.check(api.quantize_fp16_per_token(s, T, H, ptr(self.mid), H, ptr(self.q8), ptr(self.scales)))
        (K, N, gelu), (w, channel, bias) = self.shapes["up"], self.dw["up"]
        q = capi.Int8TokenLinearParams(a=ptr(self.q8), token_scale=ptr(self.scales), w=ptr(w), channel_scale=ptr(channel), bias=ptr(bias),
                                       out=ptr(self.up), T=T, K=K, N=N, epilogue=int(gelu))
        api.check(api.int8_token_linear(s, C.byref(q)))
        self.dynamic(s, "down", self.up, self.down)
        self.norm(s, self.down, self.mid, self.out)

    def check(self):
        sync()
        t = {n: host(getattr(self, n)) for n in ("x", "qkv_in", "qkv", "ctx", "ao", "mid", "up", "down", "out")}
        for name, x, y in (("qkv", "x", "qkv_in"), ("proj", "ctx", "ao"), ("up", "mid", "up"), ("down", "up", "down")):
            assert np.isfinite(t[x]).all()
            want, tol = reference(*quantised(t[x]), *self.w[name], self.shapes[name][2])
            assert_within(t[y], want, tol, name)
        before, after = (t[n].reshape(self.T, self.heads, 3, D) for n in ("qkv_in", "qkv"))
        for i in range(2):
            p = self.rotary
            want, tol = definition(before[:, :, i], p.vectors[i], p.vectors[2 + i], p.case, p.frequencies, p.positions)
            assert_within(after[:, :, i], want, tol, "qk"[i])
        assert np.array_equal(after[:, :, 2], before[:, :, 2])
        want = np.zeros((self.T, self.heads, D))
        for lo, hi in zip(self.cu[:-1], self.cu[1:]):
            for h in range(self.heads):
                if hi > lo:
                    want[lo:hi, h] = attention_f64(after[lo:hi, h, 0], after[lo:hi, h, 1], after[lo:hi, h, 2], 0.125)
        assert_fp_close(t["ctx"], want.reshape(self.T, self.H), what="attention")
        for a, b, y in (("ao", "x", "mid"), ("down", "mid", "out")):
            v = (t[a] + t[b]).astype(np.float64)  # the residual sum is formed in FP16
            assert_fp_close(t[y], layer_norm_f64(v, self.gamma, self.beta, 2.0 ** -10 if self.H in (768, 1024) else 0.0), what=y)


CASES = [([1], 4, 256, 1), ([5, 1, 9], 4, 512, 1), ([33, 128, 1, 77], 12, 1536, 1), ([100, 100], 6, 1024, 3), ([300, 17, 256, 384, 64], 4, 640, 1)]


@pytest.mark.parametrize("lens,heads,ffn,axes", CASES)
def test_layer(api, lens, heads, ffn, axes):
    layer = EncoderLayer(api, lens, heads, ffn, axes, seed=len(lens) + heads)
    layer.run()
    layer.check()


@pytest.mark.parametrize("lens", [[7, 2], [60, 130, 5]])
def test_captured_layer(api, lens):
    """The whole layer as a graph: each replay follows what the input holds, with an eager pass on buffers of its own between the replays."""
    import torch
    layer, other = (EncoderLayer(api, lens, 4, 512, 1, seed=3) for _ in range(2))
    layer.run()  # the first launches of the kernels, outside the capture
    sync()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer.run(side.cuda_stream)
    for replay in range(3):
        x = dev(activations(rng(replay), layer.T, layer.H))
        layer.x.copy_(x)
        other.x.copy_(x)
        layer.out.fill_(-7)
        other.run()
        graph.replay()
        sync()
        assert np.array_equal(host(layer.out).view(np.uint16), host(other.out).view(np.uint16)), replay
        layer.check()
    del graph
