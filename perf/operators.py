"""Operators of an encoder layer without calibrated activations and with rotary positions, as measurable cases.

    dynamic_linear   a linear layer on FP16 activations in INT8 arithmetic: every token is quantised with a scale of its
                     own, every output channel's weights have theirs (trtamd_int8_dynamic_linear)
    token_linear     the same product on tokens that are quantised already, for layers that share their input
                     (trtamd_int8_token_linear)
    rotary           norms of queries and keys for each head and the rotation by the token's position, one position per
                     token or several axes of them, in one pass (trtamd_qk_norm_rotary)

`run` computes them in elementary torch operations, or with `own` set through the library.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

TORCH = {"fp32": torch.float32, "fp16": torch.float16}
SIZE = {"fp32": 4, "fp16": 2}
TRT = {"fp32": 0, "fp16": 1}
EPS = 1e-6


def _linear(kind, T, K, N, gelu=False, bias=True, **more):
    return dict(kind=kind, T=T, K=K, N=N, gelu=gelu, bias=bias, **more)


def _rotary(T, heads, kv_heads, head, **more):
    """Defaults: FP16, RMS norm, the whole head rotated in halves, one position per token."""
    case = dict(kind="rotary", T=T, heads=heads, kv_heads=kv_heads, head=head, dtype="fp16", norm="rms", rotary=head,
                adjacent=False, theta=10000.0, far=0, axes="tokens")
    case.update(more)
    return case


def listed():
    return [
        # one token through the first feed-forward layer: latency, and the weights once
        dict(name="dynamic linear one token", **_linear("dynamic_linear", 1, 1024, 4096, gelu=True)),
        # one short request through the second feed-forward layer: long rows, few tokens
        dict(name="dynamic linear one request", **_linear("dynamic_linear", 40, 4096, 1024)),
        # a server's ordinary dynamic batch through the QKV projection
        dict(name="dynamic linear batch of 32", **_linear("dynamic_linear", 4963, 768, 2304)),
        # throughput: the benchmark batch through the first feed-forward layer
        dict(name="dynamic linear batch of 128", **_linear("dynamic_linear", 33289, 1024, 4096, gelu=True)),
        # a few queued requests, an odd number of tokens
        dict(name="token linear small batch", **_linear("token_linear", 777, 4096, 1024)),
        # the attention output projection of the benchmark batch, without a bias
        dict(name="token linear batch of 128", **_linear("token_linear", 33289, 1024, 1024, bias=False)),
        # the next token of one conversation, far into its context
        dict(name="norm rotary one token", **_rotary(1, 16, 16, 64, far=120000)),
        # packed sequences of an ordinary batch
        dict(name="norm rotary batch of 32", **_rotary(4963, 12, 12, 64)),
        # full precision, shared keys, part of an uncommon head rotated in adjacent pairs
        dict(name="norm rotary fp32 shared keys", **_rotary(1999, 12, 4, 80, dtype="fp32", norm="layer", rotary=32,
                                                            adjacent=True, far=1000000)),
        # the benchmark batch
        dict(name="norm rotary batch of 128", **_rotary(33289, 16, 16, 64)),
        # eight images of 37 x 37 patches: height and width, frequencies of their own, no norm
        dict(name="rotary images", **_rotary(8 * 37 * 37, 16, 16, 80, norm="none", axes="image", theta=100.0)),
        # a clip of 13 latent frames of 30 x 52: time, height and width
        dict(name="norm rotary video", **_rotary(13 * 30 * 52, 12, 12, 128, axes="video")),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        T = _log(rng, 1, 33289)
        while True:  # no more work than the benchmark batch's feed-forward layer
            K, N = 64 * _log(rng, 2, 64), 32 * _log(rng, 2, 160)
            if T * K * N <= 33289 * 1024 * 4096:
                break
        return _linear(rng.choice(("dynamic_linear", "token_linear")), T, K, N, gelu=rng.random() < 0.3,
                       bias=rng.random() < 0.7)
    head = rng.choice((32, 64, 64, 72, 80, 96, 128))
    heads = rng.choice((4, 8, 12, 16))
    axes = rng.choice(("tokens", "tokens", "image", "video"))
    more = dict(dtype=rng.choice(("fp16", "fp16", "fp32")), norm=rng.choice(("rms", "rms", "layer", "none")),
                adjacent=rng.random() < 0.3, theta=rng.choice((100.0, 10000.0, 500000.0)),
                far=_log(rng, 1, 1000000), axes=axes)
    if axes == "tokens":
        more["rotary"] = rng.choice((head, head, head // 2))
    elif axes == "video":
        more["cycled"] = rng.random() < 0.4
    return _rotary(_log(rng, 1, 20280), heads, rng.choice((heads, heads, heads // 4)), head, **more)


# ---- inputs ------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_linear(case, seed):
    T, K, N = case["T"], case["K"], case["N"]
    g = _generator(seed)
    # normal activations, some channels larger than the rest, and tokens of different size
    x = torch.randn((T, K), generator=g, device="cuda")
    loud = torch.rand((K,), generator=g, device="cuda") < 0.01
    x *= torch.where(loud, 8.0, 1.0) * torch.exp(0.3 * torch.randn((T, 1), generator=g, device="cuda"))
    x = x.half()
    w = torch.randn((N, K), generator=g, device="cuda") / math.sqrt(K)
    channel_scale = w.abs().amax(1) / 127
    state = dict(w=(w / channel_scale[:, None]).round_().to(torch.int8), channel_scale=channel_scale,
                 bias=0.1 * torch.randn((N,), generator=g, device="cuda") if case["bias"] else None, gelu=case["gelu"])
    if case["kind"] == "dynamic_linear":
        state["x"] = x
    else:
        scale = x.float().abs().amax(1) / 127
        state.update(a=(x.float() / scale[:, None]).round_().to(torch.int8), token_scale=scale)
    return state


def _sections(case):
    """How the pairs of a head are shared between the axes, and the frequency of each pair."""
    pairs, theta = case["rotary"] // 2, case["theta"]
    spread = lambda n: theta ** (-np.arange(n) / n)
    if case["axes"] == "tokens":
        return [pairs], spread(pairs)
    if case["axes"] == "image":  # every axis has the whole range of frequencies
        parts = [pairs // 2, pairs - pairs // 2]
        return parts, np.concatenate([spread(n) for n in parts])
    # height and width; time has the rest, and where the axes take turns the pairs behind the last turn
    side = pairs // 3 - 1 if case.get("cycled") else 3 * pairs // 8
    return [pairs - 2 * side, side, side], spread(pairs)


def _axis_of_pair(case, sections):
    n = len(sections)
    if case.get("cycled"):
        return [i % n if i // n < sections[i % n] else 0 for i in range(case["rotary"] // 2)]
    return [axis for axis, pairs in enumerate(sections) for _ in range(pairs)]


def _positions(case, seed):
    T, far, r = case["T"], case["far"], np.random.default_rng(seed)
    if case["axes"] == "tokens":  # packed sequences, each somewhere up to `far` into its context
        lens = []
        while sum(lens) < T:
            lens.append(int(r.integers(1, 513)))
        return np.concatenate([np.arange(n) + r.integers(0, far + 1) for n in lens])[None, :T]
    if case["axes"] == "image":
        side = int(r.integers(16, 41)) if T != 8 * 37 * 37 else 37
        return np.stack([np.arange(T) // side % side, np.arange(T) % side])
    h, w = (30, 52) if T == 13 * 30 * 52 else map(int, r.integers(8, 53, 2))
    return np.stack([np.arange(T) // (h * w) + r.integers(0, far + 1), np.arange(T) // w % h, np.arange(T) % w])


def _prepare_rotary(case, seed):
    T, hq, hk, d = case["T"], case["heads"], case["kv_heads"], case["head"]
    g = _generator(seed)
    # what the QKV projection leaves: [token][head][q|k|v] where all have the same heads, otherwise one behind the other
    qkv = torch.randn((T, hq + 2 * hk, d), generator=g, device="cuda").to(TORCH[case["dtype"]])
    if hq == hk:
        by_head = qkv.view(T, hq, 3, d)
        q, k = by_head[:, :, 0], by_head[:, :, 1]
    else:
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    vector = lambda mean, std: mean + std * torch.randn((d,), generator=g, device="cuda")
    sections, frequencies = _sections(case)
    return dict(q=q, k=k, norm=case["norm"], weights=(vector(1.0, 0.2), vector(1.0, 0.2)),
                biases=(vector(0.0, 0.1), vector(0.0, 0.1)), dtype=case["dtype"], rotary=case["rotary"],
                adjacent=case["adjacent"], sections=sections, cycled=case.get("cycled", False),
                axis_of_pair=torch.tensor(_axis_of_pair(case, sections), device="cuda"),
                frequencies=torch.from_numpy(frequencies.astype(np.float32)).cuda(),
                positions=torch.from_numpy(np.ascontiguousarray(_positions(case, seed)).astype(np.int32)).cuda())


def prepare(case, seed):
    state = (_prepare_rotary if case["kind"] == "rotary" else _prepare_linear)(case, seed)
    state["kind"] = case["kind"]
    return state


# ---- the operators through the library ---------------------------------------------------------------------------

def _address(t):
    return None if t is None else t.data_ptr()


def _bind(state):
    """The call as a program keeps it from pass to pass: its parameters, its output and its workspace."""
    from tensorrt_amd import capi
    api = capi.api()
    if state["kind"] == "rotary":
        q, k = state["q"], state["k"]
        (T, hq, d), hk = q.shape, k.shape[1]
        outs = torch.empty((T, hq, d), dtype=q.dtype, device="cuda"), torch.empty((T, hk, d), dtype=k.dtype, device="cuda")
        norms = {"none": capi.QK_NORM_NONE, "rms": capi.QK_NORM_RMS, "layer": capi.QK_NORM_LAYER}
        p = capi.QkNormRotaryParams()
        p.q, p.k, p.q_out, p.k_out = (t.data_ptr() for t in (q, k, *outs))
        p.q_token_stride, p.q_head_stride, p.k_token_stride, p.k_head_stride = *q.stride()[:2], *k.stride()[:2]
        p.q_out_token_stride, p.q_out_head_stride = p.k_out_token_stride, p.k_out_head_stride = hq * d, d
        p.k_out_token_stride = hk * d
        p.T, p.q_heads, p.k_heads, p.d, p.norm, p.eps = T, hq, hk, d, norms[state["norm"]], EPS
        if state["norm"] != "none":
            p.q_weight, p.k_weight = map(_address, state["weights"])
        if state["norm"] == "layer":
            p.q_bias, p.k_bias = map(_address, state["biases"])
        p.rotary_dim, p.adjacent_pairs = state["rotary"], int(state["adjacent"])
        p.frequencies, p.positions = _address(state["frequencies"]), _address(state["positions"])
        p.axes, p.axes_cycled = len(state["sections"]), int(state["cycled"])
        for i, n in enumerate(state["sections"]):
            p.sections[i] = n
        state["call"] = lambda stream: api.qk_norm_rotary(stream, TRT[state["dtype"]], ctypes.byref(p))
        state["result"] = outs
    else:
        dynamic = state["kind"] == "dynamic_linear"
        a, w = state["x"] if dynamic else state["a"], state["w"]
        (T, K), N = a.shape, w.shape[0]
        out = torch.empty((T, N), dtype=torch.float16, device="cuda")
        p = capi.Int8DynamicLinearParams() if dynamic else capi.Int8TokenLinearParams()
        p.a, p.w, p.channel_scale, p.bias, p.out = map(_address, (a, w, state["channel_scale"], state["bias"], out))
        p.T, p.K, p.N, p.epilogue = T, K, N, capi.LINEAR_GELU if state["gelu"] else capi.LINEAR_AFFINE
        if dynamic:
            size = api.int8_dynamic_linear_workspace_size(T, K, N)
            state["workspace"] = torch.empty((size,), dtype=torch.uint8, device="cuda")
            p.a_stride, p.workspace, p.workspace_bytes = K, state["workspace"].data_ptr(), size
            state["call"] = lambda stream: api.int8_dynamic_linear(stream, ctypes.byref(p))
        else:
            p.token_scale = state["token_scale"].data_ptr()
            state["call"] = lambda stream: api.int8_token_linear(stream, ctypes.byref(p))
        state["result"] = out
    state["check"] = api.check


def _run_own(state):
    if "call" not in state:
        _bind(state)
    state["check"](state["call"](torch.cuda.current_stream().cuda_stream))
    return state["result"]


# ---- the same in elementary operations, binary32 -----------------------------------------------------------------

def _run_linear(state):
    if state["kind"] == "dynamic_linear":
        x = state["x"].float()
        amax = x.abs().amax(1, keepdim=True)
        # binary32 holds 127 x exactly and divides it correctly, so ties are seen as such; a token of zeros stays zeros
        a, scale = torch.round(127 * x / amax.clamp_min(2.0 ** -24)), amax / 127
    else:
        a, scale = state["a"].float(), state["token_scale"][:, None]
    y = torch.matmul(a, state["w"].float().t()) * scale * state["channel_scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    if state["gelu"]:
        y = 0.5 * y * torch.erfc(y * -math.sqrt(0.5))
    return y.half()


def _run_rotary(state):
    half = state["rotary"] // 2
    # angles in binary64: binary32 has no digits left behind the point for far positions
    angle = state["positions"].double()[state["axis_of_pair"]].t() * state["frequencies"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    outs = []
    for x, weight, bias in zip((state["q"], state["k"]), state["weights"], state["biases"]):
        y = x.float()
        if state["norm"] == "layer":
            y = y - y.mean(-1, keepdim=True)
        if state["norm"] != "none":
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight
        if state["norm"] == "layer":
            y = y + bias
        rest = y[..., 2 * half:]
        if state["adjacent"]:
            a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:2 * half]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        outs.append(torch.cat((turned, rest), -1).to(x.dtype))
    return tuple(outs)


def run(state):
    if own:
        return _run_own(state)
    return _run_rotary(state) if state["kind"] == "rotary" else _run_linear(state)


# ---- the definitions in binary64 ---------------------------------------------------------------------------------

def _exact_linear(state):
    if "x" in state:
        x = state["x"].double()
        top = torch.linalg.vector_norm(x, math.inf, dim=1)
        scale = top / 127
        a = (x.mul(127) / top.unsqueeze(1)).round()
    else:
        a, scale = state["a"].double(), state["token_scale"].double()
    w = state["w"].double()
    w *= state["channel_scale"].double().unsqueeze(1)
    y = torch.addmm(torch.zeros((), dtype=torch.float64, device="cuda"), a, w.t()).mul_(scale.unsqueeze(1))
    if state["bias"] is not None:
        y += state["bias"].double()
    if state["gelu"]:
        y *= torch.special.ndtr(y)
    return y


def _exact_rotary(state):
    rot, sections = state["rotary"], state["sections"]
    positions, frequencies = state["positions"].double(), state["frequencies"].double()
    angles = torch.zeros((positions.shape[1], rot // 2), dtype=torch.float64, device="cuda")
    begin = 0
    for axis, n in enumerate(sections):
        if state["cycled"]:  # pairs that no other axis takes are the first one's
            own_pairs = [i for i in range(rot // 2) if i % len(sections) == axis and i // len(sections) < n]
            if axis == 0:
                angles[:] = positions[:1].t() * frequencies
        else:
            own_pairs = list(range(begin, begin + n))
            begin += n
        angles[:, own_pairs] = positions[axis].unsqueeze(1) * frequencies[own_pairs]
    turn = torch.polar(torch.ones_like(angles), angles).unsqueeze(1)
    outs = []
    for i, name in enumerate("qk"):
        x = state[name].double().clone()
        if state["norm"] == "rms":
            x /= torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
            x *= state["weights"][i].double()
        elif state["norm"] == "layer":
            variance, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            x = (x - mean) / (variance + EPS).sqrt() * state["weights"][i].double() + state["biases"][i].double()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if state["adjacent"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        outs.append(x)
    return tuple(outs)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rotary(state) if case["kind"] == "rotary" else _exact_linear(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "rotary":
        size, values = SIZE[case["dtype"]], case["T"] * (case["heads"] + case["kv_heads"]) * case["head"]
        axes = {"tokens": 1, "image": 2, "video": 3}[case["axes"]]
        vectors = {"none": 0, "rms": 2, "layer": 4}[case["norm"]] * case["head"]
        return dict(bytes=2 * values * size + 4 * axes * case["T"] + 4 * vectors + 2 * case["rotary"],
                    flops=values * ({"none": 0, "rms": 4, "layer": 7}[case["norm"]] + 3 * case["rotary"] / case["head"]))
    T, K, N = case["T"], case["K"], case["N"]
    tokens = 2 * T * K if case["kind"] == "dynamic_linear" else T * (K + 4)
    return dict(bytes=tokens + N * K + 4 * N * (2 if case["bias"] else 1) + 2 * T * N, flops=2 * T * K * N)
