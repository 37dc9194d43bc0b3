"""Norms of queries and keys for each head with their rotation, against the definition in binary64.

Tolerances. Everything but the angle is binary32. A mean of squares of up to 256 values: a lane adds up to 16 of them
(two roundings each with the square), lanes meet in 6 steps, so it is within 24 steps of 2^-24; the division, the
addition of eps, the root and the reciprocal add four more, the root halves what came before them, and the products
with the scale and the weight are two: a normed value is within 20 * 2^-24 of itself. A LayerNorm's mean is within 24
* 2^-24 of the largest |x| and is subtracted with one more rounding: 25 * 2^-24 max|x| scale |w| more, and the
variance takes that twice over (relative to the deviation, which is no less than max|x| / 4 in these inputs): 60 *
2^-24 of the value instead of 20; the bias adds one rounding. The angle is reduced to half a turn in binary64 (two
products of 2^-53 of the turns) and rounded to binary32 (2^-25 of half a turn, 1e-7 = 1.6 * 2^-24); the library's sine
and cosine are within 4 steps of 2^-24 of 1. Two products and a sum: three roundings. Together a rotated value is
within (20 or 60 + 1.6 + 4 + 3) * 2^-24 (|a| + |b|), where a and b are the normed pair. FP16 results round once more:
2^-11 of the value or 2^-25."""
import ctypes as C

import numpy as np
import pytest

from helpers import dev, dev_empty, host, ptr, rng, stream, sync
from tensorrt_amd import capi

pytestmark = pytest.mark.gpu
EPS = 1e-6
STEP = 2.0 ** -24


@pytest.fixture(scope="module")
def api():
    return capi.api()


def axis_of(i, case):
    sections, n = case["sections"], len(case["sections"])
    if case["cycled"]:
        return i % n if i // n < sections[i % n] else 0
    return int(np.searchsorted(np.cumsum(sections), i, side="right"))


def definition(x, w, b, case, frequencies, positions):
    """(result, tolerance) of x [T][heads][d] in binary64."""
    x = x.astype(np.float64)
    norm, rot, d = case["norm"], case["rotary"], x.shape[-1]
    off = np.zeros_like(x)
    if norm == "rms":
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
        off = 20 * STEP * np.abs(y)
    elif norm == "layer":
        scale = 1 / np.sqrt(x.var(-1, keepdims=True) + EPS)
        y = (x - x.mean(-1, keepdims=True)) * scale * w
        off = 60 * STEP * np.abs(y) + 25 * STEP * np.abs(x).max(-1, keepdims=True) * scale * np.abs(w) + STEP * (np.abs(y) + np.abs(b))
        y = y + b
    else:
        y = x.copy()
    half = rot // 2
    if half:
        axes = np.array([axis_of(i, case) for i in range(half)])
        turns = positions.astype(np.float64)[axes].T * frequencies.astype(np.float64)
        c, s = np.cos(turns)[:, None], np.sin(turns)[:, None]
        at = (slice(0, rot, 2), slice(1, rot, 2)) if case["adjacent"] else (slice(0, half), slice(half, rot))
        a, b2 = y[..., at[0]].copy(), y[..., at[1]].copy()
        both = off[..., at[0]] + off[..., at[1]] + (8.6 * STEP + 2.0 ** -51 * np.abs(turns)[:, None]) * (np.abs(a) + np.abs(b2))
        y[..., at[0]], y[..., at[1]] = a * c - b2 * s, b2 * c + a * s
        off[..., at[0]] = off[..., at[1]] = both
    if case["dtype"] == np.float16:
        off = off + np.maximum(2.0 ** -11 * (np.abs(y) + off), 2.0 ** -25)
    else:
        off = off + 2.0 ** -149
    return y, off


def case_of(**change):
    case = dict(T=37, hq=3, hk=3, d=64, rotary=64, dtype=np.float16, norm="rms", adjacent=False, sections=[32], cycled=False, far=1000)
    case.update(change)
    if len(case["sections"]) == 1:
        case["sections"] = [case["rotary"] // 2]
    return case


class Problem:
    def __init__(self, api, case, seed=0):
        self.api, self.case = api, case
        r = self.r = rng([case["T"], case["d"], case["rotary"], seed])
        T, d, dt = case["T"], case["d"], case["dtype"]
        self.q, self.k = (r.standard_normal((T, h, d)).astype(dt) for h in (case["hq"], case["hk"]))
        self.vectors = [(1 + 0.3 * r.standard_normal(d)).astype(np.float32) for _ in range(2)]
        self.vectors += [(0.2 * r.standard_normal(d)).astype(np.float32) for _ in range(2)]
        half = case["rotary"] // 2
        self.frequencies = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
        self.positions = r.integers(-case["far"], case["far"] + 1, (len(case["sections"]), T)).astype(np.int32)
        self.fixed = [dev(v) for v in (*self.vectors, self.frequencies, self.positions)]

    def want(self):
        return [definition(x, self.vectors[i], self.vectors[2 + i], self.case, self.frequencies, self.positions)
                for i, x in enumerate((self.q, self.k))]

    def params(self, q, k, qo, ko):
        case, (qw, kw, qb, kb, f, pos) = self.case, self.fixed
        p = capi.QkNormRotaryParams()
        for name, t in (("q", q), ("k", k), ("q_out", qo), ("k_out", ko)):
            setattr(p, name, ptr(t))
            if t is not None:
                setattr(p, name + "_token_stride", t.stride(0))
                setattr(p, name + "_head_stride", t.stride(1))
        p.T, p.q_heads, p.k_heads, p.d = case["T"], case["hq"], case["hk"], case["d"]
        p.norm, p.eps = {"none": 0, "rms": 1, "layer": 2}[case["norm"]], EPS
        p.q_weight, p.k_weight, p.q_bias, p.k_bias = ptr(qw), ptr(kw), ptr(qb), ptr(kb)
        p.rotary_dim, p.adjacent_pairs, p.frequencies, p.positions = case["rotary"], int(case["adjacent"]), ptr(f), ptr(pos)
        p.axes, p.axes_cycled = len(case["sections"]), int(case["cycled"])
        for i, n in enumerate(case["sections"]):
            p.sections[i] = n
        return p

    def call(self, q, k, qo, ko, s=None):
        p = self.params(q, k, qo, ko)
        self.api.check(self.api.qk_norm_rotary(s or stream(), 1 if self.case["dtype"] == np.float16 else 0, C.byref(p)))

    def outs(self):
        c = self.case
        return [dev_empty((c["T"] + 1, h, c["d"]), c["dtype"], fill=-7) for h in (c["hq"], c["hk"])]

    def check(self, got, what=""):
        for g, (want, tol), name in zip(got, self.want(), "qk"):
            g = host(g)[:self.case["T"]].astype(np.float64)
            bad = ~(np.abs(g - want) <= tol)
            assert not bad.any(), (f"{what} {name}: {bad.sum()} of {bad.size} outside, first at {np.argwhere(bad)[0]}: "
                                   f"{g[bad][0]} for {want[bad][0]} +- {tol[bad][0]}")


def run(api, seed=0, **change):
    p = Problem(api, case_of(**change), seed)
    outs = p.outs()
    p.call(dev(p.q), dev(p.k), *outs)
    sync()
    p.check(outs, str(change))
    for o in outs:
        assert (host(o)[p.case["T"]] == -7).all(), "something behind the last token was written"
    return outs


DTYPES = [np.float16, np.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 64), (32, 32), (128, 128), (256, 256), (80, 80), (72, 72), (96, 48), (64, 16), (80, 32), (88, 88), (128, 2),
                                      (100, 60), (10, 6), (63, 62), (255, 254), (255, 120), (2, 2), (17, 4), (160, 96), (248, 200)])
def test_heads(api, dtype, norm, adjacent, d, rotary):
    run(api, dtype=dtype, norm=norm, adjacent=adjacent, d=d, rotary=rotary)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,norm", [(1, "rms")] + [(d, norm) for d in (8, 33, 64, 72, 256) for norm in ("rms", "layer")])
def test_norms_without_rotation(api, dtype, d, norm):
    run(api, dtype=dtype, d=d, rotary=0, norm=norm)


@pytest.mark.parametrize("T", [1, 2, 3, 7, 64, 513, 3001])
@pytest.mark.parametrize("hq,hk", [(1, 1), (12, 12), (16, 4), (5, 0), (0, 3), (7, 1), (40, 8), (96, 96)])
def test_tokens_and_heads(api, T, hq, hk):
    run(api, T=T, hq=hq, hk=hk)
    run(api, T=T, hq=hq, hk=hk, d=32, rotary=32, dtype=np.float32, norm="layer")


@pytest.mark.parametrize("T", [20011])
@pytest.mark.parametrize("dtype,d,norm", [(np.float16, 64, "rms"), (np.float16, 128, "none"), (np.float32, 80, "layer"), (np.float16, 72, "rms")])
def test_many_tokens(api, T, dtype, d, norm):
    run(api, T=T, hq=8, hk=2, d=d, rotary=d, dtype=dtype, norm=norm)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("d,rotary,sections,cycled", [
    (64, 64, [16, 16], False), (80, 80, [20, 20], False), (128, 128, [16, 24, 24], False), (128, 128, [24, 20, 20], True), (72, 72, [12, 11, 13], False),
    (64, 32, [5, 4, 4, 3], False), (64, 32, [4, 4, 4, 4], True), (96, 96, [48, 0], False), (96, 96, [0, 48], False), (64, 64, [0, 0, 32], False),
    (64, 64, [32, 0, 0, 0], True), (64, 64, [11, 11, 10], True), (10, 10, [2, 2, 1], True), (10, 10, [1, 3, 1], False)])
def test_axes(api, dtype, adjacent, d, rotary, sections, cycled):
    run(api, T=61, dtype=dtype, adjacent=adjacent, d=d, rotary=rotary, sections=sections, cycled=cycled, norm="none")
    run(api, T=61, dtype=dtype, adjacent=adjacent, d=d, rotary=rotary, sections=sections, cycled=cycled)


@pytest.mark.parametrize("far", [0, 1, 100000, 16777217, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(api, far, dtype):
    run(api, T=200, far=far, dtype=dtype)


def test_position_zero_and_no_norm_change_nothing(api):
    for d, dtype in ((64, np.float16), (72, np.float16), (33, np.float32)):
        p = Problem(api, case_of(norm="none", far=0, d=d, rotary=d - d % 2, dtype=dtype))
        outs = p.outs()
        p.call(dev(p.q), dev(p.k), *outs)
        sync()
        for o, x in zip(outs, (p.q, p.k)):
            assert np.array_equal(host(o)[:p.case["T"]], x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rotary,adjacent", [(64, 64, False), (64, 32, True), (80, 80, False), (72, 40, False), (33, 32, True)])
def test_in_place_in_packed_layouts(api, dtype, d, rotary, adjacent):
    """[token][head][q|k|v][d] and [token][q heads, k heads, v heads][d]: V, and what lies between, stays as it was; the bits are those
    of the call with outputs of their own."""
    T, h = 45, 4
    p = Problem(api, case_of(T=T, hq=h, hk=h, d=d, rotary=rotary, adjacent=adjacent, dtype=dtype))
    outs = p.outs()
    p.call(dev(p.q), dev(p.k), *outs)
    for layout in range(2):
        qkv = np.full((T + 1, h, 3, d) if layout == 0 else (T + 1, 3, h, d), 5, dtype)
        q, k = (qkv[:T, :, 0], qkv[:T, :, 1]) if layout == 0 else (qkv[:T, 0], qkv[:T, 1])
        q[:], k[:] = p.q, p.k
        t = dev(qkv)
        dq, dk = (t[:T, :, 0], t[:T, :, 1]) if layout == 0 else (t[:T, 0], t[:T, 1])
        p.call(dq, dk, dq, dk)
        sync()
        got = host(t)
        gq, gk, gv = (got[:T, :, i] for i in range(3)) if layout == 0 else (got[:T, i] for i in range(3))
        assert (gv == 5).all() and (got[T] == 5).all()
        for g, o in zip((gq, gk), outs):
            assert np.array_equal(g, host(o)[:T])
        p.check([np_as_dev(gq), np_as_dev(gk)])


def np_as_dev(a):
    return dev(np.ascontiguousarray(a))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_addresses_and_strides_of_any_alignment(api, dtype, shift):
    """Heads that start anywhere, in rows of odd strides, and vectors that are not 16-byte aligned."""
    import torch
    T, h, d = 29, 3, 64
    p = Problem(api, case_of(T=T, hq=h, hk=h, dtype=dtype, norm="layer"))
    dt = p.outs()[0].dtype
    views = []
    for x in (p.q, p.k, None, None):
        flat = torch.full((T * (h * (d + shift) + 3 * shift) + shift + 8,), -7.0, dtype=dt, device="cuda")
        v = flat[shift:].as_strided((T, h, d), (h * (d + shift) + 3 * shift, d + shift, 1), shift)
        if x is not None:
            v.copy_(dev(x))
        views.append((flat, v))
    before = [f.clone() for f, _ in views]
    if shift == 1:
        p.fixed[:4] = [torch.cat([torch.zeros(1, device="cuda"), v])[1:] for v in p.fixed[:4]]
    p.call(*[v for _, v in views])
    sync()
    p.check([views[2][1].contiguous(), views[3][1].contiguous()])
    for (flat, v), was in zip(views, before):
        was.as_strided(v.shape, v.stride(), v.storage_offset()).copy_(v)
        assert torch.equal(flat, was), "something between the heads was written"


def test_keys_shared_by_a_stride_of_zero(api):
    """A broadcast input (the same head for all): read where it is."""
    p = Problem(api, case_of(T=20, hq=4, hk=4))
    p.k[:] = p.k[:, :1]
    k = dev(np.ascontiguousarray(p.k[:, :1])).expand(20, 4, 64)
    outs = p.outs()
    p.call(dev(p.q), k, *outs)
    sync()
    p.check(outs)


@pytest.mark.parametrize("norm", ["rms", "layer", "none"])
def test_values_that_are_not_finite_stay_in_their_head(api, norm):
    p = Problem(api, case_of(norm=norm, T=9))
    q = p.q.copy()
    q[2, 1, 5], q[4, 0, 63], q[8, 2, 32] = np.nan, np.inf, -np.inf
    outs = p.outs()
    p.call(dev(q), dev(p.k), *outs)
    sync()
    got = host(outs[0])[:9].copy()
    hit = ~np.isfinite(got)
    heads = {(t, h) for t, h, _ in np.argwhere(hit)}
    assert heads == {(2, 1), (4, 0), (8, 2)}
    for t, h in heads:
        got[t, h] = 0
    want, tol = p.want()[0]
    for t, h in heads:
        want[t, h] = 0
    assert (np.abs(got - want) <= tol).all()


def test_heads_of_zeros(api):
    """Without a value the norms leave zeros (eps), a LayerNorm its bias."""
    for norm in ("rms", "layer"):
        p = Problem(api, case_of(norm=norm, T=5))
        p.q[:, 1] = 0
        outs = p.outs()
        p.call(dev(p.q), dev(p.k), *outs)
        sync()
        p.check(outs, norm)


def test_offsets_beyond_32_bits(api):
    """Tokens 2^31 elements apart, in place."""
    import torch
    p = Problem(api, case_of(T=3, hq=2, hk=1))
    stride = (1 << 31) + 64
    flat = torch.empty((2 * stride + 3 * 64,), dtype=torch.float16, device="cuda")
    q, k = flat.as_strided((3, 2, 64), (stride, 64, 1), 0), flat.as_strided((3, 1, 64), (stride, 64, 1), 128)
    q.copy_(dev(p.q))
    k.copy_(dev(p.k))
    p.call(q, k, q, k)
    sync()
    p.check([q.contiguous(), k.contiguous()])


def test_captured_and_replayed(api):
    import torch
    p = Problem(api, case_of(T=50, hq=12, hk=12))
    q, k, outs, eager = dev(p.q), dev(p.k), p.outs(), p.outs()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    sync()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            p.call(q, k, *outs, s=side.cuda_stream)
    for replay in range(3):
        p.q[:] = p.r.standard_normal(p.q.shape)
        p.positions[:] = p.r.integers(0, 5000, p.positions.shape)
        q.copy_(dev(p.q))
        p.fixed[5].copy_(dev(p.positions))
        for o in outs:
            o.fill_(-7)
        p.call(q, k, *eager)
        graph.replay()
        sync()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), replay
        p.check(outs)
    del graph


def test_the_turned_inner_product_depends_on_the_distance_only(api):
    """What the rotation is for: q at position m against k at position n gives the same as both moved on by the same distance."""
    T = 64
    p = Problem(api, case_of(T=T, hq=2, hk=2, dtype=np.float32, norm="none"))
    p.q[:], p.k[:] = p.q[:1], p.k[:1]
    for shift in (1000, 70000):
        p.positions[0] = np.arange(T)
        p.positions[0, T // 2:] += shift - T // 2
        p.fixed[5].copy_(dev(p.positions))
        outs = p.outs()
        p.call(dev(p.q), dev(p.k), *outs)
        sync()
        q, k = (host(o)[:T].astype(np.float64) for o in outs)
        near, far = (np.einsum("thd,uhd->htu", q[s], k[s]) for s in (slice(0, T // 2), slice(T // 2, T)))
        # 64 products of values off by 8.6 steps of |a| + |b| each
        bound = 2 * 8.6 * STEP * 4 * (np.abs(p.q[0]).max() * np.abs(p.k[0]).sum(-1)).max() * 2
        assert np.abs(near - far).max() <= bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 255, 1000])
@pytest.mark.parametrize("hq,hk,d,rotary,norm", [(1, 0, 64, 64, "rms"), (0, 1, 64, 64, "layer"), (1, 0, 256, 256, "rms"), (1, 0, 7, 2, "layer"),
                                                 (0, 1, 32, 0, "rms"), (1, 0, 2, 2, "none")])
def test_one_head_in_all(api, dtype, T, hq, hk, d, rotary, norm):
    """Each row of a workgroup is a token of its own, with angles of its own."""
    run(api, dtype=dtype, T=T, hq=hq, hk=hk, d=d, rotary=rotary, norm=norm)
