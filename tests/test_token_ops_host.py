"""What the token-scaled INT8 layers and the norm-and-rotation pass refuse, and that they do so before anything is
launched: no GPU is needed here, and no address that is given is ever read."""
import ctypes as C
import os
import re

import numpy as np
import pytest
from scipy.special import ndtr

import tensorrt_amd
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


def token(**change):
    f = dict(a=A, w=A, token_scale=A, channel_scale=A, bias=A, out=A, T=4, K=128, N=64, epilogue=0)
    f.update(change)
    return C.byref(capi.Int8TokenLinearParams(**f))


def dynamic(**change):
    f = dict(a=A, a_stride=128, w=A, channel_scale=A, bias=A, out=A, workspace=A, workspace_bytes=1 << 20, T=4, K=128, N=64,
             epilogue=0)
    f.update(change)
    return C.byref(capi.Int8DynamicLinearParams(**f))


def rotary(**change):
    f = dict(q=A, k=A, q_out=A, k_out=A, q_token_stride=192, q_head_stride=64, k_token_stride=192, k_head_stride=64,
             q_out_token_stride=192, q_out_head_stride=64, k_out_token_stride=192, k_out_head_stride=64,
             T=4, q_heads=1, k_heads=1, d=64, norm=1, eps=1e-6, q_weight=A, k_weight=A, q_bias=A, k_bias=A,
             rotary_dim=64, frequencies=A, positions=A, axes=1)
    f.update(change)
    return C.byref(capi.QkNormRotaryParams(**f))


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T=-1"), (dict(C=0), "C=0"), (dict(C=48), "multiple of 32"), (dict(stride=32), "stride"),
    (dict(stride=68), "stride"), (dict(x=0), "null"), (dict(out=0), "null"), (dict(scales=0), "null"), (dict(x=A + 2), "aligned"),
    (dict(out=A + 8), "aligned"), (dict(scales=A + 2), "aligned"), (dict(T=1 << 24), "2^24"), (dict(C=1 << 30, stride=1 << 30), "2^30")])
def test_quantiser_refuses(api, change, word):
    f = dict(T=3, C=64, x=A, stride=64, out=A, scales=A)
    f.update(change)
    refused(api, api.quantize_fp16_per_token(None, f["T"], f["C"], f["x"], f["stride"], f["out"], f["scales"]), word)


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T=-1"), (dict(K=0), "K=0"), (dict(K=96), "multiple of 64"), (dict(N=0), "N=0"), (dict(N=48), "of 32"),
    (dict(epilogue=2), "epilogue"), (dict(epilogue=3), "epilogue"), (dict(epilogue=7), "epilogue"), (dict(epilogue=-1), "epilogue"),
    (dict(a=0), "null"), (dict(w=0), "null"), (dict(token_scale=0), "null"), (dict(channel_scale=0), "null"), (dict(out=0), "null"),
    (dict(a=A + 8), "aligned"), (dict(w=A + 4), "aligned"), (dict(out=A + 2), "aligned"), (dict(channel_scale=A + 4), "aligned"),
    (dict(bias=A + 4), "aligned"), (dict(token_scale=A + 2), "aligned"),
    (dict(T=1 << 24), "2 GiB"), (dict(N=1 << 24), "2 GiB")])
def test_token_linear_refuses(api, change, word):
    refused(api, api.int8_token_linear(None, token(**change)), word, "int8_token_linear")


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T=-1"), (dict(K=96), "multiple of 64"), (dict(N=48), "of 32"), (dict(epilogue=2), "epilogue"),
    (dict(a=0), "null"), (dict(w=0), "null"), (dict(channel_scale=0), "null"), (dict(out=0), "null"), (dict(a=A + 4), "aligned"),
    (dict(a_stride=120), "stride"), (dict(a_stride=132), "stride"), (dict(workspace=0), "workspace"),
    (dict(workspace=A + 8), "workspace"), (dict(workspace_bytes=4 * 128), "workspace"), (dict(T=1 << 24, workspace_bytes=1 << 40), "2 GiB")])
def test_dynamic_linear_refuses(api, change, word):
    refused(api, api.int8_dynamic_linear(None, dynamic(**change)), word, "int8_dynamic_linear")


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "T=-1"), (dict(q_heads=-1), "q_heads=-1"), (dict(k_heads=-2), "k_heads=-2"), (dict(d=0), "d=0"), (dict(d=257), "d=257"),
    (dict(norm=3), "norm 3"), (dict(norm=-1), "norm -1"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(rotary_dim=66), "rotary_dim=66"), (dict(rotary_dim=31), "rotary_dim=31"), (dict(rotary_dim=-2), "rotary_dim=-2"),
    (dict(rotary_dim=0, norm=0), "neither"), (dict(q=0), "null"), (dict(k=0), "null"), (dict(q_out=0), "null"), (dict(k_out=0), "null"),
    (dict(q_weight=0), "null"), (dict(k_weight=0), "null"), (dict(norm=2, k_bias=0), "null"), (dict(frequencies=0), "null"),
    (dict(positions=0), "null"), (dict(q=A + 1), "aligned"), (dict(k_out=A + 1), "aligned"), (dict(q_weight=A + 2), "aligned"),
    (dict(frequencies=A + 1), "aligned"), (dict(positions=A + 2), "aligned"), (dict(axes=0), "axes=0"), (dict(axes=5), "axes=5"),
    (dict(axes=2, sections=(16, 17)), "33 pairs"), (dict(axes=2, sections=(-1, 33)), "sections[0]"),
    (dict(axes=3, sections=(16, 33, 0)), "sections[1]"), (dict(axes=3, sections=(8, 12, 12), axes_cycled=1), "sections[1]"),
    (dict(q_out_token_stride=128), "in place"), (dict(k_out_head_stride=32, k_heads=2), "in place"),
    (dict(T=1 << 16, q_heads=512, k_heads=512), "2^26"), (dict(q_heads=(1 << 31) - 1, k_heads=(1 << 31) - 1), "2^26")])
def test_norm_rotary_refuses(api, change, word):
    sections = change.pop("sections", ())
    ref = rotary(**change)
    ref._obj.sections[:len(sections)] = sections
    refused(api, api.qk_norm_rotary(None, 1, ref), word)


def test_null_parameters_and_unknown_types(api):
    refused(api, api.int8_token_linear(None, None), "null")
    refused(api, api.int8_dynamic_linear(None, None), "null")
    refused(api, api.qk_norm_rotary(None, 1, None), "null")
    for data_type in (-1, 2, 3):
        assert api.qk_norm_rotary(None, data_type, rotary()) == 3
    # four-byte values need four-byte addresses, two-byte ones two
    refused(api, api.qk_norm_rotary(None, 0, rotary(q=A + 2)), "aligned")


def test_no_tokens_no_work(api):
    """Empty tensors have no address, and nothing is launched for them (there is no GPU here)."""
    assert api.quantize_fp16_per_token(None, 0, 64, None, 64, None, None) == 0
    assert api.int8_token_linear(None, token(T=0, a=0, token_scale=0, out=0)) == 0
    assert api.int8_dynamic_linear_workspace_size(0, 128, 64) == 0
    assert api.int8_dynamic_linear(None, dynamic(T=0, a=0, out=0, workspace=0, workspace_bytes=0)) == 0
    assert api.qk_norm_rotary(None, 1, rotary(T=0, q=0, k=0, q_out=0, k_out=0, positions=0)) == 0
    assert api.qk_norm_rotary(None, 1, rotary(q_heads=0, k_heads=0)) == 0
    # sizes are checked all the same
    refused(api, api.int8_token_linear(None, token(T=0, K=96)), "multiple of 64")
    refused(api, api.int8_dynamic_linear(None, dynamic(T=0, N=48)), "of 32")
    refused(api, api.quantize_fp16_per_token(None, 0, 48, None, 48, None, None), "multiple of 32")


def test_workspace_size(api):
    size = api.int8_dynamic_linear_workspace_size
    assert size(-1, 64, 32) == size(1, 0, 32) == size(1, 64, 0) == 0
    for T, K, N in ((1, 64, 32), (777, 4096, 1024), (33289, 1024, 4096)):
        assert size(T, K, N) >= T * K + 4 * T
        # what is one byte short is refused
        refused(api, api.int8_dynamic_linear(None, dynamic(T=T, K=K, N=N, a_stride=K, workspace_bytes=size(T, K, N) - 1)), "workspace")


def test_gelu_polynomial():
    """The polynomial of gelu_f16 as it stands in the source, evaluated in binary32 as the kernels do: what the layers' tolerances count on."""
    path = os.path.join(os.path.dirname(tensorrt_amd.__file__), "csrc", "token_ops.hpp")
    body = open(path).read().split("float gelu_f16(float y)")[1].split("return fmaf(-a")[0]
    c = [np.float32(v) for v in re.findall(r"(-?\d\.\d+e[-+]\d+)f", body)]
    assert len(c) == 6 and c[0] < 0
    y = np.linspace(-12, 12, 480001).astype(np.float32)
    a = np.abs(y).astype(np.float64)
    p = np.full(y.shape, c[0])
    for v in c[1:]:  # the products are exact in binary64, so this rounds once, as an fma
        p = (p.astype(np.float64) * a + np.float64(v)).astype(np.float32)
    got = np.maximum(y, 0).astype(np.float64) - a * np.exp2(p.astype(np.float64)).astype(np.float32)
    want = y * ndtr(y.astype(np.float64))
    assert (np.abs(got - want) <= np.where(np.abs(want) >= 2.0 ** -14, 8.5e-5 * np.abs(want), 5.2e-9)).all()
    # behind the interval the term vanishes
    far = 10.0 ** np.arange(1, 9)
    poly = np.polyval([float(v) for v in c], far)
    assert (poly < -70).all() and (np.diff(poly) < 0).all()


@pytest.mark.parametrize("T", [0, 1])
@pytest.mark.parametrize("K", [131072, 133184, 262144, (1 << 31) - 64])
def test_rows_whose_sums_could_pass_int32_are_refused(api, T, K):
    """131072 products of -128 and -128 are 2^31; 131008, the next shorter row, has sums of 2146435072 at most."""
    refused(api, api.int8_token_linear(None, token(T=T, K=K, N=32)), "131072", "int8_token_linear")
    ref = dynamic(T=T, K=K, N=32, a_stride=K, workspace_bytes=1 << 40)
    refused(api, api.int8_dynamic_linear(None, ref), "131072", "int8_dynamic_linear")
