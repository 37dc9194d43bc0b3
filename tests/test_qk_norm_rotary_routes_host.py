"""Which kernel a norm-and-rotation call leads to, asked of the launcher itself (include/trtamd_test_hooks.h); no launch is made, and no
address is read."""
import ctypes as C

import pytest

from tensorrt_amd import capi

FP32, FP16 = 0, 1
A = 0x10000  # an aligned address


def route(dtype, T, heads, d, rotary, adjacent=0, norm=1, **change):
    """(values a load, lanes a head, whether the stores go past the caches) of packed Q and K of `heads` heads each."""
    stride = dict(q_token_stride=3 * heads * d, q_head_stride=3 * d, k_token_stride=3 * heads * d, k_head_stride=3 * d,
                  q_out_token_stride=heads * d, q_out_head_stride=d, k_out_token_stride=heads * d, k_out_head_stride=d)
    f = dict(q=A, k=A + (1 << 40), q_out=A + (2 << 40), k_out=A + (3 << 40), T=T, q_heads=heads, k_heads=heads, d=d, norm=norm, eps=1e-6,
             q_weight=A, k_weight=A, q_bias=A, k_bias=A, rotary_dim=rotary, adjacent_pairs=adjacent, frequencies=A, positions=A, axes=1)
    r = capi.api().test_qk_norm_rotary_route(dtype, C.byref(capi.QkNormRotaryParams(**{**f, **stride, **change})))
    return r if r < 0 else (r & 255, r >> 8 & 255, r >> 16)


@pytest.mark.parametrize("dtype,d,rotary,adjacent,values,lanes", [
    (FP16, 64, 64, 0, 8, 4), (FP16, 128, 128, 0, 8, 8), (FP16, 32, 32, 0, 8, 2), (FP16, 80, 80, 0, 8, 8), (FP16, 72, 72, 0, 4, 16),
    (FP16, 72, 72, 1, 8, 8), (FP16, 72, 36, 0, 2, 16), (FP16, 64, 32, 0, 8, 4), (FP16, 256, 256, 0, 8, 16), (FP16, 63, 62, 0, 1, 8),
    (FP32, 64, 64, 0, 4, 8), (FP32, 80, 32, 1, 4, 16), (FP32, 32, 16, 0, 4, 4), (FP32, 10, 6, 0, 1, 8), (FP32, 256, 254, 0, 1, 32)])
def test_width_of_loads_and_lanes(dtype, d, rotary, adjacent, values, lanes):
    assert route(dtype, 100, 4, d, rotary, adjacent)[:2] == (values, lanes)


# A store instruction writes the rotated part and the rest of a head, and the first and second chunks of each, in places of their own:
# (type, head, rotated, adjacent) and the least of those rows in bytes.
SHORT = [(FP16, 64, 32, 0, 32), (FP16, 72, 36, 0, 8), (FP16, 80, 40, 0, 40), (FP16, 96, 48, 0, 48), (FP16, 48, 48, 0, 48),
         (FP16, 80, 32, 0, 32), (FP16, 128, 32, 0, 32), (FP16, 32, 32, 0, 32), (FP16, 32, 32, 1, 32), (FP32, 32, 16, 0, 32),
         (FP32, 64, 16, 0, 32), (FP16, 96, 32, 0, 32), (FP16, 48, 48, 1, 48), (FP16, 63, 62, 0, 2)]
HALF_LINES = [(FP16, 64, 64, 0), (FP16, 64, 64, 1), (FP32, 32, 32, 0), (FP32, 64, 32, 0), (FP16, 128, 64, 0), (FP16, 72, 72, 1)]
LONG = [(FP16, 72, 72, 0), (FP16, 80, 80, 0), (FP16, 80, 80, 1), (FP16, 96, 96, 0), (FP16, 128, 128, 0), (FP16, 128, 128, 1),
        (FP16, 256, 256, 0), (FP32, 64, 64, 0), (FP32, 80, 80, 0), (FP32, 128, 128, 1)]


@pytest.mark.parametrize("T", [1, 500, 4963, 33289])
@pytest.mark.parametrize("dtype,d,rotary,adjacent,row", SHORT)
def test_rows_below_64_bytes_go_through_the_caches(T, dtype, d, rotary, adjacent, row):
    """Past the caches they would reach the memory one by one, and take 5 to 40 % more."""
    assert row < 64 and route(dtype, T, 16, d, rotary, adjacent)[2] == 0


@pytest.mark.parametrize("dtype,d,rotary,adjacent", HALF_LINES)
def test_rows_of_64_bytes_go_past_the_caches_up_to_16_mib(dtype, d, rotary, adjacent):
    tokens = (16 << 20) // (2 * 16 * d * (2 if dtype == FP16 else 4))
    assert [route(dtype, T, 16, d, rotary, adjacent)[2] for T in (1, 500, tokens, tokens + 1, 33289)] == [1, 1, 1, 0, 0]


@pytest.mark.parametrize("T", [1, 500, 4963, 33289])
@pytest.mark.parametrize("dtype,d,rotary,adjacent", LONG)
def test_longer_rows_go_past_the_caches(T, dtype, d, rotary, adjacent):
    assert route(dtype, T, 16, d, rotary, adjacent)[2] == 1


def test_without_a_launch():
    assert route(FP16, 0, 4, 64, 64) == route(FP16, 8, 4, 64, 66) == route(2, 8, 4, 64, 64) == -1


def in_place(T, heads, d, token_stride, head_stride, dtype=FP16):
    """Q alone, in place."""
    p = capi.QkNormRotaryParams(q=A, q_out=A, q_token_stride=token_stride, q_head_stride=head_stride, q_out_token_stride=token_stride,
                                q_out_head_stride=head_stride, T=T, q_heads=heads, d=d, norm=1, q_weight=A, rotary_dim=d, frequencies=A,
                                positions=A, axes=1)
    return capi.api().test_qk_norm_rotary_route(dtype, C.byref(p)), capi.api().last_error_str()


@pytest.mark.parametrize("T,heads,d,token_stride,head_stride", [
    (4, 2, 64, 64, 0), (4, 1, 64, 0, 64), (4, 1, 64, 32, 0), (1, 3, 64, 999, 63), (4, 4, 64, 64, 64), (3, 5, 64, 320, 160 - 1),
    (9, 2, 64, 64, 8 * 64), (3, 3, 64, -64, 128), (2, 2, 64, 1 << 62, (1 << 62) + 32), (4, 2, 64, -64, 0), (1000, 3, 64, 100, 50)])
def test_heads_that_overlap_are_refused_in_place(T, heads, d, token_stride, head_stride):
    """One would be read after another has been written over it."""
    status, text = in_place(T, heads, d, token_stride, head_stride)
    assert status == -1 and "overlap" in text


@pytest.mark.parametrize("T,heads,d,token_stride,head_stride", [
    (4, 2, 64, 128, 64), (4, 2, 64, 384, 192), (4, 2, 64, 64, 256), (4, 1, 64, 64, 0), (1, 4, 64, 0, 64), (1, 1, 64, 0, 0), (3, 2, 64, 128, 192),
    (8, 2, 64, 64, 8 * 64), (4, 2, 64, -128, 64), (4, 2, 64, -128, -64), (2, 2, 64, 1 << 62, (1 << 62) + 64), (5, 5, 64, 5 * 64, 64)])
def test_heads_side_by_side_are_taken_in_place(T, heads, d, token_stride, head_stride):
    assert in_place(T, heads, d, token_stride, head_stride)[0] > 0


def test_heads_that_overlap_may_be_read():
    assert route(FP16, 8, 4, 64, 64, k_head_stride=0)[0] == route(FP16, 8, 4, 64, 64, q_token_stride=0, q_head_stride=0)[0] == 8


def test_pointers_that_are_not_used_may_be_anything():
    odd = A + 1
    assert route(FP16, 8, 4, 64, 64, norm=0, q_weight=odd, k_weight=odd, q_bias=odd, k_bias=odd)[0] == 8
    assert route(FP16, 8, 4, 64, 64, norm=1, q_bias=odd, k_bias=odd)[0] == 8
    assert route(FP16, 8, 4, 64, 0, norm=1, frequencies=odd, positions=odd)[0] == 8
    assert route(FP16, 8, 4, 64, 64, norm=2, q_bias=odd) == route(FP16, 8, 4, 64, 64, norm=1, k_weight=odd) == -1
