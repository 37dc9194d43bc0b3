"""Which kernel a token-scaled INT8 layer's sizes lead to, asked of the launcher itself (include/trtamd_test_hooks.h); no launch is made."""
import pytest

from tensorrt_amd import capi

LINEAR = 0
# the plans (TRTAMD_LINEAR_PLAN) that have a kernel: rows of whole lines of 128 bytes, rows that end within a line
KERNELS = {1536: {2, 4, 5, 8, 9, 10, 11, 12, 13, 14}, 1472: {1, 2, 3, 4, 8, 9, 10, 11, 12}}
LARGER_TILES = {10, 11, 12}  # 256 x 256, 256 x 192, 128 x 192: of rows that end within a line only these layers have them


def plan(T, K, N, gelu=0):
    return capi.api().test_token_linear_plan(T, K, N, gelu)


def other_plan(T, K, N, gelu=0):
    return capi.api().test_linear_plan(LINEAR, T, K, N, gelu)


@pytest.fixture
def forced():
    api = capi.api()
    yield lambda n: api.check(api.test_set_tuning(b"TRTAMD_LINEAR_PLAN", n))
    api.check(api.test_reset_tuning(b"TRTAMD_LINEAR_PLAN"))


def test_sizes_that_no_layer_has():
    for sizes in ((0, 64, 32), (1, 0, 32), (1, 96, 32), (1, 64, 0), (1, 64, 48), (-1, 64, 32)):
        assert plan(*sizes) == -1


@pytest.mark.parametrize("K", KERNELS)
def test_a_plan_is_taken_where_it_has_a_kernel_and_passed_over_where_not(forced, K):
    chosen = plan(130, K, 96)
    for n in range(0, 16):
        forced(n)
        assert plan(130, K, 96) == (n if n in KERNELS[K] else chosen), n


@pytest.mark.parametrize("T,K,N", [(33289, 960, 4096), (33289, 704, 2816), (33289, 4032, 1024), (16384, 960, 4096), (16384, 704, 2816),
                                   (8000, 960, 1056), (8000, 576, 2304), (4963, 576, 2304), (4963, 4032, 1024)])
@pytest.mark.parametrize("gelu", [0, 1])
def test_many_tokens_with_rows_that_end_within_a_line(T, K, N, gelu):
    """The tiles that shorten these layers most (33289 x 960 -> 4096: 247 us without them, 157 with); with GELU those of 128 x 256 are as
    good where there are several rounds of them."""
    assert plan(T, K, N, gelu) in LARGER_TILES | ({1} if gelu and T > 16384 else set())
    assert other_plan(T, K, N, gelu) not in LARGER_TILES


@pytest.mark.parametrize("T,K,N,gelu,want", [(1, 192, 1056, 0, 9), (8, 960, 4096, 1, 9), (40, 4032, 1024, 0, 9), (300, 960, 1056, 0, 8),
                                             (130, 704, 2816, 1, 4), (300, 960, 4096, 0, 3), (1000, 960, 4096, 1, 2), (33191, 704, 384, 0, 1)])
def test_each_plan_of_rows_that_end_within_a_line_has_its_sizes(T, K, N, gelu, want):
    assert plan(T, K, N, gelu) == want


@pytest.mark.parametrize("T,K,N,gelu", [(1, 1024, 4096, 1), (40, 4096, 1024, 0), (777, 4096, 1024, 0), (4963, 768, 2304, 0),
                                        (33289, 1024, 4096, 1), (33289, 1024, 1024, 0)])
def test_rows_of_whole_lines_take_the_other_layers_plans(T, K, N, gelu):
    assert plan(T, K, N, gelu) == other_plan(T, K, N, gelu)


@pytest.mark.parametrize("T,K,N,gelu", [(5003, 960, 1056, 0), (4963, 704, 2816, 1), (16384, 4032, 1024, 0), (33289, 960, 4096, 0)])
def test_choices_are_remembered_apart(T, K, N, gelu):
    """The two kinds of layers at the same sizes differ here, in either order, and are worked out once each."""
    first = plan(T, K, N, gelu), other_plan(T, K, N, gelu)
    assert first[0] in LARGER_TILES and first[1] not in LARGER_TILES
    before = capi.api().test_linear_estimates()
    for _ in range(3):
        assert (other_plan(T, K, N, gelu), plan(T, K, N, gelu)) == first[::-1]
        assert (plan(T, K, N, gelu), other_plan(T, K, N, gelu)) == first
    assert capi.api().test_linear_estimates() == before


@pytest.mark.parametrize("T,K,N", [(30413, 192, 1888), (20637, 192, 3104), (11369, 192, 3488), (16384, 64, 1024), (33289, 64, 512)])
def test_short_rows_without_gelu_do_not_go_in_tiles_of_128_x_256(T, K, N):
    """Of these it took 59, 56 and 33 us where the best of the others took 31, 33 and 22."""
    assert plan(T, K, N) != 1


def test_a_plan_that_the_other_layers_lack_is_not_theirs(forced):
    for n in LARGER_TILES:
        forced(n)
        assert plan(5003, 960, 1056) == n and other_plan(5003, 960, 1056) not in LARGER_TILES
        assert plan(5003, 960, 1056) == n


def test_results_that_layers_gain_by_go_past_the_last_level_cache():
    """Layers of both kinds of feed-forward layers, projection, quantisers and norms: 0.7 to 4 % shorter with them past the cache."""
    streams = capi.api().test_token_linear_streams
    for T, K, N in ((33289, 1024, 4096), (24000, 1024, 4096), (16384, 1024, 4096), (15000, 1024, 4096), (33289, 768, 2304), (30000, 768, 2304),
                    (26000, 768, 2304), (33289, 512, 2048), (40000, 512, 2048), (30000, 512, 2048), (33289, 4096, 1024), (33289, 1024, 1024)):
        assert streams(T, K, N), (T, K, N)


def test_results_that_layers_lose_by_stay_in_the_caches():
    """The same at fewer tokens: 0.5 to 1.3 % longer past the cache."""
    streams = capi.api().test_token_linear_streams
    for T, K, N in ((9000, 1024, 4096), (10000, 1024, 4096), (11000, 1024, 4096), (12000, 1024, 4096), (20000, 512, 2048), (24000, 512, 2048),
                    (24000, 1024, 1024), (28000, 1024, 1024), (4963, 768, 2304), (1, 64, 32)):
        assert not streams(T, K, N), (T, K, N)
