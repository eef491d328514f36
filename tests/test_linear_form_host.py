"""CPU: which of its two forms the W8A8 linear takes shows in the workspace that it asks for."""

import pytest

OK = 4096


@pytest.mark.parametrize("N,K", [(151936, 4096), (24576, 4096), (12288, 12288), (49152, 1024)])
def test_partial_sums_never_outgrow_the_weights(lib, N, K):
    """Wide products of many rows go to tiles, and their workspace stays small (an LM head's
    256 rows took 622 MB)."""
    for M in (16, 32, 64, 128, 256):
        assert lib.s8b_linear_workspace_size(M, N, K) <= 256 + N * K // 4


@pytest.mark.parametrize("N,K", [(1024, 4096), (4096, 4096), (8192, 12288), (24576, 4096), (256, 1024)])
def test_a_workspace_serves_calls_of_fewer_rows(lib, N, K):
    sizes = [lib.s8b_linear_workspace_size(M, N, K) for M in range(1, 257)]
    assert sizes == sorted(sizes) and sizes[0] > 256
    assert sizes[15] == 256 + 16 * (sizes[0] - 256)  # up to 16 rows: always the split-K stream


def test_what_a_call_needs(lib):
    """A call of few rows is refused for less than its partial sums, one that is tiled for less than the
    status word."""
    def call(M, N, K, size):
        return lib.s8b_linear_w8a8(OK, OK, OK, OK, None, 0, None, OK, M, N, K, 0, OK, size, None)

    n = lib.s8b_linear_workspace_size(16, 151936, 4096)
    assert call(16, 151936, 4096, n - 1) == -7
    assert call(256, 151936, 4096, 255) == -7
    assert call(300, 4096, 4096, 255) == -7


@pytest.mark.parametrize("M,N,K", [(2 ** 31 - 1, 64, 16), (2 ** 31 - 100, 64, 128), (300, 2 ** 31 - 1, 16),
                                   (1, 2 ** 31 - 1, 128), (4, 2 ** 31 - 500, 128)])
def test_sides_whose_last_tile_passes_32_bits_are_refused(lib, M, N, K):
    assert lib.s8b_linear_w8a8(OK, OK, OK, OK, None, 0, None, OK, M, N, K, 0, OK, 2 ** 62, None) == -1
    assert lib.s8b_linear_workspace_size(M, N, K) == 256


@pytest.mark.parametrize("N,K", [(151936, 4096), (24576, 1024), (4096, 12288)])
def test_asking_for_the_size_is_quick(lib, N, K):
    """A call without a workspace asks every time: well below the launch's own host time."""
    import time

    took = []
    for _ in range(200):
        t = time.perf_counter()
        lib.s8b_linear_workspace_size(256, N, K)
        took.append(time.perf_counter() - t)
    assert min(took) < 20e-6
