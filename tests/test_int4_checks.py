"""Checks of the 4-bit operators' C entry points that need no GPU: what is refused is refused before anything is launched."""
import ctypes

import pytest

from carbon_engine_b200 import ops_int4
from carbon_engine_b200.csrc.kernel_lib import KernelError, kernels

ERR_SIZE = -1
ADDR = 1 << 20                     # an aligned address that nothing reads


def attention(n=1, window=0, splits=1, share=1):
    """32 heads over 8 of 128, groups of 64, pages of 64 tokens."""
    return kernels().ce_int4_attention(ops_int4._ATTENTION(1, ADDR, 4096, ADDR, ADDR, ADDR, ADDR, ADDR, ADDR, ADDR, 0, n, 32, 8, 128, 64, 64, 200, 1000,
                                                           window, splits, share, ADDR, ADDR, 0.1, 0))


@pytest.mark.parametrize("splits,share", [(64, 1 << 26), (2, 1 << 30), (1, 1 << 31), (1, -1), (48, 1 << 40), (1, 1 << 62)])
def test_shares_of_keys_that_32_bits_do_not_count_are_refused(splits, share):
    """A block's first tile is its number times the share: beyond 31 bits it would lie before the first."""
    assert attention(splits=splits, share=share) == ERR_SIZE


@pytest.mark.parametrize("max_ctx", [1, 8192, 1 << 31, 1 << 36, 1 << 40, (1 << 63) - 1])
@pytest.mark.parametrize("window", [0, 100, 1 << 40])
@pytest.mark.parametrize("jobs", [1, 8, 512])
def test_a_bound_on_the_keys_may_be_any_number(max_ctx, window, jobs):
    splits, share = ops_int4._shares(jobs, max_ctx, window, 1)
    assert 1 <= splits <= 64 and 1 <= share and splits * share < 1 << 30
    tiles = -(-min(max_ctx, (1 << 31) - 1, window + 16 if window else max_ctx) // 16)
    assert splits * share >= tiles


def kv(fn, T=1, page_size=16, max_pages=4, num_pages=8):
    return fn(ops_int4._KV(1, ADDR, ADDR, 64, 64, 64, 64, ADDR, ADDR, ADDR, ADDR, ADDR, ADDR, T, 1, 64, 32, page_size, max_pages, num_pages, 0))


def product(M=2, N=40, K=128, ldo=40):
    return kernels().ce_int4_gemm(ops_int4._GEMM(1, ADDR, K, ADDR, ADDR, ldo, M, N, K, 64, 0, ADDR, ADDR, 0))


def test_sizes_beyond_32_bits_are_refused():
    """(Cut to 32 bits, each would be a size that is taken.)"""
    beyond = 1 << 32
    assert attention(window=beyond + 5) == ERR_SIZE and attention(n=beyond * 8 + 1) == ERR_SIZE
    for fn in (kernels().ce_int4_kv_write, kernels().ce_int4_kv_read):
        assert kv(fn, T=beyond + 1) == kv(fn, page_size=beyond + 16) == kv(fn, max_pages=beyond + 4) == kv(fn, num_pages=beyond + 8) == ERR_SIZE
    assert product(M=beyond + 2) == product(N=beyond + 40) == product(K=beyond + 128) == product(ldo=39) == ERR_SIZE
    for rows, width in ((1 << 30, 64), (64, 1 << 30), ((1 << 32) + 16, 64)):
        with pytest.raises(KernelError, match="2\\^30"):
            ops_int4.Int4Weight(rows, width, device="cpu")
