"""CPU-only: which kernels a product of given sizes runs (tests/_fp4_routes.py)."""
import pytest

import duqlinear4bitcuda_b200.lib as L
from tests import _fp4_routes as R


def pair_columns(m, n, k, sms=R.SMS):
    return L.cdll.duq4_linear_fp4_pair_columns(m, n, k, sms)


def tiles(m, n):
    return -(-m // 256) * -(-n // 256)


@pytest.mark.parametrize("m,n,k", R.PAIR_ROUNDS)
def test_pair_rounds(m, n, k):
    assert pair_columns(m, n, k) == n and tiles(m, n) > 3 * (R.SMS // 2) and -(-k // 256) > 6


@pytest.mark.parametrize("m,n,k", R.TWO_LAUNCHES)
def test_two_launches(m, n, k):
    n0 = pair_columns(m, n, k)
    assert 0 < n0 < n and n0 % 256 == 0


@pytest.mark.parametrize("m,n,k", R.FEW_TOKEN_BLOCKS)
def test_few_token_blocks(m, n, k):
    assert m > 128 and pair_columns(m, n, k) == 0


@pytest.mark.parametrize("m,n,k", R.PAIR_ONE_ROUND)
def test_pair_one_round(m, n, k):
    assert pair_columns(m, n, k) == n and tiles(m, n) <= R.SMS // 2


def test_row_alignments_are_all_there():
    assert {32 if 2 * n % 32 == 0 else 16 if 2 * n % 16 == 0 else 2 for _, n, _ in R.PAIR_ROUNDS} == {32, 16, 2}


def test_bounds():
    assert all(pair_columns(m, 4096, 4096) == 0 for m in (0, 1, 128)) and pair_columns(4096, 28672, 8192) == 28672
    assert pair_columns(300, 0, 64) == pair_columns(300, 64, 0) == pair_columns(300, 64, 64, 1) == pair_columns(300, 0x80000000, 64) == 0
    assert pair_columns(0x7FFFFFFF, 64, 64) == 64      # more blocks of 128 tokens than the other kernel's grid takes
    for m in (129, 1000, 5000):                        # never a strip of no columns, whatever the GPU
        for n in (1, 255, 256, 257, 9473, 30000):
            for k in (32, 2048, 8224):
                for sms in (2, 132, 148, 160):
                    n0 = pair_columns(m, n, k, sms)
                    assert n0 in (0, n) or (n0 % 256 == 0 and 0 < n0 < n)


def test_selftest_refuses():
    assert L.cdll.duq4_fp4_wait_selftest(None, None) == -1 and L.cdll.duq4_fp4_wait_selftest(0x1002, None) == -5
