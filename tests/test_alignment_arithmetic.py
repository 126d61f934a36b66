"""The arithmetic of the fp32 attention operators, in numpy: an fp32 value as three bf16 numbers, a product as six of theirs
(csrc/cross_attention.h).  What the kernels make of it: tests/test_gpu_alignment_edges.py."""
import numpy as np
import pytest

BF16_MAX = np.float32(3.3895313892515355e38)


def nearest_bf16(x):
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def planes(x):
    a = nearest_bf16(np.clip(x, -BF16_MAX, BF16_MAX))
    b = nearest_bf16(x - a)
    return a, b, nearest_bf16((x - a) - b)


def values():
    rng = np.random.default_rng(3)
    ones = (0x3F800000 + (np.arange(128, dtype=np.uint32) << 16) + 0xFFFF).view(np.float32)        # every top half, its rest all ones
    edges = np.array([0x3F80FF7F, 0x3F808000, 0x3F807FFF, 0x3F80FF80, 0x3F800001, 0x3FFFFFFF, 0x7F7FFFFF, 0xFF7FFFFF, 0x7F7F8000, 0x7F7F7FFF,
                      0x00000000, 0x80000000], dtype=np.uint32).view(np.float32)
    return np.concatenate([ones, edges, rng.standard_normal(200000).astype(np.float32), (rng.standard_normal(1000) * 1e30).astype(np.float32)])


def test_three_planes_hold_an_fp32_value():
    x = values()
    a, b, c = planes(x)
    assert np.array_equal(a.astype(np.float64) + b + c, x.astype(np.float64))
    size = np.abs(x.astype(np.float64))
    inside = size <= BF16_MAX
    assert (np.abs(b) <= 2.0 ** -8 * size)[inside].all() and (np.abs(c) <= 2.0 ** -17 * size)[inside].all()


@pytest.mark.parametrize("order", [0, 1])
def test_six_products_are_the_product(order):
    """to 2^-24 of it, and not to one side"""
    x = values()
    x = x[np.abs(x) < 1e18]
    x = x[x != 0]
    y = x if order == 0 else np.random.default_rng(4).permutation(x)
    (a, b, c), (p, q, r) = [[t.astype(np.float64) for t in planes(v)] for v in (x, y)]
    exact = x.astype(np.float64) * y
    off = ((a * p + (a * q + b * p) + (a * r + b * q + c * p)) - exact) / exact
    assert np.abs(off).max() <= 2.0 ** -24 + 2.0 ** -34
    if order == 1:
        assert abs(off[140:].mean()) <= 2.0 ** -24 / 1000              # 2e5 pairs: deviation 2^-24 / 5, of the mean 2^-24 / 2000
