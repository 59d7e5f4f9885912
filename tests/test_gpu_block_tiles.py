"""The feed-forward block's tiled products by the tiles they take: lbk_product_tiling says which, the sizes here reach every one of
them, whole and with the summed dimension split, with remainders in every direction, in each product's layout. The CPU checks that
they do, so that another choice of tiles cannot leave one untested."""
import ctypes

import pytest
import torch

import test_gpu_block_ffn as ffn
from loopback_amd import block_ops as ops

SHAPES = {0: "128 x 128", 1: "256 x 256", 2: "192 x 256"}
# columns, rows, summed: the tiles, and whether the sum is split
PLAIN = {(129, 300, 71): (0, False), (56, 125, 523): (0, True), (8087, 1405, 331): (1, False), (247, 6397, 16391): (1, True),
         (408, 7293, 8203): (1, True), (920, 8317, 73): (2, False), (151, 8317, 4109): (2, True)}
# tokens, inner, width: the tiles of the gate and up projection and of the two's gradients
GATED = {(300, 152, 200): (0, 0), (6013, 665, 201): (1, 0), (8317, 919, 2057): (0, 1)}


def tiling(product, columns, rows, summed):
    splits = ctypes.c_int(-1)
    return ops.LIB.lbk_product_tiling(product, columns, rows, summed, ctypes.byref(splits)), splits.value


def test_every_tiling_is_reached():
    assert set(PLAIN.values()) == {(s, split) for s in SHAPES for split in (False, True)}
    for sizes, (shape, split) in PLAIN.items():
        got, splits = tiling(0, *sizes)
        assert (got, splits > 1) == (shape, split) and (ops.LIB.lbk_linear_scratch(*sizes) > 0) == split, sizes
    assert {a for a, _ in GATED.values()} == {b for _, b in GATED.values()} == {0, 1}
    for (t, n, d), want in GATED.items():
        assert (tiling(1, 2 * n, t, d), tiling(2, n, t, d)) == tuple((s, 1) for s in want), (t, n, d)


def test_tiling_refuses():
    null, s = ops.LIB.lbk_product_tiling, ctypes.c_int()
    for bad, code in (((-1, 8, 8, 8), -1), ((3, 8, 8, 8), -1), ((0, 0, 8, 8), -2), ((0, 8, 0, 8), -2), ((0, 8, 8, 0), -2), ((1, 7, 8, 8), -2)):
        assert null(*bad, ctypes.byref(s)) == code
    assert null(0, 8, 8, 8, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", PLAIN)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_plain_products(sizes, dtype):
    """Forward, input gradient and weight gradient: one rounding of the fp32 sum, the same bits twice, nothing past the result."""
    ffn.test_products(*sizes, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", GATED)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_products(sizes, dtype, act):
    """The block and its gradients, with both gated products' tiles among the sizes."""
    t, n, d = sizes
    ffn.check(t, d, n, d, dtype, act)
