"""qv_mm8 with so many column blocks in a CTA that every ring (tiles, accumulators, scale slots) goes round
more than twice, in each of its kernels."""
import numpy as np
import pytest

from oracle import eight_bit as E

from .test_eight_bit import F32, _codes, _mm8

# ring stages, accumulators, CTAs an SM
FEW = {16: (6, 4, 2), 32: (5, 4, 2), 64: (4, 2, 2), 128: (6, 2, 1)}
MANY = (4, 2)
SMS = 148
SIZES = [(9, 20480, 300), (20, 16384, 300), (50, 16384, 301), (100, 16384, 300), (300, 16384, 301),
         (300, 5120, 13000), (2000, 2064, 5001)]


def fewest_blocks(tokens, width, rows):
    """Column blocks that go through the rings of the CTA with the fewest, and the slots of those rings."""
    blocks, row_tiles = -(-width // 128), -(-rows // 128)
    if tokens > 128 and -(-tokens // 128) * row_tiles > SMS:
        stages, buffers = MANY
        return -(-tokens // 128) * -(-rows // 256) // SMS * blocks, stages + buffers
    nt = next(n for n in (16, 32, 64, 128) if tokens <= n or n == 128)
    stages, buffers, ctas = FEW[nt]
    splits = max(1, min(6, SMS * ctas // (row_tiles * -(-tokens // nt)), blocks // 4))
    return blocks // splits, stages + buffers


@pytest.mark.parametrize('tokens,width,rows', SIZES)
def test_the_sizes_go_round_the_rings(tokens, width, rows):
    blocks, slots = fewest_blocks(tokens, width, rows)
    assert blocks > 2 * slots


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,width,rows', SIZES)
@pytest.mark.parametrize('whole', [True, False], ids=['whole numbers', 'every code'])
def test_mm8_on_every_lap_of_its_rings(hot, tokens, width, rows, whole):
    """Small whole numbers with powers of two as scales, where no sum is rounded, and codes of every size."""
    rng = np.random.default_rng(7700 + tokens + width + rows + whole)
    blocks = -(-width // 128)
    codes, weights = _codes(rng, (tokens, width), not whole), _codes(rng, (rows, width), not whole)
    if whole:
        scales = np.exp2(rng.integers(-3, 2, size=(blocks, tokens))).astype(np.float32)
        weight_scales = np.exp2(rng.integers(-3, 2, size=(-(-rows // 128), blocks))).astype(np.float32)
    else:
        scales = (0.5 + rng.random((blocks, tokens))).astype(np.float32) * np.float32(0.01)
        weight_scales = (rng.random((-(-rows // 128), blocks)) - 0.5).astype(np.float32)
    got = _mm8(hot, codes, scales, weights, weight_scales)
    want, size = E.product(codes, scales, weights, weight_scales)
    if whole:                                            # sums below 2^24 of their smallest step, 2^-6
        assert size.max() < 2.0 ** 18 and np.array_equal(got, want)
    else:                                                # 128 products, the blocks, at most 6 splits and two scales
        assert (np.abs(got - want) <= (128 + blocks + 6 + 2) * F32 * size).all()
    again = _mm8(hot, codes, scales, weights, weight_scales)
    assert np.array_equal(got, again)
