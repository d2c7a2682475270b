"""qv_mm8 with scales of any fp32 size: their product may leave fp32 where a term or the output does not."""
import numpy as np
import pytest

from oracle import eight_bit as E

from .test_eight_bit import F32, _codes, _mm8

# one size for each kernel: 16, 32, 64, 128 tokens a tile, and the one for many tiles
SIZES = [(3, 300), (20, 300), (50, 131), (100, 300), (131, 19100)]


def _scales(rng, shape):
    """Mantissas in [1, 2) times powers of two over all of fp32's range, subnormal numbers among them."""
    with np.errstate(over='ignore'):
        s = ((1 + rng.random(shape)) * np.exp2(rng.integers(-149, 127, size=shape).astype(np.float64))).astype(np.float32)
    return s * rng.choice([-1, 1], size=shape).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize('width', [128, 700])
@pytest.mark.parametrize('tokens,rows', SIZES)
def test_scales_of_every_size(hot, tokens, rows, width):
    rng = np.random.default_rng(7900 + tokens + width)
    blocks = -(-width // 128)
    width = -(-width // 16) * 16
    codes, weights = _codes(rng, (tokens, width), True), _codes(rng, (rows, width), True)
    codes[0] = 0                                         # sums of zero stay zero
    codes[1, 1:], weights[1, 1:] = 0, 0                  # and the smallest product, 2^-18
    codes[1, 0], weights[1, 0] = 1, 1
    scales, weight_scales = _scales(rng, (blocks, tokens)), _scales(rng, (-(-rows // 128), blocks))
    want, size = E.product(codes, scales, weights, weight_scales)
    got = _mm8(hot, codes, scales, weights, weight_scales).astype(np.float64)
    assert not got[0].any()
    # 128 products, the blocks, at most 6 splits; the factor of a block is rounded, its product with the sum,
    # and a result among the subnormal numbers at each of its additions by half their step
    bound = (128 + blocks + 6 + 3) * F32 * size + (blocks + 6) * 2.0 ** -150
    inside = size < 2.0 ** 127
    assert (np.abs(got - want) <= bound)[inside].all()
    assert (np.abs(got[1]) > 0)[inside[1] & (size[1] > 2.0 ** -140)].any()
    # terms beyond fp32: infinity with their sign, where no other term could meet them
    if blocks == 1:
        far = np.abs(want) > 2.0 ** 128 * (1 + 2.0 ** -10)
        assert far.any() and np.array_equal(got[far], np.copysign(np.inf, want[far]))


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,rows', SIZES)
def test_products_of_scales_at_the_ends_of_fp32(hot, tokens, rows):
    """One term for each output, of an exact value: 2^100 * 2^30 * 2^-18, and 2^-100 * 1.5 2^-40 * 2^16."""
    codes, weights = np.zeros((tokens, 256), np.uint8), np.zeros((rows, 256), np.uint8)
    one = {v: int(np.flatnonzero(E.e4m3_values() == v)[0]) for v in (2.0 ** -9, 256.0)}
    codes[::2, 5], codes[1::2, 5] = one[2.0 ** -9], one[256.0]
    weights[:, 5] = np.where(np.arange(rows) // 128 % 2 == 0, one[2.0 ** -9], one[256.0])
    scales, weight_scales = np.ones((2, tokens), np.float32), np.ones((-(-rows // 128), 2), np.float32)
    scales[0, ::2], scales[0, 1::2] = 2.0 ** 100, 2.0 ** -100
    weight_scales[::2, 0], weight_scales[1::2, 0] = 2.0 ** 30, 1.5 * 2.0 ** -40
    want, _ = E.product(codes, scales, weights, weight_scales)
    assert np.abs(want).max() == 2.0 ** 112 and np.abs(want).min() == 1.5 * 2.0 ** -124
    assert np.array_equal(_mm8(hot, codes, scales, weights, weight_scales), want)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,rows', SIZES)
def test_infinite_scales_keep_to_their_tokens_and_rows(hot, tokens, rows):
    rng = np.random.default_rng(7950 + tokens)
    codes, weights = _codes(rng, (tokens, 256), False), _codes(rng, (rows, 256), False)
    codes[2, 128:] = 0                                   # a sum of zero: no number
    scales, weight_scales = np.ones((2, tokens), np.float32), np.ones((-(-rows // 128), 2), np.float32)
    scales[1, 1:3] = np.inf, -np.inf
    weight_scales[1, 0] = -np.inf
    with np.errstate(invalid='ignore'):
        want, _ = E.product(codes, scales, weights, weight_scales)
    got = _mm8(hot, codes, scales, weights, weight_scales)
    assert np.isnan(want[2]).all() and np.isinf(want[1]).any() and np.isfinite(want[0, :128]).all()
    np.testing.assert_array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('block', [0, 17, 31])
@pytest.mark.parametrize('tokens,rows', SIZES + [(300, 300)])
def test_one_far_block_among_ordinary_ones(hot, tokens, rows, block):
    """The width is long enough to be split: one CTA of a cluster sees the scale, all of them have outputs of
    it.  Every other token keeps the bits that it has in a call without that scale."""
    rng = np.random.default_rng(7980 + tokens + block)
    width, blocks = 4096, 32
    codes, weights = _codes(rng, (tokens, width), True), _codes(rng, (rows, width), True)
    scales = (0.5 + rng.random((blocks, tokens))).astype(np.float32) * np.float32(0.01)
    weight_scales = (rng.random((-(-rows // 128), blocks)) - 0.5).astype(np.float32)
    weight_scales[-1, block] = 1.25 * 2.0 ** -40
    far = tokens - 2
    codes[far] = 0
    codes[far, 128 * block + 7] = int(np.flatnonzero(E.e4m3_values() == 256.0)[0])
    plain = _mm8(hot, codes, scales, weights, weight_scales)
    scales[block, far] = 1.5 * 2.0 ** -100
    got = _mm8(hot, codes, scales, weights, weight_scales)
    assert np.array_equal(np.delete(got, far, 0), np.delete(plain, far, 0))
    want = (E.decode(weights[:, 128 * block + 7]) * 256 * scales[block, far].astype(np.float64)
            * weight_scales[np.arange(rows) // 128, block].astype(np.float64))
    # one product, its factor and its sums with zeros: three roundings, none where the value has few bits
    assert (np.abs(got[far] - want) <= 3 * F32 * np.abs(want)).all()
    last = (rows - 1) // 128 * 128
    assert (got[far, last:] == want[last:].astype(np.float32)).all() and got[far, last:].any()
