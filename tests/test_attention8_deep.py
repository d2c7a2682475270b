"""qv_attention8 where a CTA has several tiles and the running maximum moves inside it.

The maximum of a row moves when a tile's is more than 8 (log2 units, with the logarithm of the value
scale) above it; the sums and the output so far are then scaled down.  `moves` replays that rule on the
host, so that every test says how often it happens in its inputs.
"""
import numpy as np
import pytest

from oracle.hotpath import prepare_rows, sigmoid

from .test_attention8 import Layer

F32 = 2.0 ** -24
CTAS, TILE, THRESHOLD = 37, 64, 8.0


class Deep(Layer):
    """A Layer of several tiles a CTA, with scales that its subclasses' tests set before the call."""

    def __init__(self, batch, position, seed):
        super().__init__(batch, position, position // 64 * 64, 128, seed)
        self.total = -(-(position + batch) // TILE)
        self.per = -(-self.total // CTAS)                # tiles of a CTA

    def definition(self):
        """want, the sum of p |v|, the largest probability times value scale ([T][24]), the largest sum
        |q k| / 16, and every tile's largest score in log2 units with its value scale ([T][24][tiles])."""
        n = self.position + self.batch
        at = np.arange(self.packed, n) % self.tail
        tails = [t.cpu().numpy()[at].astype(np.float64) for t in self.d_tails]
        T = self.batch
        q = prepare_rows(self.q_gate[..., :256], self.q_norm, self.position + np.arange(T)[:, None], 1e-6)
        gate = sigmoid(self.q_gate[..., 256:].astype(np.float64))
        want, size = np.zeros((T, 24, 256)), np.zeros((T, 24, 256))
        largest, top, tiles = np.zeros((T, 24)), 0.0, np.full((T, 24, self.total), -np.inf)
        for h in range(24):
            g = h // 6
            k, v = (np.concatenate([(c[:, g] * s[:, g].astype(np.float64)[:, None, None]).reshape(-1, 256), t[:, g]])
                    for c, s, t in zip(self.codes, self.scales, tails))
            vs = np.concatenate([np.repeat(self.scales[1][:, g].astype(np.float64), 64), np.ones(n - self.packed)])
            vs_log2 = np.log2(np.maximum(vs, 2.0 ** -100))
            for t in range(T):
                m = self.position + t + 1
                s = k[:m] @ q[t, h] / 16
                top = max(top, float((np.abs(k[:m]) @ np.abs(q[t, h])).max()) / 16)
                p = np.exp(s - s.max())
                p /= p.sum()
                want[t, h], size[t, h] = p @ v[:m] * gate[t, h], p @ np.abs(v[:m]) * gate[t, h]
                largest[t, h] = (p * vs[:m]).max()
                padded = np.full(self.total * TILE, -np.inf)
                padded[:m] = s * np.log2(np.e) + vs_log2[:m]
                tiles[t, h] = padded.reshape(-1, TILE).max(1)
        return want, size, largest, top, tiles

    def moves(self, tiles):
        """Moves of a row's maximum behind its CTA's first tile: in even tiles, in odd tiles, and the tiles in
        which some rows of a K/V head move and others do not; then the largest move."""
        even = odd = mixed = 0
        largest = 0.0
        for first in range(0, self.total, self.per):
            part = tiles[..., first:first + self.per]
            top = part[..., 0].copy()
            for j in range(1, part.shape[-1]):
                moved = part[..., j] > top + THRESHOLD
                if moved.any():
                    finite = moved & np.isfinite(top)
                    largest = max(largest, float((part[..., j] - top)[finite].max(initial=0)))
                top = np.where(moved, part[..., j], top)
                if j & 1:
                    odd += int(moved.sum())
                else:
                    even += int(moved.sum())
                by_head = moved.reshape(self.batch, 4, 6).transpose(1, 0, 2).reshape(4, -1)
                mixed += int((by_head.any(1) & ~by_head.all(1)).sum())
        return even, odd, mixed, largest

    def check_output(self, got):
        want, size, largest, top, tiles = self.definition()
        even, odd, mixed, jump = self.moves(tiles)
        # Relative error of a probability: queries as fp16 hi + lo and their fp32 norm and rotation (24 steps),
        # products summed in fp32 (16 groups of a matrix instruction, hi + lo), the exponent's argument, the
        # SFU's 2^x and fp16 hi + lo (2^-22); twice, for the numerator and the sum.  A move scales by one more
        # 2^x, whose argument is off by half a step of the move.  The sums over the positions: in fp32 along a
        # CTA's tiles, the splits and the instruction's groups of 16.
        rel = 2 * (top * (24 + 32 + 4) + 16 + self.per * (4 + jump)) * F32 + (self.per + CTAS + 16) * 4 * F32
        # fp16 hi + lo resolve 2^-25, where the largest probability times value scale of a row is 2^6 or more
        n = self.position + self.batch
        floor = n * 127 * 2.0 ** -31 * largest[..., None] * np.ones(256)
        assert (np.abs(got - want) <= rel * size + floor).all(), np.abs(got - want).max()
        return even, odd, mixed


@pytest.mark.gpu
@pytest.mark.parametrize('position', [9000, 13005])
def test_scores_that_rise_inside_a_cta(hot, position):
    """Each tile's scores are some times larger than those of the tile before, in every CTA."""
    layer = Deep(3, position, 9300 + position)
    step = np.arange(position // 64) % layer.per
    layer.scales[0][:] = (2.0 ** -5 * np.array([1, 4, 10, 18, 27, 38])[step])[:, None].astype(np.float32)
    even, odd, mixed = layer.check_output(layer.run(hot))
    assert layer.per >= 4 and even > 500 and odd > 1000


@pytest.mark.gpu
@pytest.mark.parametrize('when', [0, 1])
def test_one_tile_in_two_rises(hot, when):
    """Large scores in the even (odd) tiles only: the other warp of a row carries the maximum on."""
    layer = Deep(2, 13001, 9400 + when)
    step = np.arange(13001 // 64) % layer.per
    layer.scales[0][:] = np.where(step % 2 == when, 2.0 ** -4 * (1 + 4 * step), 2.0 ** -6)[:, None].astype(np.float32)
    even, odd, mixed = layer.check_output(layer.run(hot))
    assert (even > 800 and odd < 200) if when == 0 else (odd > 800 and even < 200)


@pytest.mark.gpu
@pytest.mark.parametrize('batch', [1, 5, 10])
def test_some_rows_of_a_warp_move_and_others_do_not(hot, batch):
    """Key and value scales of every size: rows move at different tiles."""
    rng = np.random.default_rng(9500 + batch)
    layer = Deep(batch, 11003, 9500 + batch)
    blocks = len(layer.scales[0])
    layer.scales[0][:] = np.exp2(rng.uniform(-6, -2, (blocks, 4))).astype(np.float32)
    layer.scales[1][:] = np.exp2(rng.uniform(-9, 1, (blocks, 4))).astype(np.float32)
    even, odd, mixed = layer.check_output(layer.run(hot))
    assert layer.per >= 4 and even > 60 * batch and odd > 120 * batch and mixed > 40


@pytest.mark.gpu
def test_blocks_of_zeros_inside_a_cta(hot):
    """Values of zero have no logarithm: the tiles behind them raise the maximum by far more than fp16's range."""
    layer = Deep(4, 12000, 9600)
    step = np.arange(12000 // 64) % layer.per
    layer.codes[1][step == 0], layer.scales[1][step == 0] = 0, 0
    layer.codes[1][(step == 2)], layer.scales[1][step == 2] = 0, 0
    layer.codes[0][7:11], layer.scales[0][7:11] = 0, 0
    even, odd, mixed = layer.check_output(layer.run(hot))
    assert odd > 3000


@pytest.mark.gpu
def test_a_scale_that_is_nan_inside_a_cta_reaches_its_head_alone(hot):
    layer = Deep(2, 12000, 9700)
    layer.scales[0][layer.per * 3 + 2, 0] = np.nan
    layer.scales[1][layer.per * 5 + 1, 3] = np.nan
    got = layer.run(hot)
    bad = np.zeros((2, 24, 256), bool)
    bad[:, 0:6], bad[:, 18:24] = True, True
    assert np.array_equal(np.isnan(got), bad)
