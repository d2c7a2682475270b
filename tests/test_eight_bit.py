"""The 8-bit serving operators beside the attention: qv_norm8 / qv_quantize8, qv_mm8 and the
packing of the int8 K/V cache, against their definitions in 64 bits (oracle/eight_bit.py).

Rounding steps: fp32 2^-24, fp16 2^-11, e4m3 2^-4 of the value (2^-10 below its smallest
normal number), each half a step.
"""
import ctypes as ct

import numpy as np
import pytest

from oracle import eight_bit as E

F32, F16, E4M3 = 2.0 ** -24, 2.0 ** -11, 2.0 ** -4


# ------------------------------------------------------------------ refusals (no GPU)
def test_rejects_invalid_arguments_before_accessing_buffers(lib):
    v, odd = ct.c_void_p(4096), ct.c_void_p(4104)    # never dereferenced
    for tokens, width, eps in ((0, 128, 1e-6), (139265, 128, 1e-6), (1, 0, 1e-6), (1, 17409, 1e-6), (1, 128, 0.),
                               (1, 128, float('nan'))):
        assert lib.qv_norm8(v, v, v, v, v, v, v, tokens, width, eps, None) == -1
        assert lib.qv_error()
    for null in (0, 1, 4, 6):                         # codes, scales, x, weights
        args = [v] * 7
        args[null] = None
        assert lib.qv_norm8(*args, 1, 128, 1e-6, None) == -1
        assert lib.qv_error() == b'null normalization buffer'
    assert lib.qv_norm8(v, v, odd, odd, v, v, v, 1, 128, 1e-6, None) == -1       # one buffer for both
    assert b'must not share' in lib.qv_error()
    assert lib.qv_quantize8(v, v, v, 0, 128, None) == -1
    assert lib.qv_quantize8(v, v, None, 1, 128, None) == -1
    assert lib.qv_quantize8(v, v, v, 1, 17409, None) == -1
    for tokens, width, rows in ((0, 128, 1), (1, 120, 1), (1, 0, 1), (1, 65552, 1), (1, 128, 0), (1, 128, 248321),
                                (139265, 128, 1)):
        assert lib.qv_mm8(v, v, v, v, v, tokens, width, rows, None) == -1
    assert lib.qv_mm8(v, v, v, v, None, 1, 128, 1, None) == -1
    assert lib.qv_error() == b'null projection buffer'
    assert lib.qv_mm8(v, odd, v, v, v, 1, 128, 1, None) == -1
    assert lib.qv_mm8(v, v, v, odd, v, 1, 128, 1, None) == -1
    assert b'16-byte aligned' in lib.qv_error()
    for begin, end, ring in ((-64, 64, 128), (0, 63, 128), (32, 64, 128), (128, 64, 128), (0, 139328, 139328),
                             (0, 128, 64), (0, 128, 100), (64, 128, 96), (0, 64, 0)):
        assert lib.qv_cache8_pack(v, v, v, v, v, v, begin, end, ring, None) == -1, (begin, end, ring)
    assert lib.qv_cache8_pack(v, v, v, v, v, None, 0, 64, 64, None) == -1
    assert lib.qv_cache8_pack(odd, v, v, v, v, v, 0, 64, 64, None) == -1
    for begin, end in ((-1, 5), (6, 5), (0, 139265)):
        assert lib.qv_cache8_unpack(v, v, v, v, v, v, begin, end, None) == -1
    assert lib.qv_cache8_unpack(v, None, v, v, v, v, 0, 5, None) == -1
    off = ct.c_void_p(4098)                               # no fp32 buffer starts there
    for i in range(1, 7):
        assert lib.qv_norm8(*[off if k == i else ct.c_void_p(4096 + 65536 * k) for k in range(7)], 1, 128, 1e-6, None) == -1
        assert b'4-byte aligned' in lib.qv_error()
    for i in (1, 2):
        assert lib.qv_quantize8(*[off if k == i else v for k in range(3)], 1, 128, None) == -1
    for i in (0, 2, 4):
        assert lib.qv_mm8(*[off if k == i else v for k in range(5)], 1, 128, 1, None) == -1
        assert b'4-byte aligned' in lib.qv_error()
    for i in (1, 3):
        assert lib.qv_cache8_pack(*[off if k == i else v for k in range(6)], 0, 64, 64, None) == -1
        assert lib.qv_cache8_unpack(*[off if k == i + 2 else v for k in range(6)], 0, 64, None) == -1
    # an empty range is no work, and no error
    assert lib.qv_cache8_pack(v, v, v, v, v, v, 64, 64, 128, None) == 0
    assert lib.qv_cache8_unpack(v, v, v, v, v, v, 5, 5, None) == 0


def test_tensors_that_do_not_fit_are_refused():
    import torch
    from redshift_b200 import HotPath
    hot = HotPath()
    f = torch.zeros
    with pytest.raises(ValueError, match='x must be a contiguous CUDA tensor'):
        hot.norm8(f(2, 128, dtype=torch.uint8), f(1, 2), f(2, 128), f(128))
    with pytest.raises(ValueError, match='x must be'):
        hot.quantize8(f(2, 128, dtype=torch.uint8), f(1, 2), f(2, 128))
    with pytest.raises(ValueError, match='codes must be'):
        hot.mm8(f(2, 8), f(8, 128, dtype=torch.uint8), f(1, 1), f(2, 128, dtype=torch.uint8), f(1, 2))
    cache = [f(1, 4, 64, 256, dtype=torch.int8), f(1, 4), f(1, 4, 64, 256, dtype=torch.int8), f(1, 4)]
    rows = f(64, 4, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match='key_codes must be'):
        hot.cache8_pack(*cache, rows, rows, 0, 64)
    with pytest.raises(ValueError, match='key_codes must be'):
        hot.cache8_unpack(rows, rows, *cache, 0, 64)


@pytest.mark.gpu
def test_tensors_of_another_type_are_refused(hot):
    """Types of the same size are not taken for one another."""
    import torch
    f = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device='cuda')  # noqa: E731
    codes, scales, x = f(2, 128, dtype=torch.uint8), f(1, 2), f(2, 128)
    for bad in (codes.view(torch.int8), codes.view(torch.float8_e5m2)):
        with pytest.raises(ValueError, match='codes must be'):
            hot.quantize8(bad, scales, x)
        with pytest.raises(ValueError, match='weights must be'):
            hot.mm8(f(2, 2), bad, f(1, 1), codes, scales)
    with pytest.raises(ValueError, match='x must be'):
        hot.norm8(codes, scales, x.to(torch.int32), f(128))
    cache = [f(1, 4, 64, 256, dtype=torch.int8), f(1, 4), f(1, 4, 64, 256, dtype=torch.int8), f(1, 4)]
    rows = f(64, 4, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='key_rows must be'):
        hot.cache8_pack(*cache, rows, rows, 0, 64)
    with pytest.raises(ValueError, match='key_codes must be'):
        hot.cache8_pack(cache[0].view(torch.uint8), *cache[1:], rows.half(), rows.half(), 0, 64)
    hot.quantize8(codes.view(torch.float8_e4m3fn), scales, x)
    assert hot.status() == 0


# ------------------------------------------------------------------ norm8 / quantize8
def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _check_codes(y, codes, scales, slack):
    """Codes and scales of the rows y (float64), each value and scale at most `slack` off relative."""
    want = E.column_scales(y)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(scales), nan)
    assert (np.abs(scales - want)[~nan] <= (slack + F32) * want[~nan] + 2.0 ** -150).all()
    width = y.shape[1]
    per_col = np.repeat(scales.T.astype(np.float64), 128, 1)[:, :width]
    bad = np.isnan(per_col)
    assert not codes[bad].any()
    got = E.decode(codes) * np.where(bad, 0, per_col)
    # half a step of e4m3 around y / scale, whose own error is the value's and the scale's
    room = np.abs(y) * (E4M3 * (1 + 4 * slack + 4 * F32) + 2 * slack + 2 * F32) + 2.0 ** -10 * np.where(bad, 0, per_col)
    assert (np.abs(got - y)[~bad] <= room[~bad]).all()


def _norm_slack(width):
    """Relative error of a normed value: each square and its additions (4 in a lane's block, 5 blocks,
    10 shuffle steps and up to 28 warps in 5 steps) in fp32, halved by the root, then a division,
    the root and two products."""
    return (0.5 * (1 + 3 + 3 + 10) + 0.5 + 1 + 2 + 1) * F32


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,width', [(1, 1), (3, 5), (2, 127), (1, 128), (5, 130), (7, 640), (2, 641), (4, 5120),
                                          (3, 17408), (2, 17407), (300, 256)])
@pytest.mark.parametrize('form', ['plain', 'residual', 'in place'])
def test_norm8_matches_its_definition(hot, tokens, width, form):
    import torch
    rng = np.random.default_rng(7000 + 31 * width + tokens)
    x = rng.standard_normal((tokens, width)).astype(np.float32) * np.float32(3)
    x[:, ::7] *= 50
    x[-1, :128] = 0                                    # a block of zeros (a whole row of them at small widths)
    r = None if form == 'plain' else rng.standard_normal((tokens, width)).astype(np.float32)
    if r is not None:
        r[-1, :128] = 0
    w = (1 + 0.3 * rng.standard_normal(width)).astype(np.float32)
    dx, dr, dw = _dev(x), None if r is None else _dev(r), _dev(w)
    blocks = -(-width // 128)
    codes = torch.full((tokens, width), 0x55, dtype=torch.uint8, device='cuda')
    scales = torch.full((blocks, tokens), -1.0, device='cuda')
    normed = torch.empty_like(dx)
    out = dr if form == 'in place' else torch.empty_like(dx)
    hot.norm8(codes, scales, dx, dw, residual=dr, residual_out=out, normed=normed, epsilon=1e-5)
    torch.cuda.synchronize()
    s, y = E.norm(x, w, r, 1e-5)
    assert np.array_equal(out.cpu().numpy(), s)
    assert np.array_equal(dx.cpu().numpy(), x)
    slack = _norm_slack(width)
    assert (np.abs(normed.cpu().numpy() - y) <= slack * np.abs(y) + 2.0 ** -140).all()
    _check_codes(y, codes.cpu().numpy(), scales.cpu().numpy(), slack)


@pytest.mark.gpu
@pytest.mark.parametrize('exponent', [-60, 55, 63, 64, 90, 118])
def test_norm8_of_rows_whose_squares_leave_fp32(hot, exponent):
    """Rows whose squares underflow or overflow; a value of infinity makes its block NaN and the others zero."""
    import torch
    rng = np.random.default_rng(7150 + exponent)
    x = np.ldexp(rng.standard_normal((5, 900)), exponent).astype(np.float32)
    x[1, 300:] *= np.float32(2.0 ** -80)
    x[4, 200] = np.inf
    w = (1 + 0.3 * rng.standard_normal(900)).astype(np.float32)
    codes = torch.full((5, 900), 0x55, dtype=torch.uint8, device='cuda')
    scales, normed, out = torch.zeros((8, 5), device='cuda'), torch.empty((5, 900), device='cuda'), torch.empty((5, 900), device='cuda')
    hot.norm8(codes, scales, _dev(x), _dev(w), residual_out=out, normed=normed)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), x)
    y = E.norm(x[:4], w)[1]
    slack = _norm_slack(900)
    keep = np.abs(y) > 2.0 ** -100                     # a product below fp32's normal range has fewer bits
    assert (np.abs(normed.cpu().numpy()[:4] - y)[keep] <= slack * np.abs(y)[keep]).all()
    s = scales.cpu().numpy()
    assert np.isnan(s[1, 4]) and not np.delete(s[:, 4], 1).any() and not codes.cpu().numpy()[4].any()
    rows = [0, 2, 3]
    _check_codes(y[rows], codes.cpu().numpy()[rows], s[:, rows], slack)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,width', [(1, 1), (2, 129), (1, 256), (9, 6144), (2, 17408), (131, 144)])
def test_quantize8_of_values_of_every_size(hot, tokens, width):
    import torch
    rng = np.random.default_rng(7100 + width)
    x = rng.standard_normal((tokens, width)).astype(np.float32)
    x *= np.exp2(rng.integers(-130, 100, size=(tokens, 1))).astype(np.float32)   # rows down to subnormal numbers
    codes = torch.zeros((tokens, width), dtype=torch.uint8, device='cuda')
    scales = torch.zeros((-(-width // 128), tokens), device='cuda')
    hot.quantize8(codes, scales, _dev(x))
    torch.cuda.synchronize()
    got_scales = scales.cpu().numpy()
    want = E.column_scales(x.astype(np.float64))
    # correctly rounded, down to the smallest subnormal number
    assert np.array_equal(got_scales, want.astype(np.float32))
    normal = want > 2.0 ** -125
    keep = np.repeat(normal.T, 128, 1)[:, :width].all(1)
    if keep.any():
        _check_codes(x[keep].astype(np.float64), codes.cpu().numpy()[keep], got_scales[:, keep], 0.0)


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_inside_their_block(hot):
    import torch
    rng = np.random.default_rng(7200)
    x = rng.standard_normal((6, 300)).astype(np.float32)
    x[1, 5], x[2, 130], x[3, 299] = np.nan, np.inf, -np.inf
    codes = torch.zeros((6, 300), dtype=torch.uint8, device='cuda')
    scales = torch.zeros((3, 6), device='cuda')
    hot.quantize8(codes, scales, _dev(x))
    torch.cuda.synchronize()
    s = scales.cpu().numpy()
    assert np.isnan(s).sum() == 3 and np.isnan(s[0, 1]) and np.isnan(s[1, 2]) and np.isnan(s[2, 3])
    with np.errstate(invalid='ignore'):
        _check_codes(x.astype(np.float64), codes.cpu().numpy(), s, 0.0)


@pytest.mark.gpu
def test_norm8_of_unaligned_rows(hot):
    """Rows that start between 16-byte borders take the element-wise path and give the same bits."""
    import torch
    tokens, width = 3, 640
    g = torch.Generator(device='cuda')
    g.manual_seed(5)
    base = torch.randn(tokens * width + 1, generator=g, device='cuda')
    x, w = base[1:].view(tokens, width), torch.rand(width, generator=g, device='cuda')
    results = []
    for t in (x, x.clone()):
        codes = torch.zeros((tokens, width), dtype=torch.uint8, device='cuda')
        scales = torch.zeros((5, tokens), device='cuda')
        hot.norm8(codes, scales, t, w)
        results.append((codes, scales))
    torch.cuda.synchronize()
    assert x.data_ptr() % 16 and torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


# ------------------------------------------------------------------ mm8
def _mm8(hot, codes, scales, weights, weight_scales):
    import torch
    out = torch.full((codes.shape[0], weights.shape[0]), float('nan'), device='cuda')
    hot.mm8(out, _dev(weights), _dev(weight_scales), _dev(codes), _dev(scales))
    torch.cuda.synchronize()
    assert hot.status() == 0
    return out.cpu().numpy()


def _codes(rng, shape, spread):
    """Random e4m3 codes: every finite value (`spread`) or a few small integers."""
    if spread:
        c = rng.integers(0, 256, size=shape, dtype=np.uint8)
        return np.where((c & 127) == 127, c ^ 1, c).astype(np.uint8)
    table = np.array([np.flatnonzero(E.e4m3_values() == v)[0] for v in (0, 1, 2, 3, -1, -2, -3)], np.uint8)
    return table[rng.integers(0, 7, size=shape)]


SIZES = [(1, 16, 1), (1, 128, 128), (2, 144, 129), (3, 256, 300), (8, 1024, 127), (16, 512, 256), (17, 2048, 200),
         (33, 656, 513), (64, 1280, 384), (65, 4096, 130), (128, 384, 640), (129, 272, 250), (200, 2064, 520),
         (1, 5120, 5120), (5, 17408, 640), (131, 144, 25700), (1000, 400, 3300), (1, 65536, 20), (2, 128, 19000)]


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,width,rows', SIZES)
def test_mm8_matches_its_definition(hot, tokens, width, rows):
    rng = np.random.default_rng(7300 + tokens + width + rows)
    blocks = -(-width // 128)
    codes, weights = _codes(rng, (tokens, width), True), _codes(rng, (rows, width), True)
    scales = (0.5 + rng.random((blocks, tokens))).astype(np.float32) * np.float32(0.01)
    weight_scales = (rng.random((-(-rows // 128), blocks)) - 0.5).astype(np.float32)
    want, size = E.product(codes, scales, weights, weight_scales)
    got = _mm8(hot, codes, scales, weights, weight_scales)
    # Every one of a block's 128 products is exact, their sum is rounded at most at every addition, and
    # so is the sum over the blocks (and over at most 8 splits); the two scales cost a product each.
    assert (np.abs(got - want) <= (128 + blocks + 8 + 2) * F32 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,width,rows', SIZES)
def test_mm8_is_exact_where_every_sum_is(hot, tokens, width, rows):
    """Small whole numbers and scales that are powers of two: no sum is rounded, so no product may be
    missing, doubled or scaled by a neighbour's scale."""
    rng = np.random.default_rng(7400 + tokens + width + rows)
    blocks = -(-width // 128)
    codes, weights = _codes(rng, (tokens, width), False), _codes(rng, (rows, width), False)
    scales = np.exp2(rng.integers(-3, 2, size=(blocks, tokens))).astype(np.float32)
    weight_scales = np.exp2(rng.integers(-3, 2, size=(-(-rows // 128), blocks))).astype(np.float32)
    want, _ = E.product(codes, scales, weights, weight_scales)
    assert np.array_equal(_mm8(hot, codes, scales, weights, weight_scales), want)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens', [2, 40, 130])
def test_mm8_keeps_nan_and_infinite_scales_to_their_tokens_and_rows(hot, tokens):
    rng = np.random.default_rng(7500 + tokens)
    codes, weights = _codes(rng, (tokens, 256), True), _codes(rng, (26000, 256), True)
    scales, weight_scales = np.ones((2, tokens), np.float32), np.ones((204, 2), np.float32)
    scales[1, 1] = np.nan
    codes[1, 128:] = 0
    weight_scales[2, 0] = np.nan
    got = _mm8(hot, codes, scales, weights, weight_scales)
    bad = np.zeros(got.shape, bool)
    bad[1], bad[:, 256:384] = True, True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.gpu
def test_mm8_takes_what_norm8_writes_on_a_stream_of_its_own_and_in_a_graph(hot):
    """norm8 -> mm8 on another stream, then captured once and replayed on new inputs."""
    import torch
    rng = np.random.default_rng(7600)
    tokens, width, rows = 6, 640, 1000
    x = rng.standard_normal((3, tokens, width)).astype(np.float32)
    gamma = (1 + 0.1 * rng.standard_normal(width)).astype(np.float32)
    weights = _codes(rng, (rows, width), True)
    weight_scales = (rng.random((8, 5)) * 0.01).astype(np.float32)
    dx, dg, dw, dws = _dev(x[0]), _dev(gamma), _dev(weights), _dev(weight_scales)
    codes = torch.zeros((tokens, width), dtype=torch.uint8, device='cuda')
    scales, out = torch.zeros((5, tokens), device='cuda'), torch.zeros((tokens, rows), device='cuda')

    def step():
        hot.norm8(codes, scales, dx, dg)
        hot.mm8(out, dw, dws, codes, scales)

    def expect():
        want, size = E.product(codes.cpu().numpy(), scales.cpu().numpy(), weights, weight_scales)
        return (np.abs(out.cpu().numpy() - want) <= (128 + 5 + 8 + 2) * F32 * size).all()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    assert expect()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in (1, 2, 0):
        dx.copy_(_dev(x[k]))
        graph.replay()
        torch.cuda.synchronize()
        assert expect()
    assert torch.equal(out, first)                     # the first inputs again: the same bits


# ------------------------------------------------------------------ cache8
def _cache(blocks):
    import torch
    c = lambda: torch.full((blocks, 4, 64, 256), 99, dtype=torch.int8, device='cuda')  # noqa: E731
    s = lambda: torch.full((blocks, 4), -7.0, device='cuda')  # noqa: E731
    return c(), s(), c(), s()


def _rows(rng, n):
    x = rng.standard_normal((n, 4, 256)).astype(np.float16)
    x[:, :, 3] *= np.float16(9)                        # a channel far larger than the others
    return x


@pytest.mark.gpu
@pytest.mark.parametrize('begin,end,ring', [(0, 64, 64), (64, 128, 128), (64, 128, 64), (0, 320, 333), (128, 256, 128),
                                            (1024, 1088, 128), (192, 448, 448)])
def test_pack_is_the_nearest_code_exactly(hot, begin, end, ring):
    rng = np.random.default_rng(7700 + begin + end)
    k, v = _rows(rng, ring), _rows(rng, ring)
    k[5 % ring, 1] = 0
    cache = _cache(end // 64 + 2)
    hot.cache8_pack(*cache, _dev(k), _dev(v), begin, end)
    hot.status()
    at = np.arange(begin, end) % ring
    b0, b1 = begin // 64, end // 64
    for rows, codes, scales in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        want_codes, want_scales = E.pack(rows[at])
        codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
        assert np.array_equal(scales[b0:b1], want_scales)
        assert np.array_equal(codes[b0:b1], want_codes)
        # nothing else is written
        assert (np.delete(codes, np.s_[b0:b1], 0) == 99).all() and (np.delete(scales, np.s_[b0:b1], 0) == -7).all()


@pytest.mark.gpu
def test_pack_ties_go_to_the_even_code(hot):
    """Maximum 127 gives the scale 1: halves lie on the border between two codes."""
    x = np.zeros((64, 4, 256), np.float16)
    x[0, :, 0] = 127
    x[1, :, :100] = np.arange(-50, 50)[None] + 0.5
    x[2, :, :100] = np.nextafter(x[1, :, :100], np.float16(200))
    x[3, :, :100] = np.nextafter(x[1, :, :100], np.float16(-200))
    cache = _cache(1)
    hot.cache8_pack(*cache, _dev(x), _dev(-x), 0, 64)
    hot.status()
    assert np.array_equal(cache[0].cpu().numpy(), E.pack(x)[0]) and np.array_equal(cache[2].cpu().numpy(), E.pack(-x)[0])


@pytest.mark.gpu
def test_blocks_of_zeros_subnormal_and_not_finite_values(hot):
    rng = np.random.default_rng(7800)
    x = _rows(rng, 256)
    x[0:64, 0] = 0
    x[64:128, 1] = np.float16(6e-8) * np.sign(x[64:128, 1])       # the smallest fp16 number
    x[130, 2, 200] = np.nan
    x[250, 3, 0] = -np.inf
    cache = _cache(4)
    hot.cache8_pack(*cache, _dev(x), _dev(x), 0, 256)
    hot.status()
    codes, scales = cache[0].cpu().numpy(), cache[1].cpu().numpy()
    want_codes, want_scales = E.pack(x)
    np.testing.assert_array_equal(scales, want_scales)
    assert np.array_equal(codes, want_codes) and np.isnan(scales[2, 2]) and np.isnan(scales[3, 3])
    import torch
    back = torch.empty((256, 4, 256), dtype=torch.float16, device='cuda')
    hot.cache8_unpack(back, torch.empty_like(back), *cache, 0, 256)
    hot.status()
    got = back.cpu().numpy()
    assert np.isnan(got[128:192, 2]).all() and np.isnan(got[192:, 3]).all() and not got[0:64, 0].any()
    assert np.isfinite(np.delete(got, 2, 1)[128:192]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('begin,end,origin', [(0, 64, 0), (0, 1, 0), (63, 65, 60), (100, 300, 100), (64, 256, 0), (319, 320, 5)])
def test_unpack_is_the_rounded_value_and_writes_nothing_else(hot, begin, end, origin):
    import torch
    rng = np.random.default_rng(7900 + begin)
    codes = rng.integers(-127, 128, size=(2, 5, 4, 64, 256)).astype(np.int8)
    scales = (rng.random((2, 5, 4)) * 0.05).astype(np.float32)
    rows = [torch.full((end - origin + 3, 4, 256), 5.0, dtype=torch.float16, device='cuda') for _ in range(2)]
    hot.cache8_unpack(*rows, _dev(codes[0]), _dev(scales[0]), _dev(codes[1]), _dev(scales[1]), begin, end, origin=origin)
    hot.status()
    for i in range(2):
        got = rows[i].cpu().numpy()
        want = E.unpack(codes[i], scales[i])[begin:end]
        part = got[begin - origin:end - origin]
        # the fp32 product, then half a step of fp16 (2^-25 among its subnormal numbers)
        assert (np.abs(part - want) <= np.abs(want) * (F16 + 2 * F32) + 2.0 ** -25).all()
        assert (np.delete(got, np.s_[begin - origin:end - origin], 0) == 5).all()
