"""Decode / verify attention over the 8-bit K/V cache (qv_attention8), its cache object, and a run of the
8-bit serving operators together, against their definitions in 64 bits (oracle/eight_bit.py)."""
import ctypes as ct

import numpy as np
import pytest

from oracle import eight_bit as E
from oracle.hotpath import prepare_rows

F32, F16 = 2.0 ** -24, 2.0 ** -11


# ------------------------------------------------------------------ refusals (no GPU)
def _call(lib, batch=1, position=100, packed=64, tail=128, eps=1e-6, ws_bytes=1 << 30, **replace):
    names = ['out', 'kc', 'ks', 'vc', 'vs', 'kt', 'vt', 'q_gate', 'key', 'value', 'q_norm', 'k_norm', 'ws']
    v = {n: ct.c_void_p(4096) for n in names}          # never dereferenced: the arguments are rejected first
    v.update(replace)
    return lib.qv_attention8(v['out'], v['kc'], v['ks'], v['vc'], v['vs'], packed, v['kt'], v['vt'], tail, v['q_gate'],
                             v['key'], v['value'], v['q_norm'], v['k_norm'], batch, position, eps, v['ws'], ws_bytes, None)


def test_rejects_invalid_arguments_before_accessing_buffers(lib):
    for bad in (dict(batch=0), dict(batch=11), dict(position=-1), dict(position=139264), dict(packed=-64), dict(packed=65),
                dict(packed=128), dict(tail=36), dict(tail=0), dict(eps=0.), dict(eps=float('inf')), dict(ws_bytes=1000),
                dict(position=2 ** 31 - 1), dict(batch=10, position=139255)):
        assert _call(lib, **bad) == -1, bad
        assert lib.qv_error()
    for name in ('out', 'kc', 'ks', 'vc', 'vs', 'kt', 'vt', 'q_gate', 'key', 'value', 'q_norm', 'k_norm', 'ws'):
        assert _call(lib, **{name: None}) == -1
        assert lib.qv_error() == b'null attention buffer'
    for name in ('kc', 'vc', 'kt', 'vt', 'q_gate', 'key', 'value', 'q_norm', 'k_norm', 'ws'):
        assert _call(lib, **{name: ct.c_void_p(4104)}) == -1
        assert b'aligned' in lib.qv_error()
    for name in ('out', 'ks', 'vs'):
        assert _call(lib, **{name: ct.c_void_p(4098)}) == -1
        assert lib.qv_error() == b'fp32 buffers must be 4-byte aligned'
    assert lib.qv_attention8_workspace(0, 5) == 0 and lib.qv_attention8_workspace(11, 5) == 0
    assert lib.qv_attention8_workspace(1, 139264) == 0 and lib.qv_attention8_workspace(10, 139254) > 0


def test_cache_object_refuses_what_does_not_fit():
    from redshift_b200 import Cache8
    for context, tail in ((0, 128), (139265, 128), (1000, 64), (1000, 100)):
        with pytest.raises(ValueError):
            Cache8(None, context, tail_rows=tail)


def test_a_position_behind_a_gap_or_in_the_packed_part_is_refused():
    from redshift_b200 import Cache8
    calls = []

    class Recorder:
        def __getattr__(self, name):
            return lambda *args: calls.append(name)
    cache = Cache8(Recorder(), 256, device='cpu:0')
    step = lambda batch, position: cache.attention(None, None, None, None, None, None, batch, position)  # noqa: E731
    with pytest.raises(ValueError, match='leaves a gap'):
        step(1, 1)
    step(8, 0)
    step(8, 3)                                           # five of the eight were not kept
    with pytest.raises(ValueError, match='holds 11 rows'):
        step(1, 12)
    for position in range(11, 64):
        step(1, position)
    assert 'cache8_pack' not in calls and cache.packed == 0
    step(8, 64)
    assert calls.count('cache8_pack') == 1 and cache.packed == 64
    with pytest.raises(ValueError, match='packed part'):
        step(1, 63)
    step(10, 70)
    for position in range(80, 250):
        step(1, position)
    with pytest.raises(ValueError, match='holds 256 positions'):
        step(10, 250)
    with pytest.raises(ValueError, match='outside the cache'):
        cache.unload(cache.key_tail, cache.value_tail, 251)


# ------------------------------------------------------------------ the operator
def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Layer:
    """Random inputs of one call, on the host and on the device."""

    def __init__(self, batch, position, packed, tail, seed, k_scale=None, v_scale=None):
        rng = np.random.default_rng(seed)
        blocks = packed // 64
        self.batch, self.position, self.packed, self.tail = batch, position, packed, tail
        f = np.float32
        self.codes = [np.clip(np.rint(rng.standard_normal((blocks, 4, 64, 256)) * 30), -127, 127).astype(np.int8) for _ in 'kv']
        self.scales = [(0.03 + 0.01 * rng.random((blocks, 4))).astype(f) for _ in 'kv']
        if k_scale:
            self.scales[0] = np.exp2(rng.uniform(*k_scale, (blocks, 4))).astype(f)
        if v_scale:
            self.scales[1] = np.exp2(rng.uniform(*v_scale, (blocks, 4))).astype(f)
        self.tails = [rng.standard_normal((tail, 4, 256)).astype(np.float16) for _ in 'kv']
        self.q_gate = rng.standard_normal((batch, 24, 512)).astype(f)
        self.key, self.value = (rng.standard_normal((batch, 4, 256)).astype(f) for _ in 'kv')
        self.q_norm, self.k_norm = ((1 + 0.2 * rng.standard_normal(256)).astype(f) for _ in 'qk')

    def run(self, hot, workspace=None):
        import torch
        # the null pointers that an empty packed part may have are tested through the library itself
        self.d_codes = [_dev(c) for c in self.codes]
        self.d_scales = [_dev(s) for s in self.scales]
        self.d_tails = [_dev(t) for t in self.tails]
        self.d_in = [_dev(a) for a in (self.q_gate, self.key, self.value, self.q_norm, self.k_norm)]
        self.out = torch.full((self.batch, 24, 256), float('nan'), device='cuda')
        self.again(hot, workspace)
        torch.cuda.synchronize()
        assert hot.status() == 0
        return self.out.cpu().numpy()

    def again(self, hot, workspace=None):
        (kc, vc), (ks, vs), (kt, vt) = self.d_codes, self.d_scales, self.d_tails
        hot.attention8(self.out, kc, ks, vc, vs, self.packed, kt, vt, *self.d_in, self.batch, self.position, 1e-6, workspace)

    def check(self, got, rows=None):
        """The tail's new rows, everything else in it, and the output (of the tokens `rows`)."""
        n = self.position + self.batch
        new = np.arange(self.position, n) % self.tail
        kt, vt = (t.cpu().numpy() for t in self.d_tails)
        want_k = prepare_rows(self.key, self.k_norm, self.position + np.arange(self.batch)[:, None], 1e-6)
        ok = np.isfinite(want_k)
        # fp32 arithmetic (a sum of 256 squares, the root, products and the rotation), half a step of fp16
        room = np.abs(want_k).max(-1, keepdims=True) * 40 * F32 + np.abs(want_k) * F16 + 2.0 ** -25
        assert (np.abs(kt[new] - want_k) <= room)[ok].all()
        with np.errstate(over='ignore'):
            assert np.array_equal(vt[new], self.value.astype(np.float16), equal_nan=True)
        for now, before in ((kt, self.tails[0]), (vt, self.tails[1])):
            assert np.array_equal(np.delete(now, new, 0), np.delete(before, new, 0), equal_nan=True)
        assert all(np.array_equal(d.cpu().numpy(), c) for d, c in zip(self.d_codes, self.codes))
        assert all(np.array_equal(d.cpu().numpy(), s, equal_nan=True) for d, s in zip(self.d_scales, self.scales))
        at = np.arange(self.packed, n) % self.tail
        whole = [np.concatenate([E.unpack(c, s), t[at].astype(np.float64)]) for c, s, t in zip(self.codes, self.scales, (kt, vt))]
        want, size, top = E.attention(*whole, self.q_gate, self.q_norm, self.position)
        self.want = want
        rows = np.arange(self.batch) if rows is None else rows
        # Relative error of a probability: queries as fp16 hi + lo and their fp32 norm and rotation (24 steps),
        # products summed in fp32 (16 groups of a matrix instruction, hi + lo), the exponent's argument and
        # the SFU's 2^x; twice, for the numerator and the sum.  The sums over n positions: in fp32 along
        # tiles, splits and the instruction's groups of 16.
        rel = 2 * (top * (24 + 32 + 4) * F32 + 8 * F32) + (n // 64 / 37 + 37 + 16) * 4 * F32
        # A probability below 2^-36 of the largest (times the value scales) is dropped: with codes up to 127
        # that is under 2^-29, half the smallest step of the fp16 rows.
        assert (np.abs(got - want)[rows] <= rel * size[rows] + 2.0 ** -29).all(), np.abs(got - want)[rows].max()


CASES = [(1, 0, 0, 64), (10, 0, 0, 64), (1, 63, 0, 64), (1, 64, 64, 64), (3, 5, 0, 64), (8, 60, 0, 128), (8, 120, 64, 128),
         (5, 127, 64, 128), (2, 130, 64, 77), (8, 700, 640, 128), (10, 1000, 960, 128), (7, 2500, 2432, 192),
         (1, 2431, 2368, 64), (6, 1500, 0, 1506), (4, 1100, 192, 1000), (8, 5000, 4992, 128), (9, 2367, 2304, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize('batch,position,packed,tail', CASES)
def test_attention_matches_its_definition(hot, batch, position, packed, tail):
    layer = Layer(batch, position, packed, tail, 8000 + position + batch)
    layer.check(layer.run(hot))


@pytest.mark.gpu
@pytest.mark.parametrize('k_scale,v_scale', [((-12, -3), (-30, 8)), ((-6, -4), (-120, -90)), ((-9, -5), (5, 9))])
def test_scales_of_every_size(hot, k_scale, v_scale):
    layer = Layer(4, 900, 896, 128, 8100, k_scale, v_scale)
    layer.check(layer.run(hot))


@pytest.mark.gpu
def test_blocks_of_zeros_take_their_share_of_the_softmax(hot):
    layer = Layer(3, 700, 640, 128, 8200)
    layer.codes[1][2:5], layer.scales[1][2:5] = 0, 0   # values zero: their keys still count
    layer.codes[0][7], layer.scales[0][7] = 0, 0       # keys zero: every score is 0
    layer.codes[1][0], layer.scales[1][0] = 0, 0       # the very first block
    layer.check(layer.run(hot))


@pytest.mark.gpu
def test_scores_that_rise_from_block_to_block(hot):
    """Every tile raises the running maximum by far more than the rescaling threshold, and falls again."""
    layer = Layer(2, 1900, 1856, 128, 8300)
    layer.scales[0][:] = (2.0 ** -7 * (1 + 6 * (np.arange(29) % 9)[:, None] + np.zeros((29, 4)))).astype(np.float32)
    layer.check(layer.run(hot))


@pytest.mark.gpu
def test_a_scale_that_is_nan_reaches_its_head_alone(hot):
    layer = Layer(2, 300, 256, 128, 8400)
    layer.scales[0][1, 0] = np.nan
    layer.scales[1][2, 3] = np.nan
    got = layer.run(hot)
    bad = np.zeros((2, 24, 256), bool)
    bad[:, 0:6], bad[:, 18:24] = True, True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.gpu
@pytest.mark.parametrize('position', [70, 124, 126])
def test_new_tokens_that_are_not_finite_reach_those_that_see_them_alone(hot, position):
    """Token 3's value and token 5's key are not finite: tokens 0-2 (0-4) do not see them; stale rows of the
    ring behind the last position hold NaN and infinity, as rejected tokens leave them."""
    layer = Layer(8, position, 64, 128, 8500 + position)
    n = position + 8
    free = np.setdiff1d(np.arange(128), np.arange(64, n) % 128)
    layer.tails[0][free], layer.tails[1][free] = np.nan, np.inf
    layer.value[3, 1, 17] = np.inf
    layer.key[5, 2, 100] = np.nan
    got = layer.run(hot)
    bad = np.zeros((8, 24), bool)
    bad[3:, 6:12], bad[5:, 12:18] = True, True
    assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
    layer.value[3, 1, 17] = 0.0                        # the tokens before it: as if it were any number
    clean = Layer(8, position, 64, 128, 8500 + position)
    want = clean.run(hot)
    keep = ~bad
    assert np.array_equal(got[keep], want[keep])


@pytest.mark.gpu
def test_null_codes_where_nothing_is_packed(hot):
    import torch
    layer = Layer(2, 3, 0, 64, 8600)
    first = layer.run(hot).copy()
    ws = hot.attention8_workspace(torch.device('cuda', 0))
    layer.out.fill_(float('nan'))
    p = [t.data_ptr() for t in layer.d_tails]
    rc = hot.lib.qv_attention8(layer.out.data_ptr(), None, None, None, None, 0, *p, 64, *[a.data_ptr() for a in layer.d_in],
                               2, 3, 1e-6, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and hot.status() == 0
    assert np.array_equal(layer.out.cpu().numpy(), first)


@pytest.mark.gpu
def test_longest_context(hot):
    """139,264 positions: the last verify block of the longest context, six sampled heads."""
    layer = Layer(8, 139256, 139200, 128, 8700)
    got = layer.run(hot)
    at = np.arange(139200, 139264) % 128
    for h in (0, 7, 13, 23):
        g = h // 6
        k, v = (np.concatenate([(c[:, g].astype(np.float64) * s[:, g].astype(np.float64)[:, None, None]).reshape(-1, 256),
                                t.cpu().numpy()[at, g].astype(np.float64)])
                for c, s, t in zip(layer.codes, layer.scales, layer.d_tails))
        q = prepare_rows(layer.q_gate[:, h, :256], layer.q_norm, 139256 + np.arange(8), 1e-6)
        for t in (0, 7):
            s = k[:139257 + t] @ q[t] / 16
            p = np.exp(s - s.max())
            want = p @ v[:139257 + t] / p.sum() / (1 + np.exp(-layer.q_gate[t, h, 256:].astype(np.float64)))
            assert np.abs(got[t, h] - want).max() <= 2e-3 and np.linalg.norm(got[t, h] - want) <= 2e-5 * np.linalg.norm(want)


@pytest.mark.gpu
def test_two_streams_and_a_graph_with_workspaces_of_their_own(hot):
    import torch
    a, b = Layer(8, 3000, 2944, 128, 8800), Layer(3, 1700, 1664, 128, 8801)
    want = [a.run(hot).copy(), b.run(hot).copy()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        a.out.fill_(float('nan')); b.out.fill_(float('nan'))
        torch.cuda.synchronize()
        for layer, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                layer.again(hot)
        torch.cuda.synchronize()
        assert np.array_equal(a.out.cpu().numpy(), want[0]) and np.array_equal(b.out.cpu().numpy(), want[1])
    ws = hot.attention8_workspace(a.out.device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match='workspace of its own'):
            a.again(hot)
        a.again(hot, ws)
        a.again(hot, ws)
    for _ in range(3):
        a.out.fill_(float('nan'))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(a.out.cpu().numpy(), want[0])
    assert hot.status() == 0


# ------------------------------------------------------------------ the cache object in a decode loop
def _tokens(n, seed):
    import torch
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device='cuda')  # noqa: E731
    return r(n, 24, 512), r(n, 4, 256), r(n, 4, 256), 1 + 0.1 * r(256), 1 + 0.1 * r(256)


@pytest.mark.gpu
def test_decode_loop_with_rejected_tokens_keeps_the_cache_of_single_steps(hot):
    """Verify blocks of 1..10 tokens of which some are rejected (their rows are garbage), against single
    tokens: the same packed codes and scales, the same tail rows, the same outputs."""
    import torch
    from redshift_b200 import Cache8
    n = 330
    q, k, v, qn, kn = _tokens(n, 8900)
    single, blocks = Cache8(hot, 400), Cache8(hot, 400, tail_rows=192)
    outs = torch.empty((n, 24, 256), device='cuda')
    for t in range(n):
        single.attention(outs[t:t + 1], q[t:t + 1], k[t:t + 1], v[t:t + 1], qn, kn, 1, t)
    rng, t = np.random.default_rng(8901), 0
    while t < n:
        batch = int(min(rng.integers(1, 11), n - t))
        kept = int(rng.integers(1, batch + 1))
        qq, kk, vv = (x[t:t + batch].clone() for x in (q, k, v))
        kk[kept:], vv[kept:] = 1e30, float('nan')
        out = torch.empty((batch, 24, 256), device='cuda')
        blocks.attention(out, qq, kk, vv, qn, kn, batch, t)
        # Tokens behind a block border that the verify block crosses read the block before it in fp16 here and
        # as codes in their single step: half a step of a code, 1/254 of the largest value, is their difference.
        same = min(kept, 64 - t % 64)
        assert torch.allclose(out[:same], outs[t:t + same], atol=2e-5, rtol=2e-5), t
        t += kept
    single.pack(n)
    blocks.pack(n)
    assert single.packed == blocks.packed == 320 and hot.status() == 0
    for name in ('key_codes', 'value_codes', 'key_scales', 'value_scales'):
        assert torch.equal(getattr(single, name), getattr(blocks, name)), name
    rows = torch.arange(320, n, device='cuda')
    assert torch.equal(single.key_tail[rows % 128], blocks.key_tail[rows % 192])
    assert torch.equal(single.value_tail[rows % 128], blocks.value_tail[rows % 192])
    with pytest.raises(ValueError, match='packed part'):
        blocks.attention(outs[:1], q[:1], k[:1], v[:1], qn, kn, 1, 319)
    with pytest.raises(ValueError, match='400 positions'):
        blocks.attention(outs[:8], q[:8], k[:8], v[:8], qn, kn, 8, 393)


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [0, 40, 64, 200])
def test_prefill_then_decode(hot, rows):
    """An fp16 prefill (qv_attention) handed to the 8-bit cache, a verify block over it, and the rows back."""
    import torch
    from redshift_b200 import Cache8
    q, k, v, qn, kn = _tokens(rows + 8, 9000 + rows)
    fp16 = [torch.zeros((rows + 8, 4, 256), dtype=torch.float16, device='cuda') for _ in 'kv']
    if rows:
        out = torch.empty((rows, 24, 256), device='cuda')
        hot.attention(out, *fp16, q[:rows], k[:rows], v[:rows], qn, kn, rows, 0)
    cache = Cache8(hot, 512)
    cache.load(*fp16, rows)
    out8, out16 = torch.empty((8, 24, 256), device='cuda'), torch.empty((8, 24, 256), device='cuda')
    cache.attention(out8, q[rows:], k[rows:], v[rows:], qn, kn, 8, rows)
    back = [torch.zeros_like(f) for f in fp16]
    cache.unload(*back, rows + 8)
    hot.attention(out16, *fp16, q[rows:], k[rows:], v[rows:], qn, kn, 8, rows)
    torch.cuda.synchronize()
    end = cache.packed
    assert end == rows // 64 * 64
    # The rows that were handed over come back as they were, and so do the new values.  The new keys are the same
    # numbers to 32 bits (the fp16 kernel forms them in 32, this one in 64), so their fp16 roundings are at most one step
    # (2^-10 of the larger) apart; where a rotation cancels, 32 bits are off by a few 2^-24 of the pair, and a row's dims
    # are at most 16 |weight|, which is less than 2^-18 |weight|.
    small = 2.0 ** -18 * kn.abs().max()
    apart = (back[0][rows:].float() - fp16[0][rows:].float()).abs()
    assert (apart <= 2.0 ** -10 * torch.maximum(back[0][rows:].abs(), fp16[0][rows:].abs()).float() + small).all()
    assert torch.equal(back[0][end:rows], fp16[0][end:rows]) and torch.equal(back[1][end:], fp16[1][end:])
    for b, f in zip(back, fp16):
        if end:
            top = f[:end].float().abs().view(-1, 64, 4, 256).amax((1, 3)).repeat_interleave(64, 0)[:, :, None]
            # half a step of the codes, then of fp16
            assert ((b[:end].float() - f[:end].float()).abs() <= top / 254 * (1 + 2.0 ** -20) + f[:end].float().abs() * 2.0 ** -10).all()
    # the attention over the rows that were read back, in the fp16 kernel
    again = torch.empty_like(out8)
    hot.attention(again, *back, q[rows:], k[rows:], v[rows:], qn, kn, 8, rows)
    torch.cuda.synchronize()
    assert torch.allclose(again, out8, atol=2e-3, rtol=0)          # fp16 rows of the same codes: 2^-11 of keys and values
    if not end:
        # A key that rounds the other way moves the scores of its position by at most |q| |difference| / 16, with |q| of a
        # dim at most 16 sqrt(2) |weight|; the outputs are means of values, so they move by at most twice that, of |v|.
        moved = apart.sum(-1).max() * 2.0 ** 0.5 * qn.abs().max()
        assert torch.allclose(out16, out8, atol=2e-5 + float(2 * moved * v.abs().max()), rtol=2e-5)


# ------------------------------------------------------------------ the operators together
@pytest.mark.gpu
def test_an_attention_layer_in_eight_bits(hot):
    """norm8 -> mm8 (q and gate, k, v) -> attention over the 8-bit cache -> quantize8 -> mm8 -> the next norm8,
    twelve verify blocks with packing in between; every operator against its definition on its own inputs."""
    import torch
    from redshift_b200 import Cache8
    rng = np.random.default_rng(9100)
    E5, T = 640, 8                                       # a narrow residual stream: the head layout is the model's

    def weights(rows, width):
        w = (rng.standard_normal((rows, width)) * 0.5 / np.sqrt(width)).astype(np.float32)
        d = _dev(w)
        codes = torch.empty((rows, width), dtype=torch.uint8, device='cuda')
        row_scales = torch.empty((width // 128, rows), device='cuda')
        hot.quantize8(codes, row_scales, d)              # per row; a 128-block's scale is the largest of its rows
        block = torch.stack([s.view(-1, 128).amax(1) for s in row_scales], 1)
        for b in range(width // 128):
            scaled = (d[:, 128 * b:128 * b + 128] / block[:, b].repeat_interleave(128)[:, None])
            codes[:, 128 * b:128 * b + 128] = scaled.to(torch.float8_e4m3fn).view(torch.uint8)
        return codes, block.contiguous()

    w_qg, w_k, w_v, w_o = weights(24 * 512, E5), weights(1024, E5), weights(1024, E5), weights(E5, 6144)
    gamma = [_dev((1 + 0.1 * rng.standard_normal(E5)).astype(np.float32)) for _ in range(2)]
    qn, kn = (_dev((1 + 0.1 * rng.standard_normal(256)).astype(np.float32)) for _ in 'qk')
    cache = Cache8(hot, 256)
    new = lambda *s: torch.empty(s, device='cuda')  # noqa: E731
    codes = lambda t, w: (torch.empty((t, w), dtype=torch.uint8, device='cuda'), new(-(-w // 128), t))  # noqa: E731

    def product(x8, w):
        out = new(x8[0].shape[0], w[0].shape[0])
        hot.mm8(out, *w, *x8)
        want, size = E.product(x8[0].cpu().numpy(), x8[1].cpu().numpy(), w[0].cpu().numpy(), w[1].cpu().numpy())
        assert (np.abs(out.cpu().numpy() - want) <= (128 + len(x8[1]) + 10) * F32 * size).all()
        return out

    for step in range(12):
        pos = step * T
        stream = _dev(rng.standard_normal((T, E5)).astype(np.float32))
        x8 = codes(T, E5)
        hot.norm8(*x8, stream, gamma[0])
        q_gate = product(x8, w_qg).view(T, 24, 512)
        key, value = product(x8, w_k).view(T, 4, 256), product(x8, w_v).view(T, 4, 256)
        out = new(T, 24, 256)
        cache.attention(out, q_gate, key, value, qn, kn, T, pos)
        n, packed = pos + T, cache.packed
        at = np.arange(packed, n) % 128
        whole = [np.concatenate([E.unpack(c.cpu().numpy(), s.cpu().numpy())[:packed], t.cpu().numpy()[at].astype(np.float64)])
                 for c, s, t in ((cache.key_codes, cache.key_scales, cache.key_tail),
                                 (cache.value_codes, cache.value_scales, cache.value_tail))]
        want, size, top = E.attention(*whole, q_gate.cpu().numpy(), qn.cpu().numpy(), pos)
        assert (np.abs(out.cpu().numpy() - want) <= (2 * (top * 60 + 8) + 55 * 4) * F32 * size).all()
        a8 = codes(T, 6144)
        hot.quantize8(*a8, out.view(T, 6144))
        added = product(a8, w_o)
        n8 = codes(T, E5)
        hot.norm8(*n8, added, gamma[1], residual=stream, residual_out=stream)
        assert torch.isfinite(stream).all()
    assert cache.packed == 64 and hot.status() == 0


@pytest.mark.gpu
def test_packing_under_capture_is_refused(hot):
    """A replay would pack tail rows that hold other positions by then."""
    import torch
    from redshift_b200 import Cache8
    cache = Cache8(hot, 256)
    q, k, v, qn, kn = _tokens(8, 9200)
    out = torch.empty((8, 24, 256), device='cuda')
    for position in range(0, 64, 8):
        cache.attention(out, q, k, v, qn, kn, 8, position)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        out.zero_()
        with pytest.raises(RuntimeError, match='capture'):
            cache.attention(out, q, k, v, qn, kn, 8, 64)
        graph.capture_end()
    assert cache.packed == 0 and cache.rows == 64
    cache.attention(out, q, k, v, qn, kn, 8, 64)
    torch.cuda.synchronize()
    assert cache.packed == 64 and hot.status() == 0
