"""Rows that were read back from the int8 cache and packed again: the same codes and scales, bit for bit."""
import numpy as np
import pytest

from oracle import eight_bit as E

from .test_eight_bit import _cache, _dev, _rows


def test_every_code_of_every_maximum_comes_back():
    """All finite fp16 maxima with all codes that a value can have.  The largest value is code 127, whose fp16
    value is the maximum itself, so the scale is the same; a value is off by half a step of fp16, less than
    half a code.  Below 127 steps of the subnormal numbers a code is less than a step: every value comes back."""
    every = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)       # zero and the positive numbers
    for part in np.array_split(np.arange(1, 0x7C00), 200):
        for i in part if part[0] < 256 else [part]:
            largest = every[i].astype(np.float32).reshape(-1)
            scale = largest / np.float32(127)
            if part[0] < 256:                            # few values below the maximum: the codes they have
                codes = np.rint(every[:i + 1] / np.float64(scale[0]))[None]
            else:
                codes = np.broadcast_to(np.arange(128.0), (len(largest), 128))
            back = (codes.astype(np.float32) * scale[:, None]).astype(np.float16)
            assert codes.max() == 127 and np.array_equal(back[:, -1].astype(np.float32), largest)
            assert np.array_equal(np.rint(back.astype(np.float64) / scale[:, None].astype(np.float64)), codes)


@pytest.mark.gpu
def test_packed_again(hot):
    import torch
    rng = np.random.default_rng(7870)
    k, v = _rows(rng, 640), _rows(rng, 640)
    k *= np.exp2(rng.integers(-22, 12, (10, 4)).repeat(64, 0)[..., None]).astype(np.float16)     # subnormal numbers among them
    v[130, 2, 5] = np.nan
    first, second = _cache(10), _cache(10)
    hot.cache8_pack(*first, _dev(k), _dev(v), 0, 640)
    rows = [torch.empty((640, 4, 256), dtype=torch.float16, device='cuda') for _ in 'kv']
    hot.cache8_unpack(*rows, *first, 0, 640)
    hot.cache8_pack(*second, *rows, 0, 640)
    assert hot.status() == 0
    for a, b in zip(first, second):
        assert np.array_equal(a.cpu().numpy(), b.cpu().numpy(), equal_nan=True)
    assert np.array_equal(first[0].cpu().numpy(), E.pack(k)[0])
