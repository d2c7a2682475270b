"""The quotients behind the e4m3 codes: value / scale by the reciprocal and one correction (Markstein)."""
import numpy as np
import pytest

from .test_eight_bit import _dev


def _e4m3(x):
    """Nearest e4m3 code (ties to even) of fp32 values of at most 448, as bytes."""
    import torch
    return torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


@pytest.mark.gpu
@pytest.mark.parametrize('exponent', [-125, -100, -60, -3, 0, 40, 110])
def test_codes_are_those_of_a_quotient_of_fp32(hot, exponent):
    """The corrected quotient is one of the fp32 numbers next to value / scale, or the rounded quotient itself."""
    import torch
    rng = np.random.default_rng(7860 + exponent)
    x = np.ldexp(rng.standard_normal((64, 4096)), exponent).astype(np.float32)
    x[:, 1::3] = np.ldexp((rng.integers(1, 16, x[:, 1::3].shape) + 0.5), exponent - 4).astype(np.float32)   # near ties
    codes = torch.zeros((64, 4096), dtype=torch.uint8, device='cuda')
    scales = torch.zeros((32, 64), device='cuda')
    hot.quantize8(codes, scales, _dev(x))
    assert hot.status() == 0
    s = np.repeat(scales.cpu().numpy().T, 128, 1)
    q = x / s                                            # numpy's fp32 division is correctly rounded
    limit = np.float32(448)
    near = [_e4m3(np.clip(v, -limit, limit)) for v in (q, np.nextafter(q, -np.float32(np.inf)), np.nextafter(q, np.float32(np.inf)))]
    got = codes.cpu().numpy()
    assert ((got == near[0]) | (got == near[1]) | (got == near[2])).all()
    # the neighbours hardly ever have another code, so the codes are those of the quotient itself
    assert (got != near[0]).mean() < 1e-4
