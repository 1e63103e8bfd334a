"""The quantiser's scale over the whole range of fp32: every value stays within its
bits, so that sums of a window's rows stay within their counters."""
import numpy as np
import pytest


@pytest.mark.parametrize("power", [-126, -101, -100, -1, 0, 64, 99, 100, 101, 114, 126, 127])
def test_scales_hold_every_finite_maximum(orc, power):
    for m in (1.0, 1.25, 1.9999998):
        v = np.float32(np.ldexp(np.float32(m), power))
        sg, sh = orc.quantizer(np.array([[-v, v], [0.0, 0.0]], np.float32))
        for s, bits in ((sg, 17), (sh, 18)):
            q = float(v) * float(s)
            assert q <= 2.0 ** bits
            assert q >= 2.0 ** (bits - 1) or power < -100
            assert np.isfinite(np.float32(s)) and np.log2(s) == np.rint(np.log2(s))
