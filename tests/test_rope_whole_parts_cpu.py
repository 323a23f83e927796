"""CPU: the scaling by wavelength whose ramp runs between whole pairs."""
import math

import numpy as np
import pytest

import acfun_b200 as acf


def plain(rot, base, factor, trained, fast, slow):
    def index_of(turns):
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(index_of(fast)), 0), min(math.ceil(index_of(slow)), rot - 1)
    out = []
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        ramp = min(1.0, max(0.0, (i - lo) / ((hi - lo) or 0.001)))
        out.append(f * (1 - ramp) + f / factor * ramp)
    return lo, hi, np.array(out)


@pytest.mark.parametrize("rot,base,factor,trained,fast,slow,ends", [
    (128, 1e6, 4.0, 32768, 32.0, 1.0, (23, 40)), (128, 1e4, 40.0, 4096, 32.0, 1.0, (20, 46)),
    (64, 1e4, 16.0, 4096, 32.0, 1.0, (10, 23)),
    (64, 1e4, 2.0, 100, 32.0, 1.0, (0, 10)),           # the lower end would lie before pair 0
    (4, 2.0, 8.0, 10 ** 9, 32.0, 1.0, (44, 3))])       # both ends behind the last pair: nothing is divided
def test_ramp_between_whole_pairs(rot, base, factor, trained, fast, slow, ends):
    lo, hi, want = plain(rot, base, factor, trained, fast, slow)
    f, a = acf.rope_frequencies(rot, base, scaling="by_whole_parts", factor=factor, trained=trained, fast=fast, slow=slow)
    assert np.isclose(a, 0.1 * math.log(factor) + 1)
    if lo < hi:
        assert (lo, hi) == ends
        assert np.allclose(f, want, rtol=1e-6, atol=0)
        real, _ = acf.rope_frequencies(rot, base, scaling="by_parts", factor=factor, trained=trained, fast=fast, slow=slow)
        assert np.abs(f / real - 1).max() > 2e-3       # not the unrounded ramp
    else:
        assert np.allclose(f, base ** (-2 * np.arange(rot // 2) / rot), rtol=1e-6)


def test_whole_parts_refuse():
    for args in (dict(trained=0), dict(trained=100, fast=1.0, slow=1.0), dict(trained=100, factor=0.5)):
        with pytest.raises(acf.AcfunError):
            acf.rope_frequencies(64, scaling="by_whole_parts", **dict(dict(factor=2.0), **args))
    out = np.empty(32, np.float32)
    assert acf.lib().acfun_rope_frequencies(64, 1e4, 6, 2.0, 100.0, 32.0, 1.0, out.ctypes.data, None) == 1
    acf.lib().acfun_clear_error()
