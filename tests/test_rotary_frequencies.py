"""Frequencies of the scalings for long contexts with the turns left at their defaults, against their
definitions written out pair by pair."""
import math

import pytest

from kvx_b200 import ops


def _bands(dim, base, scale, length, low, high):
    out = []
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        turns = length * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - low) / (high - low)))
        out.append(f * keep + f / scale * (1 - keep))
    return out


def _ramp(dim, base, scale, length, slow, fast):
    """Pairs ahead of the one that turns `fast` times over the original length keep their frequency, those
    behind the one that turns `slow` times are divided, linear in the pair's index between."""
    at = lambda turns: dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
    first, last = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), dim - 1)
    out = []
    for i in range(dim // 2):
        f = base ** (-2.0 * i / dim)
        divided = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
        out.append(f * (1 - divided) + f / scale * divided)
    return out


@pytest.mark.parametrize("dim,base,scale,length", [(128, 10000.0, 4.0, 4096), (64, 500000.0, 8.0, 8192), (80, 1e6, 16.0, 32768)])
def test_default_turns(dim, base, scale, length):
    kw = dict(base=base, scale=scale, original_length=length)
    close = lambda got, want: all(math.isclose(a, b, rel_tol=1e-12) for a, b in zip(got.tolist(), want, strict=True))
    bands, one = ops.rotary_inv_freq(dim, scaling="bands", **kw)
    assert one == 1.0 and close(bands, _bands(dim, base, scale, length, 1.0, 4.0))
    ramp, factor = ops.rotary_inv_freq(dim, scaling="ramp", **kw)
    assert math.isclose(factor, 0.1 * math.log(scale) + 1.0)
    assert close(ramp, _ramp(dim, base, scale, length, 1.0, 32.0))
    # turns that are given are used
    assert close(ops.rotary_inv_freq(dim, scaling="ramp", low=2.0, high=8.0, **kw)[0], _ramp(dim, base, scale, length, 2.0, 8.0))
    assert close(ops.rotary_inv_freq(dim, scaling="bands", low=2.0, high=8.0, **kw)[0], _bands(dim, base, scale, length, 2.0, 8.0))
    with pytest.raises(ValueError):
        ops.rotary_inv_freq(dim, scaling="ramp", low=32.0, **kw)
