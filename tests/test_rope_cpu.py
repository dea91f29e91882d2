"""Frequencies of a rotation, and argument checks of the rotation and of the verification that need no GPU."""
import ctypes as C
import math

import numpy as np
import pytest

from llm170_amd import ffi, ops


def formula(rot, base, scaling, factor, trained, low, high):
    out = []
    at = lambda turns: rot * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    for c in range(rot // 2):
        f = base ** (-2 * c / rot)
        if scaling == ffi.ROPE_LINEAR:
            f /= factor
        elif scaling == ffi.ROPE_BANDS:
            wave = 2 * math.pi / f
            if wave > trained / low:
                f /= factor
            elif wave > trained / high:
                s = (trained / wave - low) / (high - low)
                f = (1 - s) * f / factor + s * f
        elif scaling == ffi.ROPE_RAMP:
            lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), rot - 1)
            ramp = min(max((c - lo) / max(hi - lo, 0.001), 0), 1)
            f = f * (1 - ramp) + f / factor * ramp
        out.append(f)
    return out, 0.1 * math.log(factor) + 1 if scaling == ffi.ROPE_RAMP and factor > 1 else 1.0


@pytest.mark.parametrize("rot", [2, 20, 128, 1024])
@pytest.mark.parametrize("scaling", range(4))
def test_frequencies(rot, scaling):
    for base, factor, trained, low, high in ((10000.0, 1.0, 2048.0, 1.0, 4.0), (5e5, 8.0, 8192.0, 1.0, 4.0), (1e6, 4.0, 32768.0, 1.0, 32.0), (100.0, 0.5, 10.0, 0.5, 900.0)):
        got, amp = ops.rope_freqs(rot, base, scaling, factor, trained, low, high)
        want, wamp = formula(rot, base, scaling, factor, trained, low, high)
        assert len(got) == rot // 2 and np.allclose(got, want, rtol=1e-13, atol=0) and abs(amp - wamp) < 1e-7


def test_frequency_refusals():
    ok = dict(rot_dim=8, base=10000.0, scaling=ffi.ROPE_RAMP, factor=2.0, trained=100.0, low=1.0, high=2.0)
    ops.rope_freqs(**ok)
    for change, code in ((dict(rot_dim=7), ffi.ERR_SHAPE), (dict(rot_dim=0), ffi.ERR_SHAPE), (dict(rot_dim=1026), ffi.ERR_SHAPE), (dict(scaling=4), ffi.ERR_ARG),
                         (dict(scaling=-1), ffi.ERR_ARG), (dict(base=1.0), ffi.ERR_ARG), (dict(base=math.nan), ffi.ERR_ARG), (dict(base=math.inf), ffi.ERR_ARG),
                         (dict(factor=0.0), ffi.ERR_ARG), (dict(factor=math.nan), ffi.ERR_ARG), (dict(trained=0.0), ffi.ERR_ARG), (dict(low=2.0), ffi.ERR_ARG), (dict(low=0.0), ffi.ERR_ARG),
                         (dict(high=math.inf), ffi.ERR_ARG)):
        with pytest.raises(ops.W4a16Error) as e:
            ops.rope_freqs(**{**ok, **change})
        assert e.value.code == code and "rope_freqs" in e.value.message
    amp = C.c_float()
    assert ffi.load().w4a16_rope_freqs(8, 10000.0, 0, 1, 1, 1, 1, None, C.byref(amp)) == ffi.ERR_ARG
    ops.rope_freqs(8, 10000.0, ffi.ROPE_PLAIN, math.nan, math.nan, math.nan, math.nan)  # not looked at


def test_null_context_is_refused():
    lib = ffi.load()
    assert lib.w4a16_qk_norm_rope(None, 256, 1, 0, 1, 1, 1, 8, 0, 0, 1e-6, 256, 256, 8, 1.0, 0, 256, 0, 256, 0, 1) == ffi.ERR_ARG
    assert lib.w4a16_verify_drafts(None, 256, 0, 0, 0, 0, 1, 8, 256, 1, 256, 256, 0, 256, 256) == ffi.ERR_ARG
