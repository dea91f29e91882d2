"""A launch of 2^32 threads or more: HIP counts them in 32 bits and runs the rest of the division without an error, so it is refused."""
import ctypes as C

import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import w8a8_ref as ref

pytestmark = pytest.mark.gpu


def test_a_launch_of_more_threads_than_hip_counts_is_refused():
    dec = ops.W4a16Dec()
    cc = dec.cc
    try:
        with ref.Buffers(cc) as b:
            words = b.filled(1024)
            args = [C.c_uint64(words), C.c_size_t(256)]  # the fill goes over its words with any grid
            for gx, block in ((1 << 24, 256), ((1 << 24) + 1, 256), (1 << 22, 1024), (0xffffffff, 2)):
                with pytest.raises(ops.W4a16Error) as e:
                    cc.launch("w4a16_fill0_u32", gx, 1, block, args)
                assert e.value.code == ffi.ERR_SHAPE and "2^32" in e.value.message
            assert (cc.d2h(words, (1024,), np.uint8) == 0xA5).all()
            cc.launch("w4a16_fill0_u32", 4, 1, 256, args)
            assert (cc.d2h(words, (1024,), np.uint8) == 0).all()
            # rows of the norm get a workgroup of 1024 threads each
            t = 1 << 22
            x, ab, out, nw = b.filled(t * 4), b.filled(t * 4), b.filled(t * 4), b.filled(4)
            with pytest.raises(ops.W4a16Error) as e:
                dec.norm_resid(x, nw, ab, out, t, 1)
            assert e.value.code == ffi.ERR_SHAPE and (cc.d2h(out, (t * 4,), np.uint8) == 0xA5).all()
    finally:
        cc.close()
