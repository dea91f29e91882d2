"""Layout of quantised rows and argument checks of the W8A8 and scoring entry points that need no GPU."""
import numpy as np
import pytest

from llm170_amd import ffi, ops


@pytest.mark.parametrize("t,k,want", [(1, 1, 128), (1, 128, 128), (1, 129, 256), (2, 64, 512), (4, 200, 1024), (5, 64, 2048), (16, 128, 2048),
                                      (17, 5120, 32 * 5120), (4096, 17408, 4096 * 17408), (1 << 20, 131071, (1 << 20) * 131072),
                                      (0, 8, 0), (8, 0, 0), (8, 131072, 0)])
def test_q8_bytes(t, k, want):
    assert ops.q8_bytes(t, k) == want


@pytest.mark.parametrize("t,k", [(1, 1), (1, 300), (3, 64), (4, 77), (5, 129), (16, 128), (33, 200)])
def test_unpack_follows_the_documented_place_of_every_element(t, k):
    """The header's formula, element by element, on bytes that are all different from their neighbours'."""
    buf = (np.arange(ops.q8_bytes(t, k)) * 37 % 251).astype(np.uint8).view(np.int8)
    got = ops.unpack_q8(buf, t, k)
    r, tiles = (1 if t == 1 else 4 if t <= 4 else 16), 8 * ((k + 127) // 128)
    want = np.array([[buf[((m // r * tiles + j // 16) * r + m % r) * 16 + j % 16] for j in range(k)] for m in range(t)], np.int8)
    assert got.dtype == np.int8 and np.array_equal(got, want)


def test_null_context_is_refused():
    lib = ffi.load()
    for call in (lambda: lib.w4a16_quant_rows(None, 1, 0, 0, 1, 1, 1, 1), lambda: lib.w4a16_norm_resid_q8(None, 1, 1, 1, 1, 1, 1, 0, 1),
                 lambda: lib.w4a16_upload_lin_w8a8(None, b"a", None, 0, None, 0, 1, 1, 0), lambda: lib.w4a16_lin_w8a8_info(None, b"a", None, None),
                 lambda: lib.w4a16_lin_forward_w8a8(None, b"a", 1, 0, 0, 0, 1, 1, 0), lambda: lib.w4a16_lin_forward_w8a8_glu(None, b"a", 1, 0, 0, 0, 1, 1, 0, 0),
                 lambda: lib.w4a16_token_logprobs(None, 1, 0, 0, 1, 1, 0, 0, 1, 0, 0, 0)):
        assert call() == ffi.ERR_ARG


def test_unknown_activation_is_refused_before_anything_else():
    assert ffi.load().w4a16_lin_forward_w8a8_glu(None, b"a", 1, 0, 0, 0, 1, 1, 0, 2) == ffi.ERR_ARG
    assert b"activation 2" in ffi.load().w4a16_last_error()


def test_no_barrier_with_lds_dma_in_flight():
    """Staging goes through registers: no LDS DMA that a barrier of these kernels, which leaves global loads in flight, could miss."""
    import os
    import subprocess

    from llm170_amd import build
    from tests.test_lds_dma_waits_cpu import OBJDUMP, kernels, open_barriers
    text = subprocess.run([OBJDUMP, "-d", os.path.join(build.ASSET_DIR, "w8a8.hsaco")], stdout=subprocess.PIPE, text=True, check=True).stdout
    seen = 0
    for name, insns in kernels(text).items():
        bad, dma = open_barriers(insns)
        seen += "tiled" in name
        assert not bad and dma == 0, name
    assert seen == 6
