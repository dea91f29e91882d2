"""Layout of quantised rows and argument checks of the W8A8 and scoring entry points that need no GPU."""
import ctypes as C
import itertools

import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests.w8a8_ref import BUILDS


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


def manifest(asset):
    """Kernel symbols of a code object, as the library loads them."""
    lib, name, syms = ffi.load(), C.c_char_p(), C.POINTER(C.c_char_p)()
    for i in range(lib.w4a16_manifest(0, None, None)):
        lib.w4a16_manifest(i, C.byref(name), C.byref(syms))
        if name.value == asset.encode():
            return [s.decode() for s in itertools.takewhile(lambda s: s is not None, syms)]
    raise AssertionError(asset)


@pytest.mark.parametrize("t,n,k,glu,kernel,slices", BUILDS)
def test_shapes_of_the_builds_go_where_they_say(t, n, k, glu, kernel, slices):
    p = ops.plan_w8a8(t, n, k, glu=glu)
    assert (p["kernel"], p["k_slices"] > 1) == ("w4a16_w8a8_" + kernel, slices)


def test_every_build_is_run_with_whole_k_and_in_slices():
    assert {("w4a16_w8a8_" + b[4], b[5]) for b in BUILDS} == set(itertools.product(manifest("w8a8"), (False, True)))


def test_plans_hold_what_the_kernels_count_on():
    """Two waves or more and at most eight k slices, a k tile of 64 at least for every wave of every slice, groups of up to 64 rows that cover all of them;
    grids of fewer than 2^32 threads."""
    r = np.random.default_rng(6)
    for _ in range(20000):
        t, n, k = (int(np.exp(r.uniform(0, np.log(top)))) for top in (5000, 300000, 131071))
        glu = bool(r.integers(2))
        n = max(32, n // 32 * 32) if glu else n
        p = ops.plan_w8a8(t, n, k, cu_count=int(r.integers(1, 305)), glu=glu)
        kt = (k + 127) // 128 * 2
        assert 1 <= p["k_slices"] <= 8 and p["workgroups"] * p["waves"] * 64 < 2**32
        if "skinny" in p["kernel"]:
            rb, tt = (int(p["kernel"].split("_")[i][1:]) for i in (3, 4))
            groups, columns = -(-t // 64), -(-(n // 2 if glu else n) // 16)
            assert 2 <= p["waves"] <= 8 and p["waves"] * p["k_slices"] <= kt and 16 * tt * groups >= t > 16 * tt * (groups - 1)
            assert p["workgroups"] == -(-columns // (rb // 2 if glu else rb)) * p["k_slices"] * groups
        else:
            assert p["waves"] == 4 and p["k_slices"] <= kt


def test_plan_refusals():
    for code, words, args in ((ffi.ERR_SHAPE, "t=0", (0, 16, 64)), (ffi.ERR_SHAPE, "n=0", (1, 0, 64)), (ffi.ERR_SHAPE, "k=131072", (1, 16, 131072)),
                              (ffi.ERR_SHAPE, "n=48", (1, 48, 64, 256, True)), (ffi.ERR_ARG, "cus=0", (1, 16, 64, 0)),
                              (ffi.ERR_SHAPE, "exceed the grid", (2**31 - 256, 1000, 64)), (ffi.ERR_SHAPE, "exceed the grid", (2**30, 1, 1)),
                              (ffi.ERR_SHAPE, "exceed the grid", (1, 2**31 - 256, 5120))):
        with pytest.raises(ops.W4a16Error) as e:
            ops.plan_w8a8(*args)
        assert e.value.code == code and words in e.value.message, e.value.message
    assert ffi.load().w4a16_plan_w8a8(16, 64, 1, 256, 0, C.create_string_buffer(10), 10, None, None, None) == ffi.ERR_ARG
    assert ffi.load().w4a16_plan_w8a8(16, 64, 1, 256, 0, None, 0, None, None, None) == 0


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
