"""FP8 linears: the plain forms themselves, launch plans and argument checks that need no GPU."""
import ctypes as C
import functools
import itertools

import numpy as np
import pytest
import torch

from llm170_amd import ffi, ops
from tests import f8_ref as ref
from tests.test_w8a8_cpu import manifest


def test_e4m3_values_and_rounding_are_torchs():
    bits = torch.arange(256, dtype=torch.int32).to(torch.uint8)
    want = bits.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.isnan(want), np.isnan(ref.E4M3)) and np.array_equal(np.nan_to_num(want), np.nan_to_num(ref.E4M3))
    v = np.random.default_rng(0).standard_normal(200000).astype(np.float32) * np.exp(np.random.default_rng(1).uniform(-9, 4, 200000)).astype(np.float32)
    v = np.clip(np.concatenate([v, (ref.E4M3[:126] + ref.E4M3[1:127]) / 2, [0.0, -0.0, 448, -448, 2.0**-10, 2.0**-11]]), -448, 448).astype(np.float32)
    assert np.array_equal(ref.to_e4m3(v), torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_steps_are_the_least_power_of_two():
    x = np.zeros((6, 130), np.float32)
    x[0, 3], x[1, 0], x[2, 5], x[3, 129] = 448, np.nextafter(np.float32(448), np.float32(999)), 447, np.float32(2.0**-140)
    x[4, 0] = 3.4e38
    q, s = ref.quantised(x)
    assert s[:, :4].T.tolist() == [[1, 0], [2, 0], [1, 0], [0, 2.0**-126]] and s[0, 4] == 2.0**120 and not s[:, 5].any()
    assert ref.E4M3[q[1, 0]] == 224 and q[3, 129] == 0


def test_pack_is_what_unpack_reads():
    for t, k in ((1, 5), (3, 130), (17, 256), (40, 77)):
        q = np.random.default_rng(t).integers(0, 256, (t, k)).astype(np.uint8)
        assert np.array_equal(ops.unpack_q8(ref.pack(q, t, k), t, k).view(np.uint8), q) and len(ref.pack(q, t, k)) == ops.q8_bytes(t, k)


# One shape or more, of ragged sizes, for every kernel of kernels/f8.hip with whole k and with k in slices, on 256 compute units: see shapes()
@functools.lru_cache(None)
def shapes():
    """(t, n, k, gated, row type, result type) of every build, found by the plans themselves: the first of a fixed walk that goes to it."""
    r = np.random.default_rng(13)
    found = {}
    want = set(itertools.product(manifest("f8"), (False, True)))
    for _ in range(200000):
        t = int(np.exp(r.uniform(0, np.log(2600))))
        n, k = int(np.exp(r.uniform(np.log(20), np.log(14000)))), int(np.exp(r.uniform(np.log(140), np.log(17408))))
        glu, y_type, x_type = bool(r.integers(2)), int(r.integers(3)), int(r.choice([0, 1, 2, 4, 4, 4]))
        n = max(256, n // 256 * 256) if glu else n
        if float(t) * n * k > 6e10:
            continue
        p = ops.plan_f8(t, n, k, glu=glu, x_type=x_type, y_type=y_type)
        found.setdefault((p["kernel"], p["k_slices"] > 1), (t, n, k, glu, x_type, y_type))
        if len(found) == len(want):
            break
    return found


def test_every_build_has_a_shape_with_whole_k_and_in_slices():
    assert set(shapes()) == set(itertools.product(manifest("f8"), (False, True)))


def test_plans_hold_what_the_kernels_count_on():
    """At most eight waves and eight k slices, a block of 128 at least for every wave of every slice, groups of up to 64 rows that cover all of them;
    grids of fewer than 2^32 threads; 32-bit sums for f32 results, up to 64 rows and gated up to 1024; few rows of floats without a launch to quantise them."""
    r = np.random.default_rng(6)
    for _ in range(20000):
        t, n, k = (int(np.exp(r.uniform(0, np.log(top)))) for top in (5000, 300000, 131071))
        glu, y_type, x_type = bool(r.integers(2)), int(r.integers(3)), int(r.choice([0, 1, 2, 4]))
        n = max(256, n // 256 * 256) if glu else n
        cus = int(r.integers(1, 305))
        p = ops.plan_f8(t, n, k, cu_count=cus, glu=glu, x_type=x_type, y_type=y_type)
        kb = (k + 127) // 128
        assert 1 <= p["k_slices"] <= 8 and p["workgroups"] * p["waves"] * 64 < 2**32 and ("_glu" in p["kernel"]) == glu
        if "skinny" in p["kernel"]:
            rows = p["kernel"].split("_")[4]
            itself = t <= 16 and x_type != ffi.F8 and -(-kb // p["k_slices"]) * t <= 128 and p["workgroups"] <= (4 * cus if t <= 2 else cus)  # quantised by the kernel
            assert rows == ["f32", "f16", "bf16", "", ""][x_type] if itself else rows[0] == "t"
            rb, tt = int(p["kernel"].split("_")[3][1:]), int(rows[1:]) if rows[0] == "t" else 1
            groups, columns = -(-t // 64), -(-(n // 2 if glu else n) // 16)
            assert 1 <= p["waves"] <= 8 and p["waves"] * p["k_slices"] <= kb and 16 * tt * groups >= t > 16 * tt * (groups - 1)
            assert p["workgroups"] == -(-columns // (rb // 2 if glu else rb)) * p["k_slices"] * groups
        else:
            assert p["waves"] == 4 and p["k_slices"] <= kb and t > 16 and ("exact" in p["kernel"]) == (y_type == ffi.F32 or t <= 64 or (glu and t <= 1024))


def test_plan_refusals():
    for code, words, args in ((ffi.ERR_SHAPE, "t=0", (0, 16, 64)), (ffi.ERR_SHAPE, "n=0", (1, 0, 64)), (ffi.ERR_SHAPE, "k=131072", (1, 16, 131072)),
                              (ffi.ERR_SHAPE, "n=128", (1, 128, 64, 256, True)), (ffi.ERR_ARG, "cus=0", (1, 16, 64, 0)), (ffi.ERR_ARG, "y type 3", (1, 16, 64, 256, False, 1, 3)),
                              (ffi.ERR_ARG, "x type 3", (1, 16, 64, 256, False, 3, 1)),
                              (ffi.ERR_SHAPE, "exceed the grid", (2**31 - 256, 1000, 64)), (ffi.ERR_SHAPE, "exceed the grid", (1, 2**31 - 256, 5120))):
        with pytest.raises(ops.W4a16Error) as e:
            ops.plan_f8(*args)
        assert e.value.code == code and words in e.value.message, e.value.message
    assert ffi.load().w4a16_plan_f8(16, 64, 1, 256, 0, 4, 0, C.create_string_buffer(10), 10, None, None, None) == ffi.ERR_ARG
    assert ffi.load().w4a16_plan_f8(16, 64, 1, 256, 0, 4, 0, None, 0, None, None, None) == 0


def test_null_context_and_unknown_activation_are_refused():
    lib = ffi.load()
    for call in (lambda: lib.w4a16_quant_rows_f8(None, 1, 0, 0, 1, 1, 1, 1), lambda: lib.w4a16_norm_resid_f8(None, 1, 1, 1, 1, 1, 1, 0, 1),
                 lambda: lib.w4a16_upload_lin_f8(None, b"a", None, 0, None, 0, 1, 1, 0), lambda: lib.w4a16_lin_f8_info(None, b"a", None, None),
                 lambda: lib.w4a16_lin_forward_f8(None, b"a", 1, 0, 0, 0, 1, 1, 0), lambda: lib.w4a16_lin_forward_f8_glu(None, b"a", 1, 0, 0, 0, 1, 1, 0, 0)):
        assert call() == ffi.ERR_ARG
    assert lib.w4a16_lin_forward_f8_glu(None, b"a", 1, 0, 0, 0, 1, 1, 0, 2) == ffi.ERR_ARG and b"activation 2" in lib.w4a16_last_error()
