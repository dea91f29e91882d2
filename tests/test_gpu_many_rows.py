"""More rows than one launch holds workgroups for: a launch has fewer than 2^32 threads, so the calls that give a row a workgroup go on
in another one.  Rows are compared with those of calls on a few of them, or with the formula."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import w8a8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


def near_the_joints(t, step):
    """Starts of runs of 48 rows, whole tiles: the ends, and where one launch of `step` rows or of 2^32 threads would stop."""
    last = (t - 48) // 16 * 16
    return sorted({0, last} | {min(max(0, at // 16 * 16 - 16), last) for j in range(1, t // step + 1) for at in (step * j, step * j + 128)})


def rows_of(cc, q, at, n, k):
    """n quantised rows from row `at` (a multiple of 16) on, of many."""
    return ops.unpack_q8(cc.d2h(q + at * (-(-k // 128) * 128), (ops.q8_bytes(n, k),), np.int8), n, k)


def test_quant_rows(dec):
    cc, k, t = dec.cc, 1, 2**26 + 77  # workgroups of 64 threads
    x = np.random.default_rng(1).integers(1, 0x7c00, t).astype(np.uint16).view(np.float16)
    x[::3] *= -1
    with ref.Buffers(cc) as b:
        dx, s, q = b.put(x), b.filled(t * 4), cc.alloc(ops.q8_bytes(t, k))
        try:
            dec.quant_rows(dx, q, s, t, k, x_type=ffi.F16)
            assert np.array_equal(cc.d2h(s, (t,), np.float32), (np.abs(x.astype(np.float64)) / 127).astype(np.float32))
            for at in near_the_joints(t, 2**26 - 128):
                n = min(48, t - at)
                assert np.array_equal(rows_of(cc, q, at, n, k)[:, 0], np.where(x[at:at + n] < 0, -127, 127)), at
        finally:
            cc.free(q)


def test_norm_resid_q8(dec):
    cc, h, t = dec.cc, 16, 2**22 + 77  # workgroups of 1024 threads
    r = np.random.default_rng(2)
    x, ab, nw = (r.standard_normal(n, dtype=np.float32) for n in (t * h, t * h, h))
    with ref.Buffers(cc) as b:
        dx, dab, dnw, s, q = b.put(x), b.put(ab), b.put(nw), b.filled(t * 4), b.filled(ops.q8_bytes(t, h))
        dec.norm_resid_q8(dx, dnw, dab, q, s, t, h)
        assert np.array_equal(cc.d2h(dx, (t * h,), np.float32), x + ab)
        steps = cc.d2h(s, (t,), np.float32)
        for at in near_the_joints(t, 2**22 - 128):
            n = min(48, t - at)
            x1, q1, s1 = b.put(x[at * h:(at + n) * h]), b.filled(ops.q8_bytes(n, h)), b.filled(n * 4)
            dec.norm_resid_q8(x1, dnw, dab + at * h * 4, q1, s1, n, h)
            assert np.array_equal(steps[at:at + n], cc.d2h(s1, (n,), np.float32)), at
            assert np.array_equal(rows_of(cc, q, at, n, h), ops.unpack_q8(cc.d2h(q1, (ops.q8_bytes(n, h),), np.int8), n, h)), at


def test_token_logprobs(dec):
    """Two logits a row: log p of the second is -log(1 + e^d), d = first - second.  Room: 140 units of 2^-24 for the sums and the logarithm,
    six of the result's own size."""
    cc, t, v = dec.cc, 2**24 + 77, 2  # workgroups of 256 threads
    z = (np.random.default_rng(3).standard_normal((t, v), dtype=np.float32) * 3).astype(np.float16)
    with ref.Buffers(cc) as b:
        dz, tg, lp, en, ti, tl = b.put(z), b.put(np.ones(t, np.int32)), *(b.filled(t * 4) for _ in range(4))
        dec.token_logprobs(dz, t, v, logits_type=ffi.F16, targets_dev=tg, logp_dev=lp, entropy_dev=en, top_k=1, top_idx_dev=ti, top_logp_dev=tl)
        d = z[:, 0].astype(np.float64) - z[:, 1]
        want = -np.logaddexp(0, d)
        other = -np.logaddexp(0, -d)
        got = [cc.d2h(p, (t,), np.float32) for p in (lp, en, tl)]
        assert np.array_equal(cc.d2h(ti, (t,), np.int32), (d < 0).astype(np.int32))
    entropy = -(np.exp(want) * want + np.exp(other) * other)
    u = 2.0**-24
    assert (np.abs(got[0] - want) <= (140 + 6 * np.abs(want)) * u).all()
    assert (np.abs(got[1] - entropy) <= 280 * (1 + entropy) * u).all()
    assert (np.abs(got[2] - np.maximum(want, other)) <= (140 + 6) * u).all()
