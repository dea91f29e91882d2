"""W8A8 linears on the GPU: quantised rows, the fused norm, products and their gated form, against plain forms in 64 bits.
Whole-number sums are exact and every rounding after them is fixed, so results are compared bit for bit."""
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


def say(*a):
    print(*a, flush=True)


def run_quant(dec, b, dev_x, t, k, kind, ldx=0):
    q, s = b.filled(ops.q8_bytes(t, k)), b.filled(t * 4)
    dec.quant_rows(dev_x, q, s, t, k, x_type=kind, ldx=ldx)
    return q, s


def read_quant(dec, q, s, t, k):
    return ops.unpack_q8(dec.cc.d2h(q, (ops.q8_bytes(t, k),), np.int8), t, k), dec.cc.d2h(s, (t,), np.float32)


@pytest.mark.parametrize("kind", [ffi.F32, ffi.F16, ffi.BF16])
@pytest.mark.parametrize("t,k", [(1, 1), (1, 17), (1, 5120), (1, 17408), (2, 16), (3, 2051), (4, 128), (5, 33), (16, 4096), (17, 8193), (100, 1000),
                                 (129, 40000), (300, 96)])
def test_quant_rows_exactly(dec, t, k, kind):
    say("quant", t, k, kind)
    r = np.random.default_rng(t * 100003 + k)
    bits, x = ref.narrow(r.standard_normal((t, k)).astype(np.float32) * r.uniform(1e-3, 50, (t, 1)).astype(np.float32), kind)
    with ref.Buffers(dec.cc) as b:
        q, s = read_quant(dec, *run_quant(dec, b, b.put(bits), t, k, kind), t, k)
    wq, ws = ref.quantised(x)
    assert np.array_equal(s.view(np.uint32), ws.view(np.uint32))
    assert np.array_equal(q, wq)


def test_quant_rows_halves_go_to_the_even_step(dec):
    """A row whose step is a power of two, values on and next to every half."""
    t, step = 6, np.float32(2.0**-3)
    halves = (np.arange(-126, 127) + np.float32(0.5)) * step
    row = np.concatenate([halves, np.nextafter(halves, np.float32(1e9)), np.nextafter(halves, np.float32(-1e9)), [127 * step]]).astype(np.float32)
    x = np.stack([row * np.float32(2.0**e) for e in (0, 20, -20, 90, -100, 60)])
    with ref.Buffers(dec.cc) as b:
        q, s = read_quant(dec, *run_quant(dec, b, b.put(x), t, x.shape[1], ffi.F32), t, x.shape[1])
    wq, ws = ref.quantised(x)
    assert np.array_equal(s, ws) and np.array_equal(q, wq)
    # steps that are no power of two: x = fl(s * (j + 1/2)) and its neighbours
    r = np.random.default_rng(3)
    rows = []
    for _ in range(8):
        big = np.float32(r.uniform(0.1, 300))
        st = np.float32(np.float64(big) / 127)
        h = ((np.arange(-126, 127) + 0.5) * np.float64(st)).astype(np.float32)
        rows.append(np.concatenate([h, np.nextafter(h, np.float32(1e9)), np.nextafter(h, np.float32(-1e9)), [big]]))
    x = np.stack(rows).astype(np.float32)
    with ref.Buffers(dec.cc) as b:
        q, s = read_quant(dec, *run_quant(dec, b, b.put(x), 8, x.shape[1], ffi.F32), 8, x.shape[1])
    wq, ws = ref.quantised(x)
    assert np.array_equal(s, ws) and np.array_equal(q, wq)


def test_quant_rows_of_nothing_and_of_no_number(dec):
    k = 200
    x = np.random.default_rng(5).standard_normal((9, k)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= np.float32(1e-40)  # subnormal: below any step
    x[3, 7] = np.inf
    x[4, 199] = -np.inf
    x[5, 0] = np.nan
    x[6] = np.float32(3.4e38)
    x[7, :] = 0
    x[7, 100] = np.float32(2.0**-126 * 127)  # the smallest step there is
    with ref.Buffers(dec.cc) as b:
        q, s = read_quant(dec, *run_quant(dec, b, b.put(x), 9, k, ffi.F32), 9, k)
    wq, ws = ref.quantised(x)
    assert np.array_equal(np.isnan(s), np.isnan(ws)) and np.array_equal(np.nan_to_num(s), np.nan_to_num(ws)) and np.array_equal(q, wq)
    assert s[7] > 0 and q[7, 100] == 127 and not q[:6].any(0)[[0]].any()


@pytest.mark.parametrize("kind,t,k,ldx,off", [(ffi.F16, 5, 65, 67, 2), (ffi.BF16, 37, 2051, 2051, 2), (ffi.F32, 3, 33, 41, 4), (ffi.F16, 20, 512, 1027, 6),
                                              (ffi.F32, 1, 4099, 0, 12)])
def test_quant_rows_at_any_element_alignment_and_stride(dec, kind, t, k, ldx, off):
    ld = ldx or k
    bits, x = ref.narrow(np.random.default_rng(k).standard_normal((t, ld)).astype(np.float32), kind)
    flat = bits.reshape(-1)[:(t - 1) * ld + k]  # nothing behind the last row's last element
    with ref.Buffers(dec.cc) as b:
        q, s = read_quant(dec, *run_quant(dec, b, b.put(flat, off), t, k, kind, ldx), t, k)
    wq, ws = ref.quantised(x[:, :k])
    assert np.array_equal(s, ws) and np.array_equal(q, wq)


@pytest.mark.parametrize("t,k", [(3, 100), (5, 16), (18, 200), (1, 129)])
def test_quant_rows_leaves_what_is_no_element(dec, t, k):
    n = ops.q8_bytes(t, k)
    bits, _ = ref.narrow(np.ones((t, k), np.float32), ffi.F16)
    with ref.Buffers(dec.cc) as b:
        q, s = run_quant(dec, b, b.put(bits), t, k, ffi.F16)
        raw = dec.cc.d2h(q, (n + 32,), np.uint8)
    chunks = (k + 15) // 16  # whole chunks of 16 are written: k is padded with zeros inside its last one
    assert (raw[:n] != 0xA5).sum() == t * chunks * 16


@pytest.mark.parametrize("t,hidden,w_off", [(1, 4096, 0), (1, 7, 3), (4, 5120, 0), (5, 1000, 24), (17, 8192, 0), (300, 2048, 1)])
def test_norm_resid_q8_is_norm_resid_and_quant_rows(dec, t, hidden, w_off):
    r = np.random.default_rng(t + hidden)
    x, ab = (r.standard_normal((t, hidden)) * 3).astype(np.float32), r.standard_normal((t, hidden)).astype(np.float32)
    nw = (1 + 0.2 * r.standard_normal(hidden + w_off)).astype(np.float32)
    cc = dec.cc
    with ref.Buffers(cc) as b:
        x1, x2, dab, dnw, xn = b.put(x), b.put(x), b.put(ab), b.put(nw), b.filled(t * hidden * 4)
        q2, s2 = b.filled(ops.q8_bytes(t, hidden)), b.filled(t * 4)
        dec.norm_resid(x1, dnw, dab, xn, t, hidden, w_off=w_off)
        q1, s1 = run_quant(dec, b, xn, t, hidden, ffi.F32)
        dec.norm_resid_q8(x2, dnw, dab, q2, s2, t, hidden, w_off=w_off)
        qa, sa = read_quant(dec, q1, s1, t, hidden)
        qb, sb = read_quant(dec, q2, s2, t, hidden)
        assert np.array_equal(sa.view(np.uint32), sb.view(np.uint32)) and np.array_equal(qa, qb)
        assert np.array_equal(cc.d2h(x1, (t, hidden), np.uint32), cc.d2h(x2, (t, hidden), np.uint32))
        # and both are near the formula in 64 bits: one step at most, where a value lies next to a border
        v = x.astype(np.float64) + ab
        v = v.astype(np.float32).astype(np.float64)
        want = v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6) * nw[w_off:]
        assert (np.abs(qb * sb[:, None].astype(np.float64) - want) <= sb[:, None] * 0.5001).all()


@pytest.mark.parametrize("t,hidden", [(1, 7), (3, 100), (18, 1000), (5, 8185), (2, 16)])
def test_both_ways_to_quantised_rows_write_the_same_bytes(dec, t, hidden):
    """Of the whole buffer: elements, zeros behind a row's end inside its last 16 bytes, and the bytes that neither touches; a row of no number among them."""
    r = np.random.default_rng(hidden)
    x, ab, nw = (r.standard_normal(n).astype(np.float32) for n in ((t, hidden), (t, hidden), hidden))
    if t > 1:
        x[1, 3] = np.nan
    cc, n = dec.cc, ops.q8_bytes(t, hidden)
    with ref.Buffers(cc) as b:
        x1, x2, dab, dnw, xn, s2, q2 = b.put(x), b.put(x), b.put(ab), b.put(nw), b.filled(t * hidden * 4), b.filled(t * 4), b.filled(n)
        dec.norm_resid(x1, dnw, dab, xn, t, hidden)
        q1, _ = run_quant(dec, b, xn, t, hidden, ffi.F32)
        dec.norm_resid_q8(x2, dnw, dab, q2, s2, t, hidden)
        first, second = cc.d2h(q1, (n,), np.uint8), cc.d2h(q2, (n,), np.uint8)
    assert np.array_equal(first, second)
    place = np.arange(n).reshape(-1, -(-hidden // 128) * 8, 1 if t == 1 else 4 if t <= 4 else 16, 16).transpose(0, 2, 1, 3).reshape(-1, -(-hidden // 128) * 128)
    whole = -(-hidden // 16) * 16
    assert not first[place[:t, hidden:whole]].any() and (first[place[:t, whole:]] == 0xA5).all() and (first[place[t:]] == 0xA5).all()


def test_norm_resid_q8_of_infinity(dec):
    t, h = 3, 256
    x, ab, nw = np.ones((t, h), np.float32), np.ones((t, h), np.float32), np.ones(h, np.float32)
    x[1, 5] = np.inf
    with ref.Buffers(dec.cc) as b:
        q, s = b.filled(ops.q8_bytes(t, h)), b.filled(t * 4)
        dec.norm_resid_q8(b.put(x), b.put(nw), b.put(ab), q, s, t, h)
        q, s = read_quant(dec, q, s, t, h)
    assert np.isnan(s[1]) and not q[1].any() and (q[0] == 127).all() and (q[2] == 127).all()


SHAPES = [(1, 16, 64), (1, 1, 1), (1, 4096, 4096), (1, 16500, 640), (2, 33, 130), (3, 100, 77), (4, 512, 2048), (5, 48, 63), (7, 17, 4000), (16, 512, 17408),
          (16, 16400, 256), (17, 40, 300), (31, 1000, 1024), (33, 16401, 192), (37, 5003, 2051), (48, 64, 65), (49, 256, 512), (64, 16416, 320), (64, 700, 1500),
          (65, 256, 128), (65, 1, 1), (100, 513, 1000), (128, 256, 384), (129, 300, 64), (300, 520, 2051), (1000, 257, 129), (513, 4100, 640), (2049, 1030, 256),
          # groups of 64 rows, with k whole and in slices
          (65, 256, 1000), (70, 300, 2048), (129, 1000, 2048), (66, 300, 17408), (100, 700, 12000), (257, 5, 8000), (400, 10000, 128), (577, 1300, 4100),
          # tiles of 64 x 128, 64 x 256 and 128 x 256, with k whole and in slices
          (200, 10000, 8000), (1025, 300, 128), (1100, 256, 1000), (1089, 515, 2048), (1100, 70, 8000), (1100, 4100, 128), (130, 10016, 4096), (1025, 2000, 8000),
          (129, 6000, 4096), (200, 6001, 8000)]


@pytest.mark.parametrize("t,n,k", SHAPES)
def test_linear_bit_for_bit(dec, t, n, k):
    say("linear", t, n, k)
    w, sb, sv = ref.weights(n * 7 + k, n, k)
    w[0] = -128
    w[-1] = 127
    bits, x = ref.narrow(np.random.default_rng(t).standard_normal((t, k)).astype(np.float32), ffi.F16)
    dec.upload_lin_w8a8("l", w, sb, n, k)
    assert dec.lin_w8a8_spec("l") == {"n": n, "k": k}
    q, s = ref.quantised(x)
    want = ref.product(q, s, w, sv)
    with ref.Buffers(dec.cc) as b:
        dx = b.put(bits)
        for y_type in (ffi.F32, ffi.F16, ffi.BF16):
            y = b.filled(t * n * 4 + 64)
            dec.lin_forward_w8a8("l", dx, y, t, x_type=ffi.F16, y_type=y_type)
            size = 4 if y_type == ffi.F32 else 2
            got = dec.cc.d2h(y, (t * n,), ref.bits_type(y_type)).reshape(t, n)
            assert np.array_equal(got, ref.as_type(want, y_type)), y_type
            assert (dec.cc.d2h(y + t * n * size, (64,), np.uint8) == 0xA5).all()  # nothing behind the last row


def gated(dec, b, want, gelu):
    """f16 bits of act(gate) * up of f32 products [t][n], by the separate kernel."""
    t, n = want.shape
    a = b.filled(t * n)
    dec.act_mul_f16(b.put(want), n // 2, t, a, gelu=gelu)
    return dec.cc.d2h(a, (t, n // 2), np.uint16)


@pytest.mark.parametrize("t,n,k,glu,kernel,slices", ref.BUILDS)
def test_every_build_bit_for_bit(dec, t, n, k, glu, kernel, slices):
    say("build", t, n, k, glu, kernel, slices)
    w, sb, sv = ref.weights(n * 5 + k, n, k)
    bits, x = ref.narrow(np.random.default_rng(t + k).standard_normal((t, k)).astype(np.float32), ffi.F16)
    dec.upload_lin_w8a8("b", w, sb, n, k)
    want = ref.product(*ref.quantised(x), w, sv)
    with ref.Buffers(dec.cc) as b:
        dx, y = b.put(bits), b.filled(t * n * 4 + 64)
        if glu:
            for gelu in (False, True):
                dec.lin_forward_w8a8_glu("b", dx, y, t, x_type=ffi.F16, y_type=ffi.F16, gelu=gelu)
                assert dec.cc.last_launch_symbol() == "w4a16_w8a8_" + kernel
                assert np.array_equal(dec.cc.d2h(y, (t, n // 2), np.uint16), gated(dec, b, want, gelu))
            assert (dec.cc.d2h(y + t * n, (64,), np.uint8) == 0xA5).all()  # nothing behind the last row
        else:
            for y_type, size in ((ffi.F16, 2), (ffi.BF16, 2), (ffi.F32, 4)):
                dec.lin_forward_w8a8("b", dx, y, t, x_type=ffi.F16, y_type=y_type)
                assert dec.cc.last_launch_symbol() == "w4a16_w8a8_" + kernel
                assert np.array_equal(dec.cc.d2h(y, (t, n), ref.bits_type(y_type)), ref.as_type(want, y_type)), y_type
                assert size == 4 or y_type == ffi.BF16 or (dec.cc.d2h(y + t * n * size, (64,), np.uint8) == 0xA5).all()
            assert (dec.cc.d2h(y + t * n * 4, (64,), np.uint8) == 0xA5).all()


@pytest.mark.parametrize("t,n,k,glu,kernel", [(4, 131072, 5120, False, "skinny_r4_t1"), (8, 5120, 17408, False, "skinny_r4_t1"), (16, 5120, 17408, False, "skinny_r4_t1"),
                                              (32, 34816, 5120, True, "skinny_r4_t2_glu"), (64, 34816, 5120, True, "skinny_r4_t4_glu"),
                                              (300, 34816, 5120, True, "tiled_m128_glu"), (300, 5120, 17408, False, "tiled_m128")])
def test_layers_and_a_head_of_full_size(dec, t, n, k, glu, kernel):
    """What the wide layers and heads of a model launch, at 1000 of the outputs and the ends."""
    say("layer", t, n, k, glu, kernel)
    w, sb, sv = ref.weights(7, n, k)
    bits, x = ref.narrow(np.random.default_rng(t).standard_normal((t, k)).astype(np.float32), ffi.F16)
    dec.upload_lin_w8a8("layer", w, sb, n, k)
    out = n // 2 if glu else n
    at = np.unique(np.concatenate([[0, out - 1], np.random.default_rng(1).integers(0, out, 1000)]))
    rows = np.concatenate([at, at + out]) if glu else at
    want = ref.product(*ref.quantised(x), w[rows], sv[rows])
    with ref.Buffers(dec.cc) as b:
        dx, y = b.put(bits), b.filled(t * out * 4)
        if glu:
            dec.lin_forward_w8a8_glu("layer", dx, y, t, x_type=ffi.F16, y_type=ffi.F16)
            ran = dec.cc.last_launch_symbol()
            got, want = dec.cc.d2h(y, (t, out), np.uint16)[:, at], gated(dec, b, want, False)
        else:
            dec.lin_forward_w8a8("layer", dx, y, t, x_type=ffi.F16, y_type=ffi.F32)
            ran = dec.cc.last_launch_symbol()
            got, want = dec.cc.d2h(y, (t, out), np.uint32)[:, at], want.view(np.uint32)
    assert ran == "w4a16_w8a8_" + kernel
    assert np.array_equal(got, want)


@pytest.mark.parametrize("t", [1, 3, 16, 40, 64, 65, 200])
def test_linear_on_quantised_rows_and_on_rows_of_floats(dec, t):
    """The same rows through quant_rows and through the linear's own quantisation, with a stride, every type; several linears of one q."""
    n, k, ld = 200, 777, 801
    r = np.random.default_rng(t)
    for kind in (ffi.F32, ffi.F16, ffi.BF16):
        bits, x = ref.narrow(r.standard_normal((t, ld)).astype(np.float32), kind)
        q, s = ref.quantised(x[:, :k])
        with ref.Buffers(dec.cc) as b:
            dx = b.put(bits.reshape(-1)[:(t - 1) * ld + k])
            dq, ds = run_quant(dec, b, dx, t, k, kind, ld)
            for i, s_kind in enumerate((ffi.F32, ffi.F16, ffi.BF16)):
                w, sb, sv = ref.weights(i, n, k, s_kind)
                dec.upload_lin_w8a8("p%d" % i, w, sb, n, k)
                want = ref.product(q, s, w, sv)
                for xd, x_type, xs, ldx in ((dq, ffi.Q8, ds, 0), (dx, kind, 0, ld)):
                    y = b.filled(t * n * 4)
                    dec.lin_forward_w8a8("p%d" % i, xd, y, t, x_type=x_type, xs_dev=xs, ldx=ldx, y_type=ffi.F32)
                    assert np.array_equal(dec.cc.d2h(y, (t, n), np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("k", [131071, 131008])
def test_longest_sums_do_not_overflow(dec, k):
    """-128 times -127 and 127 times 127 over the longest k: the largest sums there are."""
    n, t = 3, 2
    w = np.full((n, k), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    x = np.full((t, k), -1, np.float32)
    x[1] = 1
    sv = np.ones(n, np.float32)
    dec.upload_lin_w8a8("long", w, sv, n, k)
    q, s = ref.quantised(x)
    for rows in (2, 70):
        xx = np.repeat(x, rows // 2, 0)
        with ref.Buffers(dec.cc) as b:
            y = b.filled(rows * n * 4)
            dec.lin_forward_w8a8("long", b.put(xx), y, rows, x_type=ffi.F32, y_type=ffi.F32)
            got = dec.cc.d2h(y, (rows, n), np.uint32)
        assert np.array_equal(got, np.repeat(ref.product(q, s, w, sv), rows // 2, 0).view(np.uint32))


@pytest.mark.parametrize("t", [2, 17, 66])
def test_rows_with_no_number_stay_alone(dec, t):
    n, k = 70, 300
    w, sb, sv = ref.weights(1, n, k)
    x = np.random.default_rng(1).standard_normal((t, k)).astype(np.float32)
    x[1, 3] = np.nan
    dec.upload_lin_w8a8("nan", w, sb, n, k)
    q, s = ref.quantised(x)
    want = ref.product(q, s, w, sv)
    with ref.Buffers(dec.cc) as b:
        y = b.filled(t * n * 4)
        dec.lin_forward_w8a8("nan", b.put(x), y, t, x_type=ffi.F32, y_type=ffi.F32)
        got = dec.cc.d2h(y, (t, n), np.float32)
    assert np.isnan(got[1]).all()
    keep = np.arange(t) != 1
    assert np.array_equal(got[keep].view(np.uint32), want[keep].view(np.uint32))


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("t,n,k", [(1, 32, 64), (1, 34816, 256), (2, 96, 200), (4, 22016, 128), (16, 1056, 777), (17, 64, 64), (33, 33000 // 32 * 32, 128), (48, 320, 100),
                                   (64, 2080, 640), (65, 32, 64), (70, 544, 333), (257, 1088, 512), (70, 800, 9000), (140, 2080, 4100), (450, 9984, 128),
                                   (1030, 96, 128), (1100, 544, 2050), (1025, 64, 8000), (1100, 4128, 128), (130, 10016, 4096), (129, 6016, 4096), (201, 10016, 8000)])
def test_gated_is_the_linear_and_its_activation(dec, t, n, k, gelu):
    say("glu", t, n, k, gelu)
    w, sb, sv = ref.weights(n + k, n, k)
    bits, x = ref.narrow(np.random.default_rng(t).standard_normal((t, k)).astype(np.float32), ffi.F16)
    dec.upload_lin_w8a8("g", w, sb, n, k)
    f = n // 2
    with ref.Buffers(dec.cc) as b:
        dx, gu, a16, y = b.put(bits), b.filled(t * n * 4), b.filled(t * f * 2), b.filled(t * f * 4 + 64)
        dec.lin_forward_w8a8("g", dx, gu, t, x_type=ffi.F16, y_type=ffi.F32)
        dec.act_mul_f16(gu, f, t, a16, gelu=gelu)
        dec.lin_forward_w8a8_glu("g", dx, y, t, x_type=ffi.F16, y_type=ffi.F16, gelu=gelu)
        h = dec.cc.d2h(a16, (t, f), np.uint16)
        assert np.array_equal(dec.cc.d2h(y, (t, f), np.uint16), h)
        dec.lin_forward_w8a8_glu("g", dx, y, t, x_type=ffi.F16, y_type=ffi.F32, gelu=gelu)
        y32 = dec.cc.d2h(y, (t, f), np.float32)
        assert np.array_equal(y32.astype(np.float16).view(np.uint16), h)
        assert (dec.cc.d2h(y + t * f * 4, (64,), np.uint8) == 0xA5).all()
        dec.lin_forward_w8a8_glu("g", dx, y, t, x_type=ffi.F16, y_type=ffi.BF16, gelu=gelu)
        assert np.array_equal(dec.cc.d2h(y, (t, f), np.uint16), ref.to_bf16(y32))


def test_results_at_any_element_alignment(dec):
    n, k = 37, 128
    w, sb, sv = ref.weights(2, n, k)
    dec.upload_lin_w8a8("al", w, sb, n, k)
    for t in (3, 20, 80):
        x = np.random.default_rng(t).standard_normal((t, k)).astype(np.float32)
        want = ref.product(*ref.quantised(x), w, sv)
        for y_type, off in ((ffi.F16, 2), (ffi.BF16, 6), (ffi.F32, 4)):
            with ref.Buffers(dec.cc) as b:
                y = b.filled(t * n * 4, offset=off)
                dec.lin_forward_w8a8("al", b.put(x, 4), y, t, x_type=ffi.F32, y_type=y_type)
                assert np.array_equal(dec.cc.d2h(y, (t, n), ref.bits_type(y_type)), ref.as_type(want, y_type))


def refused(code, words, call):
    with pytest.raises(ops.W4a16Error) as e:
        call()
    assert e.value.code == code and words in e.value.message, e.value.message


def test_refusals(dec):
    w, sb, _ = ref.weights(1, 40, 64)
    dec.upload_lin_w8a8("r", w, sb, 40, 64)
    f, g, lib = dec.lin_forward_w8a8, dec.lin_forward_w8a8_glu, dec.cc.lib
    refused(ffi.ERR_NOT_FOUND, "not registered", lambda: f("absent", 256, 256, 1))
    refused(ffi.ERR_ARG, "null operand", lambda: f("r", 0, 256, 1))
    refused(ffi.ERR_ARG, "null operand", lambda: f("r", 256, 0, 1))
    refused(ffi.ERR_SHAPE, "t=0", lambda: f("r", 256, 256, 0))
    refused(ffi.ERR_ARG, "x type 4", lambda: f("r", 256, 256, 1, x_type=4))
    refused(ffi.ERR_ARG, "y type 3", lambda: f("r", 256, 256, 1, y_type=3))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.Q8))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.Q8, xs_dev=256, ldx=64))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.F16, xs_dev=256))
    refused(ffi.ERR_SHAPE, "ldx=63", lambda: f("r", 256, 256, 2, ldx=63))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 257, 256, 1))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 256, 258, 1, y_type=ffi.F32))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 264, 256, 1, x_type=ffi.Q8, xs_dev=256))
    refused(ffi.ERR_SHAPE, "multiple of 32", lambda: g("r", 256, 256, 1))
    refused(ffi.ERR_ARG, "quant_rows", lambda: dec.quant_rows(0, 256, 256, 1, 64))
    refused(ffi.ERR_ARG, "x type 3", lambda: dec.quant_rows(256, 256, 256, 1, 64, x_type=ffi.Q8))
    refused(ffi.ERR_SHAPE, "k=131072", lambda: dec.quant_rows(256, 256, 256, 1, 131072))
    refused(ffi.ERR_SHAPE, "ldx=5", lambda: dec.quant_rows(256, 256, 256, 2, 64, ldx=5))
    refused(ffi.ERR_ARG, "aligned", lambda: dec.quant_rows(256, 264, 256, 1, 64))
    refused(ffi.ERR_SHAPE, "hidden=8193", lambda: dec.norm_resid_q8(256, 256, 256, 256, 256, 1, 8193))
    refused(ffi.ERR_ARG, "null operand", lambda: dec.norm_resid_q8(256, 0, 256, 256, 256, 1, 64))
    refused(ffi.ERR_ARG, "aligned", lambda: dec.norm_resid_q8(256, 256, 256, 260, 256, 1, 64))
    refused(ffi.ERR_SHAPE, "upload_lin_w8a8", lambda: dec.upload_lin_w8a8("r", w, sb[:39], 40, 64))
    refused(ffi.ERR_SHAPE, "upload_lin_w8a8", lambda: dec.upload_lin_w8a8("r", w[:, :63], sb, 40, 64))
    refused(ffi.ERR_ARG, "int8", lambda: dec.upload_lin_w8a8("r", w.view(np.uint8), sb, 40, 64))
    refused(ffi.ERR_ARG, "int8", lambda: dec.upload_lin_w8a8("r", w, sb.astype(np.float64), 40, 64))
    q = np.zeros(8, np.int8)
    assert lib.w4a16_upload_lin_w8a8(dec.cc.h, b"r", q.ctypes.data, 8, q.ctypes.data, 4, 1, 8, 7) == ffi.ERR_ARG
    assert dec.lin_w8a8_spec("r") == {"n": 40, "k": 64}  # the refused uploads changed nothing


def test_new_weights_under_an_old_name(dec):
    """The new weights are the ones that run, and a graph that holds the old ones' address is refused."""
    n, k, t = 64, 256, 4
    x = np.random.default_rng(0).standard_normal((t, k)).astype(np.float32)
    cc = dec.cc
    with ref.Buffers(cc) as b:
        dx, y = b.put(x), b.filled(t * n * 4)
        wants = []
        for seed in (1, 2):
            w, sb, sv = ref.weights(seed, n, k)
            dec.upload_lin_w8a8("re", w, sb, n, k)
            wants.append(ref.product(*ref.quantised(x), w, sv).view(np.uint32))
            dec.lin_forward_w8a8("re", dx, y, t, x_type=ffi.F32)
            assert np.array_equal(cc.d2h(y, (t, n), np.uint32), wants[-1])
            if seed == 1:
                cc.capture_begin()
                dec.lin_forward_w8a8("re", dx, y, t, x_type=ffi.F32)
                graph = cc.capture_end()
        refused(ffi.ERR_STALE_GRAPH, "captured", graph.launch)
        graph.destroy()


def test_offsets_beyond_32_bits(dec):
    """Rows 2.2e9 elements apart on the way in; results of more than 4 GiB on the way out, by tiles."""
    k, n, cc = 1000, 32, dec.cc
    r = np.random.default_rng(8)
    x = r.standard_normal((3, k)).astype(np.float32)
    w, sb, sv = ref.weights(3, n, k)
    dec.upload_lin_w8a8("far", w, sb, n, k)
    want = ref.product(*ref.quantised(x), w, sv)
    ld = 550_000_000
    with ref.Buffers(cc) as b:
        wide, y = cc.alloc(4 * (2 * ld + k)), b.filled(3 * n * 4)
        try:
            for i in range(3):
                cc.h2d(wide + 4 * i * ld, x[i])
            dec.lin_forward_w8a8("far", wide, y, 3, x_type=ffi.F32, ldx=ld, y_type=ffi.F32)
            assert np.array_equal(cc.d2h(y, (3, n), np.float32), want)
        finally:
            cc.free(wide)
    t, n, k = 33000, 33000, 64
    w, sb, sv = ref.weights(4, n, k)
    dec.upload_lin_w8a8("far", w, sb, n, k)
    bits, x = ref.narrow(r.standard_normal((t, k)).astype(np.float32), ffi.F16)
    rows = [0, 1, 16270, 32535, 32540, t - 1]  # around 2^32 bytes, and the ends
    want = ref.product(*ref.quantised(x[rows]), w, sv)
    with ref.Buffers(cc) as b:
        dx, y = b.put(bits), cc.alloc(t * n * 4)
        try:
            dec.lin_forward_w8a8("far", dx, y, t, x_type=ffi.F16, y_type=ffi.F32)
            for i, row in enumerate(rows):
                assert np.array_equal(cc.d2h(y + row * n * 4, (n,), np.float32), want[i]), row
        finally:
            cc.free(y)


def test_captured_ffn_replays_the_eager_bits(dec):
    """norm, gated projection, down projection in one graph; replayed with eager work of other sizes in between, on new inputs."""
    h, f, cc = 384, 512, dec.cc
    w1, s1, v1 = ref.weights(1, 2 * f, h)
    w2, s2, v2 = ref.weights(2, h, f)
    dec.upload_lin_w8a8("ffn.gate_up", w1, s1, 2 * f, h)
    dec.upload_lin_w8a8("ffn.down", w2, s2, h, f)
    for t in (1, 3, 20, 90):
        r = np.random.default_rng(t)
        x, ab, nw = (r.standard_normal((t, h)).astype(np.float32) for _ in range(3))
        with ref.Buffers(cc) as b:
            dx, dab, dnw = b.put(x), b.put(ab), b.put(nw)
            q, s, a, y = b.filled(ops.q8_bytes(t, h)), b.filled(t * 4), b.filled(t * f * 2), b.filled(t * h * 4)

            def step():
                dec.norm_resid_q8(dx, dnw, dab, q, s, t, h)
                dec.lin_forward_w8a8_glu("ffn.gate_up", q, a, t, x_type=ffi.Q8, xs_dev=s, y_type=ffi.F16)
                dec.lin_forward_w8a8("ffn.down", a, y, t, x_type=ffi.F16, y_type=ffi.F32)

            step()
            # against the formulas, each linear on the rows that it was given
            rows, rs = read_quant(dec, q, s, t, h)
            gu = ref.product(rows, rs, w1, v1).astype(np.float64)
            act = gu[:, :f] / (1 + np.exp(-gu[:, :f])) * gu[:, f:]
            got = cc.d2h(a, (t, f), np.float16)
            # f32: exp, sum, quotient and product are each within two units of 2^-24, and exp adds |gate| roundings of its argument; f16: half a unit
            room = np.abs(act) * (2.0**-11 + (8 + np.abs(gu[:, :f])) * 2.0**-23) + 2.0**-25
            assert (np.abs(got.astype(np.float64) - act) <= room).all()
            want = ref.product(*ref.quantised(got.astype(np.float32)), w2, v2)
            assert np.array_equal(cc.d2h(y, (t, h), np.uint32), want.view(np.uint32))
            cc.capture_begin()
            step()
            graph = cc.capture_end()
            for i in range(3):
                cc.h2d(dx, x + i)
                graph.launch()
                replay = cc.d2h(y, (t, h), np.uint32)
                after = cc.d2h(dx, (t, h), np.uint32)
                cc.h2d(dx, x + i)
                step()
                assert np.array_equal(replay, cc.d2h(y, (t, h), np.uint32)) and np.array_equal(after, cc.d2h(dx, (t, h), np.uint32))
                small = b.filled(h * 4)
                dec.lin_forward_w8a8("ffn.down", a, small, 1, x_type=ffi.F16, y_type=ffi.F32)  # another call through the same scratch
                cc.sync()
            graph.destroy()


@pytest.mark.parametrize("t,n,k,gelu", [(16, 1024, 8000, None), (60, 640, 4096, False), (70, 512, 4096, None), (130, 2048, 8192, True), (200, 10000, 8000, None),
                                        (1100, 300, 4096, None), (1030, 256, 8000, False), (129, 6000, 4096, None)])
def test_captured_slices_of_k_replay_the_eager_bits(dec, t, n, k, gelu):
    """Slices hand their sums over through scratch and tickets that every call of the context shares: graphs and eager calls in turn."""
    cc = dec.cc
    w, sb, sv = ref.weights(n + k, n, k)
    dec.upload_lin_w8a8("big", w, sb, n, k)
    w2, sb2, sv2 = ref.weights(5, 256, 6000)
    dec.upload_lin_w8a8("other", w2, sb2, 256, 6000)
    r = np.random.default_rng(t)
    xs = [r.standard_normal((t, k)).astype(np.float32) for _ in range(3)]
    x2 = r.standard_normal((80, 6000)).astype(np.float32)
    out = n if gelu is None else n // 2
    with ref.Buffers(cc) as b:
        dx, y, dx2, y2 = b.put(xs[0]), b.filled(t * out * 4), b.put(x2), b.filled(80 * 256 * 4)

        def step():
            if gelu is None:
                dec.lin_forward_w8a8("big", dx, y, t, x_type=ffi.F32, y_type=ffi.F32)
            else:
                dec.lin_forward_w8a8_glu("big", dx, y, t, x_type=ffi.F32, y_type=ffi.F32, gelu=gelu)

        def other():
            dec.lin_forward_w8a8("other", dx2, y2, 80, x_type=ffi.F32, y_type=ffi.F32)

        step()
        other()
        cc.capture_begin()
        step()
        first = cc.capture_end()
        cc.capture_begin()
        other()
        step()
        second = cc.capture_end()
        want2 = ref.product(*ref.quantised(x2), w2, sv2)
        for x in xs:
            cc.h2d(dx, x)
            step()
            eager = cc.d2h(y, (t, out), np.float32)
            if gelu is None:
                assert np.array_equal(eager, ref.product(*ref.quantised(x), w, sv))
            for graph in (first, second, first):
                cc.h2d(y, np.zeros((t, out), np.float32))
                graph.launch()
                assert np.array_equal(cc.d2h(y, (t, out), np.float32), eager)
                other()
                assert np.array_equal(cc.d2h(y2, (80, 256), np.float32), want2)
        first.destroy()
        second.destroy()


def test_a_capture_that_would_grow_the_scratch_is_refused():
    dec = ops.W4a16Dec()
    try:
        w, sb, _ = ref.weights(1, 16, 64)
        dec.upload_lin_w8a8("c", w, sb, 16, 64)
        with ref.Buffers(dec.cc) as b:
            x, y = b.filled(100 * 64 * 2), b.filled(100 * 16 * 4)
            dec.lin_forward_w8a8("c", x, y, 2)
            dec.cc.capture_begin()
            refused(ffi.ERR_ARG, "capture", lambda: dec.lin_forward_w8a8("c", x, y, 100))
            refused(ffi.ERR_ARG, "captur", lambda: dec.upload_lin_w8a8("c", w, sb, 16, 64))
            dec.lin_forward_w8a8("c", x, y, 2)
            dec.cc.capture_end().destroy()
            dec.lin_forward_w8a8("c", x, y, 100)
            dec.cc.sync()
    finally:
        dec.cc.close()
