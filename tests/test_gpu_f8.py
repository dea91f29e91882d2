"""FP8 linears on the GPU: quantised rows and the fused norm bit for bit, products bit for bit where they are exact and within derived room where not."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import f8_ref as ref
from tests import w8a8_ref as w8
from tests.test_f8_cpu import shapes

pytestmark = pytest.mark.gpu
TYPES = [ffi.F32, ffi.F16, ffi.BF16]


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


def say(*a):
    print(*a, flush=True)


def blocks(k):
    return -(-k // 128)


def run_quant(dec, b, dev_x, t, k, kind, ldx=0):
    q, s = b.filled(ops.q8_bytes(t, k)), b.filled(t * blocks(k) * 4)
    dec.quant_rows_f8(dev_x, q, s, t, k, x_type=kind, ldx=ldx)
    return q, s


def read_quant(dec, q, s, t, k):
    return ops.unpack_q8(dec.cc.d2h(q, (ops.q8_bytes(t, k),), np.int8), t, k).view(np.uint8), dec.cc.d2h(s, (blocks(k), t), np.float32)


def same_rows(got, want):
    assert np.array_equal(np.isnan(got[1]), np.isnan(want[1])) and np.array_equal(np.nan_to_num(got[1]), np.nan_to_num(want[1]))
    assert np.array_equal(got[0], want[0])


# ------------------------------------------------------------------------------------------------ quantised rows
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("t,k", [(1, 1), (1, 17), (1, 5120), (1, 17408), (2, 16), (3, 2051), (4, 128), (4, 1300), (5, 33), (8, 129), (16, 4096), (17, 8193), (100, 1000),
                                 (129, 40000), (300, 96), (1, 131071), (2, 131071)])
def test_quant_rows_exactly(dec, t, k, kind):
    say("quant", t, k, kind)
    r = np.random.default_rng(t * 100003 + k)
    bits, x = w8.narrow(r.standard_normal((t, k)).astype(np.float32) * r.uniform(1e-3, 50, (t, 1)).astype(np.float32), kind)
    with w8.Buffers(dec.cc) as b:
        same_rows(read_quant(dec, *run_quant(dec, b, b.put(bits), t, k, kind), t, k), ref.quantised(x))


def test_quant_rows_halves_go_to_the_even_number(dec):
    """Every e4m3 number, every half between two, and the f32 numbers next to each half, in steps of 2^-100, 1 and 2^90."""
    pos = ref.E4M3[:127]
    half = ((pos[1:] + pos[:-1]) / 2).astype(np.float32)
    vals = np.concatenate([pos.astype(np.float32), half, np.nextafter(half, np.float32(1e9)), np.nextafter(half, np.float32(-1e9))])
    vals = np.concatenate([vals, -vals])
    vals = np.concatenate([vals, np.zeros(-len(vals) % 127, np.float32)]).reshape(-1, 127)
    rows = np.concatenate([np.concatenate([vals, np.full((len(vals), 1), 448, np.float32)], 1) * np.float32(2.0**e) for e in (-100, 0, 90)])
    t = len(rows)
    with w8.Buffers(dec.cc) as b:
        got = read_quant(dec, *run_quant(dec, b, b.put(rows.astype(np.float32)), t, 128, ffi.F32), t, 128)
    same_rows(got, ref.quantised(rows))
    assert set(got[1].reshape(-1)) == {np.float32(2.0**-100), 1.0, np.float32(2.0**90)}


def test_quant_rows_of_nothing_and_of_no_number(dec):
    k = 300
    x = np.random.default_rng(5).standard_normal((11, k)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= np.float32(1e-40)  # subnormal: the smallest step
    x[3, 7] = np.inf           # its block alone
    x[4, 299] = -np.inf
    x[5, 130] = np.nan
    x[6] = np.float32(3.4e38)
    x[7, :] = 0
    x[7, 100] = np.float32(2.0**-149)
    x[8, 128:] = 0
    x[9, :128] = np.float32(2.0**-126 * 448)
    x[10, :128] = np.nextafter(np.float32(2.0**-126 * 448), np.float32(1))
    with w8.Buffers(dec.cc) as b:
        got = read_quant(dec, *run_quant(dec, b, b.put(x), 11, k, ffi.F32), 11, k)
    want = ref.quantised(x)
    want[0][1] = got[0][1]  # zeros of either sign
    assert not ref.E4M3[got[0][1]].any()
    same_rows(got, want)
    assert np.isnan(got[1][0, 3]) and not np.isnan(got[1][1:, 3]).any() and not got[0][3, :128].any() and got[1][0, 9] == 2.0**-126 and got[1][0, 10] == 2.0**-125


@pytest.mark.parametrize("kind,t,k,ldx,off", [(ffi.F16, 5, 65, 67, 2), (ffi.BF16, 37, 2051, 2051, 2), (ffi.F32, 3, 33, 41, 4), (ffi.F16, 20, 512, 1027, 6),
                                              (ffi.F32, 1, 4099, 0, 12)])
def test_quant_rows_at_any_element_alignment_and_stride(dec, kind, t, k, ldx, off):
    ld = ldx or k
    bits, x = w8.narrow(np.random.default_rng(k).standard_normal((t, ld)).astype(np.float32), kind)
    flat = bits.reshape(-1)[:(t - 1) * ld + k]  # nothing behind the last row's last element
    with w8.Buffers(dec.cc) as b:
        same_rows(read_quant(dec, *run_quant(dec, b, b.put(flat, off), t, k, kind, ldx), t, k), ref.quantised(x[:, :k]))


@pytest.mark.parametrize("t,hidden", [(1, 7), (3, 100), (18, 1000), (5, 8185), (2, 16), (300, 2048), (17, 1025), (4, 8192), (6, 5117), (20, 4096), (3, 2049), (1, 5120), (2, 5124)])
def test_both_ways_to_quantised_rows_write_the_same_bytes(dec, t, hidden):
    """norm_resid_f8 against norm_resid and quant_rows_f8, of the whole buffer: elements, zeros behind a row's end inside its last block, and the bytes that neither
    touches; a row of no number among them."""
    r = np.random.default_rng(hidden)
    w_off = t % 3
    x, ab, nw = ((r.standard_normal(n) * 2).astype(np.float32) for n in ((t, hidden), (t, hidden), hidden + w_off))
    if t > 1:
        x[1, 3] = np.nan
    cc, n, m = dec.cc, ops.q8_bytes(t, hidden), t * blocks(hidden)
    with w8.Buffers(cc) as b:
        x1, x2, dab, dnw, xn, s2, q2 = b.put(x), b.put(x), b.put(ab), b.put(nw), b.filled(t * hidden * 4), b.filled(m * 4 + 32), b.filled(n + 32)
        dec.norm_resid(x1, dnw, dab, xn, t, hidden, w_off=w_off)
        q1, s1 = b.filled(n + 32), b.filled(m * 4 + 32)
        dec.quant_rows_f8(xn, q1, s1, t, hidden, x_type=ffi.F32)
        dec.norm_resid_f8(x2, dnw, dab, q2, s2, t, hidden, w_off=w_off)
        first, second = cc.d2h(q1, (n + 32,), np.uint8), cc.d2h(q2, (n + 32,), np.uint8)
        assert np.array_equal(cc.d2h(s1, (m + 8,), np.uint32), cc.d2h(s2, (m + 8,), np.uint32))
        assert np.array_equal(cc.d2h(x1, (t, hidden), np.uint32), cc.d2h(x2, (t, hidden), np.uint32))
        rows, s = read_quant(dec, q2, s2, t, hidden)
    assert np.array_equal(first, second) and (first[n:] == 0xA5).all()
    whole = blocks(hidden) * 128
    place = np.arange(n).reshape(-1, whole // 16, 1 if t == 1 else 4 if t <= 4 else 16, 16).transpose(0, 2, 1, 3).reshape(-1, whole)
    assert not first[place[:t, hidden:]].any() and (first[place[t:]] == 0xA5).all()
    # and near the formula in 64 bits: half a step of the number's own place, a thousandth of it for the 32-bit norm, where a value lies next to a border
    v = (x.astype(np.float64) + ab).astype(np.float32).astype(np.float64)
    want = v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6) * nw[w_off:]
    step = np.repeat(s.T.astype(np.float64), 128, 1)[:, :hidden]
    ok = np.arange(t) != 1
    off = np.abs(ref.E4M3[rows] * step - want)[ok]
    assert (off <= 0.501 * np.maximum(np.abs(want[ok]) / 8, step[ok] * 2.0**-9)).all()


# ------------------------------------------------------------------------------------------------ linears
@pytest.mark.parametrize("key", sorted(shapes()), ids=lambda k: k[0][10:] + ("_slices" if k[1] else ""))
def test_every_build(dec, key):
    """Bit for bit on whole numbers whose sums are exact; within their room on normal numbers."""
    t, n, k, glu, x_type, y_type = shapes()[key]
    kernel, cc = key[0], dec.cc
    say("build", key, t, n, k, glu, x_type, y_type)
    for whole in (True, False):
        if whole:
            q, s, w, sv = ref.small_whole(n + k, t, n, k)
            sb = sv
            x = (ref.E4M3[q] * np.repeat(s.T, 128, 1)[:, :k]).astype(np.float32)  # floats that quantise to what they are
            floats = x if x_type == ffi.F8 else w8.narrow(x, x_type)[0]
        else:
            floats, x = w8.narrow(np.random.default_rng(t).standard_normal((t, k)).astype(np.float32), ffi.F32 if x_type == ffi.F8 else x_type)
            q, s = ref.quantised(x)
            w, sb, sv = ref.weights(n * 5 + k, n, k)
        dec.upload_lin_f8("b", w, sb, n, k)
        assert dec.lin_f8_spec("b") == {"n": n, "k": k}
        want, a, most = ref.product(q, s, w, sv)
        size = 4 if y_type == ffi.F32 else 2
        with w8.Buffers(cc) as b:
            dq, ds = (b.put(ref.pack(q, t, k)), b.put(s)) if x_type == ffi.F8 else (b.put(floats, floats.itemsize), 0)
            y = b.filled(t * n * size + 64)
            for again in range(2):  # a second time over the same tickets
                if not glu:
                    dec.lin_forward_f8("b", dq, y, t, x_type=x_type, xs_dev=ds, y_type=y_type)
                    out, ran = n, cc.last_launch_symbol()
                    got = cc.d2h(y, (t, n), w8.bits_type(y_type))
                    if whole:
                        assert np.array_equal(got, w8.as_type(want.astype(np.float32), y_type))
                    else:
                        space = ref.room(a, most, ran, blocks(k))
                        ref.near(ref.value(got, y_type), want, space, y_type)
                        assert ref.rel_norm(ref.value(got, y_type), want) <= (1.1e-3 if "tiled" in ran else 2e-6) + ref.half_step(y_type)
                else:
                    dec.lin_forward_f8_glu("b", dq, y, t, x_type=x_type, xs_dev=ds, y_type=y_type, gelu=bool(again))
                    out, ran = n // 2, cc.last_launch_symbol()
                    got = cc.d2h(y, (t, out), w8.bits_type(y_type))
                    if whole and y_type == ffi.F16:  # the separate kernel's activation of the same f32 sums
                        act = b.filled(t * out * 2)
                        dec.act_mul_f16(b.put(want.astype(np.float32)), out, t, act, gelu=bool(again))
                        assert np.array_equal(got, cc.d2h(act, (t, out), np.uint16))
                    else:
                        g, u = want[:, :out], want[:, out:]
                        plain = (g / (1 + np.exp(-g)) if not again else 0.5 * g * (1 + np.tanh(0.7978846 * (g + 0.044715 * g**3)))) * u
                        space = np.zeros_like(want) if whole else ref.room(a, most, ran, blocks(k))
                        dg, du = space[:, :out], space[:, out:]
                        # the activation's slope is below 1.13; f32: exp or tanh, sums, quotient and product, each within two units, exp with the
                        # argument's roundings too; 1 + tanh cancels to units of 2^-24 of one
                        act_room = (np.abs(plain) * (16 + 2 * np.abs(g)) + np.abs(g * u) * 4) * 2.0**-24
                        ref.near(ref.value(got, y_type), plain, 1.13 * dg * (np.abs(u) + du) + 1.13 * np.abs(g) * du + act_room, y_type)
                assert ran == kernel
                assert (cc.d2h(y + t * out * size, (64,), np.uint8) == 0xA5).all()  # nothing behind the last row


@pytest.mark.parametrize("t,n,k", [(1, 1, 1), (1, 16, 128), (2, 33, 130), (3, 100, 77), (4, 512, 2048), (5, 48, 63), (7, 17, 4000), (16, 512, 17408), (17, 40, 300), (64, 700, 1500),
                                   (65, 1, 1), (65, 256, 128), (100, 513, 1000), (129, 300, 64), (300, 520, 2051), (1000, 257, 129), (2049, 1030, 256), (70, 300, 9000),
                                   (1, 130, 131071), (66, 129, 131071)])
def test_linear_of_floats(dec, t, n, k):
    say("linear", t, n, k)
    w, sb, sv = ref.weights(n * 7 + k, n, k)
    bits, x = w8.narrow(np.random.default_rng(t).standard_normal((t, k)).astype(np.float32), ffi.F16)
    dec.upload_lin_f8("l", w, sb, n, k)
    want, a, most = ref.product(*ref.quantised(x), w, sv)
    with w8.Buffers(dec.cc) as b:
        dx = b.put(bits)
        for y_type in TYPES:
            y = b.filled(t * n * 4 + 64)
            dec.lin_forward_f8("l", dx, y, t, x_type=ffi.F16, y_type=y_type)
            got = dec.cc.d2h(y, (t, n), w8.bits_type(y_type))
            ref.near(ref.value(got, y_type), want, ref.room(a, most, dec.cc.last_launch_symbol(), blocks(k)), y_type)
            assert (dec.cc.d2h(y + got.nbytes, (64,), np.uint8) == 0xA5).all()
            y2 = b.filled(t * n * 4)
            dec.lin_forward_f8("l", dx, y2, t, x_type=ffi.F16, y_type=y_type)
            assert np.array_equal(dec.cc.d2h(y2, (t, n), w8.bits_type(y_type)), got)  # the same bits


@pytest.mark.parametrize("t,n,k,glu", [(4, 131072, 5120, False), (16, 5120, 17408, False), (64, 34816, 5120, True), (300, 34816, 5120, True), (300, 5120, 17408, False)])
def test_layers_and_a_head_of_full_size(dec, t, n, k, glu):
    """What the wide layers and heads of a model launch, at 1000 of the outputs and the ends, on whole numbers: bit for bit."""
    say("layer", t, n, k, glu)
    q, s, w, sv = ref.small_whole(3, t, n, k)
    dec.upload_lin_f8("layer", w, sv, n, k)
    out = n // 2 if glu else n
    at = np.unique(np.concatenate([[0, out - 1], np.random.default_rng(1).integers(0, out, 1000)]))
    rows = np.concatenate([at, at + out]) if glu else at
    scale = np.repeat(sv[rows // 128], 128, 1)[:, :k]  # powers of two on whole numbers: in f64 exact
    want = ((ref.E4M3[q] * np.repeat(s.T, 128, 1)[:, :k]) @ (ref.E4M3[w[rows]] * scale).T).astype(np.float32)
    with w8.Buffers(dec.cc) as b:
        dq, ds, y = b.put(ref.pack(q, t, k)), b.put(s), b.filled(t * out * 4)
        if glu:
            dec.lin_forward_f8_glu("layer", dq, y, t, x_type=ffi.F8, xs_dev=ds, y_type=ffi.F16)
            got, act = dec.cc.d2h(y, (t, out), np.uint16)[:, at], b.filled(t * len(at) * 2)
            dec.act_mul_f16(b.put(want), len(at), t, act)
            assert np.array_equal(got, dec.cc.d2h(act, (t, len(at)), np.uint16))
        else:
            dec.lin_forward_f8("layer", dq, y, t, x_type=ffi.F8, xs_dev=ds, y_type=ffi.F32)
            assert np.array_equal(dec.cc.d2h(y, (t, out), np.float32)[:, at], want)


@pytest.mark.parametrize("t", [1, 3, 16, 40, 65, 200])
def test_linear_on_quantised_rows_and_on_rows_of_floats(dec, t):
    """The same bits either way, with a stride, of every type, through several linears of one q, with every type of scale."""
    n, k, ld = 200, 777, 801
    r = np.random.default_rng(t)
    for kind in TYPES:
        bits, x = w8.narrow(r.standard_normal((t, ld)).astype(np.float32), kind)
        q, s = ref.quantised(x[:, :k])
        with w8.Buffers(dec.cc) as b:
            dx = b.put(bits.reshape(-1)[:(t - 1) * ld + k])
            dq, ds = run_quant(dec, b, dx, t, k, kind, ld)
            for i, s_kind in enumerate(TYPES):
                w, sb, sv = ref.weights(i, n, k, s_kind)
                dec.upload_lin_f8("p%d" % i, w, sb, n, k)
                want, a, most = ref.product(q, s, w, sv)
                got = []
                for xd, x_type, xs, ldx in ((dq, ffi.F8, ds, 0), (dx, kind, 0, ld)):
                    y = b.filled(t * n * 4)
                    dec.lin_forward_f8("p%d" % i, xd, y, t, x_type=x_type, xs_dev=xs, ldx=ldx, y_type=ffi.F32)
                    got.append(dec.cc.d2h(y, (t, n), np.float32))
                assert np.array_equal(got[0], got[1])
                ref.near(got[0], want, ref.room(a, most, "", blocks(k)), ffi.F32)


@pytest.mark.parametrize("y_type", [ffi.F32, ffi.BF16])
@pytest.mark.parametrize("t", [2, 17, 66, 300])
def test_rows_with_no_number_and_scales_of_any_size(dec, t, y_type):
    """NaN stays in its row; so do a scale of 2^100 and one of 2^-100, and the zeros of an empty block."""
    n, k, cc = 70, 400, dec.cc
    q, s, w, sv = ref.small_whole(1, t, n, k)
    x = (ref.E4M3[q] * np.repeat(s.T, 128, 1)[:, :k]).astype(np.float32)
    x[0] *= np.float32(2.0**100)
    x[1, 3] = np.nan
    if t > 2:
        x[2] *= np.float32(2.0**-100)
        x[3, :] = 0
        x[4, 128:256] = 0
        x[5, 399] = -np.inf
    dec.upload_lin_f8("nan", w, sv, n, k)
    q, s = ref.quantised(x)
    want, _, _ = ref.product(q, np.nan_to_num(s), w, sv)
    with w8.Buffers(cc) as b:
        y = b.filled(t * n * 4)
        dec.lin_forward_f8("nan", b.put(x), y, t, x_type=ffi.F32, y_type=y_type)
        got = cc.d2h(y, (t, n), w8.bits_type(y_type))
    bad = np.isnan(s).any(0)
    assert np.isnan(ref.value(got[bad], y_type)).all() and bad.sum() == (1 if t == 2 else 2)
    # a row's numbers were steps of one scale for a block: still whole numbers times powers of two, 2^8 apart at most, and exact
    assert np.array_equal(got[~bad], w8.as_type(want[~bad].astype(np.float32), y_type))


def test_weights_that_are_no_number_stay_in_their_rows(dec):
    n, k, cc = 150, 200, dec.cc
    for t in (3, 100):
        q, s, w, sv = ref.small_whole(2, t, n, k)
        w[17, 150] = 0x7f
        dec.upload_lin_f8("wn", w, sv, n, k)
        w[17, 150] = 0
        want = ref.product(q, s, w, sv)[0].astype(np.float32)
        for y_type in (ffi.F32, ffi.F16):
            with w8.Buffers(cc) as b:
                y = b.filled(t * n * 4)
                dec.lin_forward_f8("wn", b.put(ref.pack(q, t, k)), y, t, x_type=ffi.F8, xs_dev=b.put(s), y_type=y_type)
                got = cc.d2h(y, (t, n), w8.bits_type(y_type))
            keep = np.arange(n) != 17
            assert np.isnan(ref.value(got, y_type)[:, 17]).all() and np.array_equal(got[:, keep], w8.as_type(want, y_type)[:, keep])


def test_results_at_any_element_alignment(dec):
    n, k = 37, 128
    for t in (3, 20, 80):
        q, s, w, sv = ref.small_whole(t, t, n, k)
        dec.upload_lin_f8("al", w, sv, n, k)
        want = ref.product(q, s, w, sv)[0].astype(np.float32)
        for y_type, off in ((ffi.F16, 2), (ffi.BF16, 6), (ffi.F32, 4)):
            with w8.Buffers(dec.cc) as b:
                y = b.filled(t * n * 4, offset=off)
                dec.lin_forward_f8("al", b.put(ref.pack(q, t, k)), y, t, x_type=ffi.F8, xs_dev=b.put(s, 4), y_type=y_type)
                assert np.array_equal(dec.cc.d2h(y, (t, n), w8.bits_type(y_type)), w8.as_type(want, y_type))


@pytest.mark.parametrize("k,tiles", [(300, False), (1024, True)])
@pytest.mark.parametrize("t", [17, 33, 64])
def test_wide_linears_of_few_rows(dec, t, k, tiles):
    """17 to 64 rows go to tiles, most of whose rows are not there, where k is long enough for them."""
    n, cc = 65536 + 40, dec.cc
    q, s, w, sv = ref.small_whole(t, t, n, k)
    dec.upload_lin_f8("wide", w, sv, n, k)
    want = ref.product(q, s, w, sv)[0].astype(np.float32)
    with w8.Buffers(cc) as b:
        y = b.filled(t * n * 2 + 64)
        dec.lin_forward_f8("wide", b.put(ref.pack(q, t, k)), y, t, x_type=ffi.F8, xs_dev=b.put(s), y_type=ffi.F16)
        assert not tiles or "exact" in cc.last_launch_symbol()
        assert np.array_equal(cc.d2h(y, (t, n), np.uint16), w8.as_type(want, ffi.F16)) and (cc.d2h(y + t * n * 2, (64,), np.uint8) == 0xA5).all()


def refused(code, words, call):
    with pytest.raises(ops.W4a16Error) as e:
        call()
    assert e.value.code == code and words in e.value.message, e.value.message


def test_refusals(dec):
    w, sb, _ = ref.weights(1, 140, 64)
    dec.upload_lin_f8("r", w, sb, 140, 64)
    f, g, lib = dec.lin_forward_f8, dec.lin_forward_f8_glu, dec.cc.lib
    refused(ffi.ERR_NOT_FOUND, "not registered", lambda: f("absent", 256, 256, 1))
    refused(ffi.ERR_NOT_FOUND, "not registered", lambda: dec.lin_forward_w8a8("r", 256, 256, 1))  # a name space of its own
    refused(ffi.ERR_ARG, "null operand", lambda: f("r", 0, 256, 1))
    refused(ffi.ERR_ARG, "null operand", lambda: f("r", 256, 0, 1))
    refused(ffi.ERR_SHAPE, "t=0", lambda: f("r", 256, 256, 0))
    refused(ffi.ERR_ARG, "x type 3", lambda: f("r", 256, 256, 1, x_type=ffi.Q8, xs_dev=256))
    refused(ffi.ERR_ARG, "y type 3", lambda: f("r", 256, 256, 1, y_type=3))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.F8))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.F8, xs_dev=256, ldx=64))
    refused(ffi.ERR_ARG, "scales", lambda: f("r", 256, 256, 1, x_type=ffi.F16, xs_dev=256))
    refused(ffi.ERR_SHAPE, "ldx=63", lambda: f("r", 256, 256, 2, ldx=63))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 257, 256, 1))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 256, 258, 1, y_type=ffi.F32))
    refused(ffi.ERR_ARG, "aligned", lambda: f("r", 264, 256, 1, x_type=ffi.F8, xs_dev=256))
    refused(ffi.ERR_SHAPE, "multiple of 256", lambda: g("r", 256, 256, 1))
    refused(ffi.ERR_ARG, "quant_rows_f8", lambda: dec.quant_rows_f8(0, 256, 256, 1, 64))
    refused(ffi.ERR_ARG, "x type 4", lambda: dec.quant_rows_f8(256, 256, 256, 1, 64, x_type=ffi.F8))
    refused(ffi.ERR_SHAPE, "k=131072", lambda: dec.quant_rows_f8(256, 256, 256, 1, 131072))
    refused(ffi.ERR_SHAPE, "ldx=5", lambda: dec.quant_rows_f8(256, 256, 256, 2, 64, ldx=5))
    refused(ffi.ERR_ARG, "aligned", lambda: dec.quant_rows_f8(256, 264, 256, 1, 64))
    refused(ffi.ERR_SHAPE, "hidden=8193", lambda: dec.norm_resid_f8(256, 256, 256, 256, 256, 1, 8193))
    refused(ffi.ERR_ARG, "null operand", lambda: dec.norm_resid_f8(256, 0, 256, 256, 256, 1, 64))
    refused(ffi.ERR_ARG, "aligned", lambda: dec.norm_resid_f8(256, 256, 256, 260, 256, 1, 64))
    refused(ffi.ERR_SHAPE, "upload_lin_f8", lambda: dec.upload_lin_f8("r", w, sb[:1], 140, 64))
    refused(ffi.ERR_SHAPE, "upload_lin_f8", lambda: dec.upload_lin_f8("r", w[:, :63], sb, 140, 64))
    refused(ffi.ERR_ARG, "uint8", lambda: dec.upload_lin_f8("r", w.view(np.int8), sb, 140, 64))
    refused(ffi.ERR_ARG, "uint8", lambda: dec.upload_lin_f8("r", w, sb.astype(np.float64), 140, 64))
    q = np.zeros(8, np.uint8)
    assert lib.w4a16_upload_lin_f8(dec.cc.h, b"r", q.ctypes.data, 8, q.ctypes.data, 4, 1, 8, 7) == ffi.ERR_ARG
    assert dec.lin_f8_spec("r") == {"n": 140, "k": 64}  # the refused uploads changed nothing


def test_new_weights_under_an_old_name(dec):
    """The new weights are the ones that run, and a graph that holds the old ones' address is refused."""
    n, k, t, cc = 64, 256, 4, dec.cc
    with w8.Buffers(cc) as b:
        for seed in (1, 2):
            q, s, w, sv = ref.small_whole(seed, t, n, k)
            dq, ds, y = b.put(ref.pack(q, t, k)), b.put(s), b.filled(t * n * 4)
            dec.upload_lin_f8("re", w, sv, n, k)
            dec.lin_forward_f8("re", dq, y, t, x_type=ffi.F8, xs_dev=ds)
            assert np.array_equal(cc.d2h(y, (t, n), np.float32), ref.product(q, s, w, sv)[0].astype(np.float32))
            if seed == 1:
                cc.capture_begin()
                dec.lin_forward_f8("re", dq, y, t, x_type=ffi.F8, xs_dev=ds)
                graph = cc.capture_end()
        refused(ffi.ERR_STALE_GRAPH, "captured", graph.launch)
        graph.destroy()


def test_offsets_beyond_32_bits(dec):
    """Rows 2.2e9 elements apart on the way in; results of more than 4 GiB on the way out, by tiles of either product."""
    k, n, cc = 1000, 32, dec.cc
    q, s, w, sv = ref.small_whole(8, 3, n, k)
    x = (ref.E4M3[q] * np.repeat(s.T, 128, 1)[:, :k]).astype(np.float32)
    dec.upload_lin_f8("far", w, sv, n, k)
    want = ref.product(q, s, w, sv)[0].astype(np.float32)
    ld = 550_000_000
    with w8.Buffers(cc) as b:
        wide, y = cc.alloc(4 * (2 * ld + k)), b.filled(3 * n * 4)
        try:
            for i in range(3):
                cc.h2d(wide + 4 * i * ld, x[i])
            dec.lin_forward_f8("far", wide, y, 3, x_type=ffi.F32, ldx=ld, y_type=ffi.F32)
            assert np.array_equal(cc.d2h(y, (3, n), np.float32), want)
        finally:
            cc.free(wide)
    for t, y_type in ((33000, ffi.F32), (66000, ffi.F16)):
        n, k = 33000, 64
        q, s, w, sv = ref.small_whole(4, t, n, k)
        dec.upload_lin_f8("far", w, sv, n, k)
        size = 4 if y_type == ffi.F32 else 2
        joint = 2**32 // (n * size)
        rows = [0, 1, joint // 2, joint, joint + 1, t - 1]  # around 2^32 bytes, and the ends
        want = w8.as_type(ref.product(q[rows], s[:, rows], w, sv)[0].astype(np.float32), y_type)
        with w8.Buffers(cc) as b:
            dq, ds, y = b.put(ref.pack(q, t, k)), b.put(s), cc.alloc(t * n * size)
            try:
                dec.lin_forward_f8("far", dq, y, t, x_type=ffi.F8, xs_dev=ds, y_type=y_type)
                for i, row in enumerate(rows):
                    assert np.array_equal(cc.d2h(y + row * n * size, (n,), w8.bits_type(y_type)), want[i]), row
            finally:
                cc.free(y)


@pytest.mark.parametrize("t,n,k,gelu,y_type", [(16, 1024, 8000, None, ffi.F16), (60, 768, 4096, False, ffi.F32), (70, 512, 4096, None, ffi.F32), (130, 2048, 8192, True, ffi.F16),
                                               (200, 10000, 8000, None, ffi.BF16), (1100, 300, 4096, None, ffi.F16), (1030, 256, 8000, False, ffi.F32)])
def test_captured_slices_of_k_replay_the_eager_bits(dec, t, n, k, gelu, y_type):
    """Slices hand their sums over through scratch and tickets that every call of the context shares, W8A8's among them: graphs and eager calls in turn."""
    cc = dec.cc
    w, sb, sv = ref.weights(n + k, n, k)
    dec.upload_lin_f8("big", w, sb, n, k)
    w2, sb2, sv2 = w8.weights(5, 256, 6000)
    dec.upload_lin_w8a8("other", w2, sb2, 256, 6000)
    r = np.random.default_rng(t)
    xs = [r.standard_normal((t, k)).astype(np.float32) for _ in range(2)]
    x2 = r.standard_normal((80, 6000)).astype(np.float32)
    out = n if gelu is None else n // 2
    with w8.Buffers(cc) as b:
        dx, y, dx2, y2 = b.put(xs[0]), b.filled(t * out * 4), b.put(x2), b.filled(80 * 256 * 4)

        def step():
            if gelu is None:
                dec.lin_forward_f8("big", dx, y, t, x_type=ffi.F32, y_type=y_type)
            else:
                dec.lin_forward_f8_glu("big", dx, y, t, x_type=ffi.F32, y_type=y_type, gelu=gelu)

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
        want2 = w8.product(*w8.quantised(x2), w2, sv2)
        for x in xs:
            cc.h2d(dx, x)
            step()
            eager = cc.d2h(y, (t, out), w8.bits_type(y_type))
            if gelu is None:
                want, a, most = ref.product(*ref.quantised(x), w, sv)
                ref.near(ref.value(eager, y_type), want, ref.room(a, most, cc.last_launch_symbol(), blocks(k)), y_type)
            for graph in (first, second, first):
                cc.h2d(y, np.zeros(t * out * 4, np.uint8))
                graph.launch()
                assert np.array_equal(cc.d2h(y, (t, out), w8.bits_type(y_type)), eager)
                other()
                assert np.array_equal(cc.d2h(y2, (80, 256), np.float32), want2)
        first.destroy()
        second.destroy()


def test_captured_ffn_replays_the_eager_bits(dec):
    """norm, gated projection, down projection in one graph; replayed with eager work of other sizes in between, on new inputs."""
    h, f, cc = 384, 512, dec.cc
    w1, s1, v1 = ref.weights(1, 2 * f, h)
    w2, s2, v2 = ref.weights(2, h, f)
    dec.upload_lin_f8("ffn.gate_up", w1, s1, 2 * f, h)
    dec.upload_lin_f8("ffn.down", w2, s2, h, f)
    for t in (1, 3, 20, 90):
        r = np.random.default_rng(t)
        x, ab, nw = (r.standard_normal((t, h)).astype(np.float32) for _ in range(3))
        with w8.Buffers(cc) as b:
            dx, dab, dnw = b.put(x), b.put(ab), b.put(nw)
            q, s, a, y = b.filled(ops.q8_bytes(t, h)), b.filled(t * blocks(h) * 4), b.filled(t * f * 2), b.filled(t * h * 4)

            def step():
                dec.norm_resid_f8(dx, dnw, dab, q, s, t, h)
                dec.lin_forward_f8_glu("ffn.gate_up", q, a, t, x_type=ffi.F8, xs_dev=s, y_type=ffi.F16)
                dec.lin_forward_f8("ffn.down", a, y, t, x_type=ffi.F16, y_type=ffi.F32)

            step()
            # against the formulas, the down projection on the rows that it was given
            got = cc.d2h(a, (t, f), np.float16)
            want, sums, most = ref.product(*ref.quantised(got.astype(np.float32)), w2, v2)
            ref.near(cc.d2h(y, (t, h), np.float32), want, ref.room(sums, most, "", blocks(f)), ffi.F32)
            cc.capture_begin()
            step()
            graph = cc.capture_end()
            for i in range(3):
                cc.h2d(dx, x + i)
                graph.launch()
                replay, after = cc.d2h(y, (t, h), np.uint32), cc.d2h(dx, (t, h), np.uint32)
                cc.h2d(dx, x + i)
                step()
                assert np.array_equal(replay, cc.d2h(y, (t, h), np.uint32)) and np.array_equal(after, cc.d2h(dx, (t, h), np.uint32))
                small = b.filled(h * 4)
                dec.lin_forward_f8("ffn.down", a, small, 1, x_type=ffi.F16, y_type=ffi.F32)  # another call through the same scratch
                cc.sync()
            graph.destroy()


def test_a_capture_that_would_grow_the_scratch_is_refused():
    dec = ops.W4a16Dec()
    try:
        w, sb, _ = ref.weights(1, 16, 64)
        dec.upload_lin_f8("c", w, sb, 16, 64)
        with w8.Buffers(dec.cc) as b:
            x, y = b.filled(100 * 64 * 2), b.filled(100 * 16 * 4)
            dec.lin_forward_f8("c", x, y, 2)
            dec.cc.capture_begin()
            refused(ffi.ERR_ARG, "capture", lambda: dec.lin_forward_f8("c", x, y, 100))
            refused(ffi.ERR_ARG, "captur", lambda: dec.upload_lin_f8("c", w, sb, 16, 64))
            dec.lin_forward_f8("c", x, y, 2)
            dec.cc.capture_end().destroy()
            dec.lin_forward_f8("c", x, y, 100)
            dec.cc.sync()
    finally:
        dec.cc.close()


def near_the_joints(t, step):
    last = (t - 48) // 16 * 16
    return sorted({0, last} | {min(max(0, at // 16 * 16 - 16), last) for j in range(1, t // step + 1) for at in (step * j, step * j + 128)})


def test_more_rows_than_a_launch_of_the_norm_has(dec):
    cc, h, t = dec.cc, 4, 2**24 + 77  # workgroups of 256 threads
    r = np.random.default_rng(2)
    x, ab, nw = (r.standard_normal(n, dtype=np.float32) for n in (t * h, t * h, h))
    with w8.Buffers(cc) as b:
        dx, dab, dnw, s, q = b.put(x), b.put(ab), b.put(nw), b.filled(t * 4), b.filled(ops.q8_bytes(t, h))
        dec.norm_resid_f8(dx, dnw, dab, q, s, t, h)
        assert np.array_equal(cc.d2h(dx, (t * h,), np.float32), x + ab)
        steps = cc.d2h(s, (t,), np.float32)
        for at in near_the_joints(t, 2**24 - 128):
            n = min(48, t - at)
            x1, q1, s1 = b.put(x[at * h:(at + n) * h]), b.filled(ops.q8_bytes(n, h)), b.filled(n * 4)
            dec.norm_resid_f8(x1, dnw, dab + at * h * 4, q1, s1, n, h)
            rows = ops.unpack_q8(cc.d2h(q + at * 128, (ops.q8_bytes(n, h),), np.int8), n, h)
            assert np.array_equal(steps[at:at + n], cc.d2h(s1, (n,), np.float32)), at
            assert np.array_equal(rows, ops.unpack_q8(cc.d2h(q1, (ops.q8_bytes(n, h),), np.int8), n, h)), at
