"""Norm and rotation of queries and keys on the GPU against the formulas in 64 bits.

Room, with u = 2^-24: the sum of squares of d elements loses at most (d + 8) u of itself, the reciprocal root half of that and 3 u, the two products 2 u: (d / 2 + 10) u of a normed
element.  An angle is off by 2^-24 of a half turn, 1.9e-7 at most, sine and cosine by two units more, times amp; a pair turns with three roundings: of the pair's size, 1.9e-7 + 7 u.  Then the
result's own rounding."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import f8_ref
from tests import w8a8_ref as w8

pytestmark = pytest.mark.gpu
TYPES = [ffi.F32, ffi.F16, ffi.BF16]
U = 2.0**-24


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


def plain(x, t, heads, dim, w, eps, pos, freqs, amp, interleaved):
    """(heads [t][heads][dim] in 64 bits, room of each element)"""
    v = x.reshape(t, heads, dim).astype(np.float64)
    rel = 0.0
    if w is not None:
        v = v / np.sqrt((v * v).mean(2, keepdims=True) + np.float32(eps).astype(np.float64)) * w
        rel = (dim / 2 + 10) * U
    space = np.abs(v) * rel
    half = len(freqs)
    if half:
        at = np.arange(2 * half)
        a, b = (at[0::2], at[1::2]) if interleaved else (at[:half], at[half:])
        angle = pos.astype(np.float64)[:, None] * freqs[None]
        cos, sin = (np.float32(amp) * f(angle)[:, None] for f in (np.cos, np.sin))
        x0, x1 = v[:, :, a].copy(), v[:, :, b].copy()
        v[:, :, a], v[:, :, b] = x0 * cos - x1 * sin, x1 * cos + x0 * sin
        # far positions: what 64 bits hold of an angle
        far = np.abs(angle)[:, None] * 2.0**-51
        size = (np.abs(x0) + np.abs(x1)) * np.abs(amp)
        space[:, :, a] = space[:, :, b] = size * (rel + 1.9e-7 + 7 * U + far)
    return v, space


def run(dec, kind, y_type, t, nq, nk, dim, rot, interleaved=False, norm=True, rest=0, scaling=ffi.ROPE_PLAIN, start=0, in_place=False, gaps=0, off=0, pos=None, x=None, eps=1e-6):
    r = np.random.default_rng(t * 31 + dim + rot)
    cols = (nq + nk) * dim
    ldx = cols + rest
    bits, val = w8.narrow((r.standard_normal((t, ldx)) * 2).astype(np.float32) if x is None else x, kind)
    qw, kw = ((1 + 0.3 * r.standard_normal(dim)).astype(np.float32) for _ in range(2))
    if norm == "q":
        kw = None
    if not norm:
        qw = kw = None
    pos = np.arange(start, start + t, dtype=np.int32) if pos is None else np.asarray(pos, np.int32)
    freqs, amp = ops.rope_freqs(rot, 10000.0, scaling, 8.0, 4096.0, 1.0, 4.0 if scaling == ffi.ROPE_BANDS else 32.0) if rot else (np.zeros(0), 1.0)
    cc, size = dec.cc, 4 if y_type == ffi.F32 else 2
    with w8.Buffers(cc) as b:
        flat = bits.reshape(-1)[:(t - 1) * ldx + cols] if rest else bits
        dx = b.put(flat, off)
        if in_place:
            q, k, ldq, ldk = dx, dx + nq * dim * size, ldx, ldx
        else:
            ldq, ldk = nq * dim + gaps, nk * dim + gaps
            q, k = b.filled(t * ldq * size + 64, offset=off), b.filled(t * ldk * size + 64, offset=off)
        dec.qk_norm_rope(dx, q if nq else 0, k if nk else 0, b.put(pos) if rot else 0, b.put(freqs) if rot else 0, t, nq, nk, dim, rot, x_type=kind, ldx=ldx if rest else 0,
                         y_type=y_type, ldq=ldq if gaps or in_place else 0, ldk=ldk if gaps or in_place else 0, qw_dev=b.put(qw) if qw is not None else 0,
                         kw_dev=b.put(kw) if kw is not None else 0, eps=eps, amp=amp, interleaved=interleaved)
        got = []
        for p, heads, ld, w, first in ((q, nq, ldq, qw, 0), (k, nk, ldk, kw, nq)):
            if not heads:
                continue
            n = (t - 1) * ld + heads * dim
            rows = np.zeros(t * ld, w8.bits_type(y_type))
            rows[:n] = cc.d2h(p, (n,), w8.bits_type(y_type))
            rows = rows.reshape(t, ld)
            if gaps:
                assert (rows[:-1, heads * dim:].view(np.uint8) == 0xA5).all()
            if in_place and first + heads == nq + nk and rest:
                assert np.array_equal(rows[:-1, heads * dim:heads * dim + rest], bits[:-1, cols:].view(w8.bits_type(y_type)))  # what the row holds besides
            if not in_place:
                assert (cc.d2h(p + n * size, (64,), np.uint8) == 0xA5).all()
            want, space = plain(val[:, first * dim:(first + heads) * dim], t, heads, dim, w, eps, pos, freqs, amp, interleaved)
            value = f8_ref.value(np.ascontiguousarray(rows[:, :heads * dim]), y_type).reshape(t, heads, dim)
            got.append((value, want, space))
    return got


def near(dec, kind, y_type, *a, **k):
    for value, want, space in run(dec, kind, y_type, *a, **k):
        f8_ref.near(value, want, space, y_type)


# (t, n_q, n_k, head_dim, rot_dim): units of 8, 2 and 1 pairs, whole heads and parts, heads of one element, more heads than lanes, many units of a lane
SHAPES = [(1, 1, 1, 2, 2), (1, 40, 8, 128, 128), (3, 5, 2, 64, 64), (7, 13, 3, 80, 20), (2, 3, 1, 96, 96), (5, 2, 2, 256, 64), (4, 3, 3, 6, 4), (9, 2, 1, 7, 2), (2, 1, 0, 1024, 1024),
          (2, 0, 3, 1022, 1022), (3, 2, 1, 1023, 510), (33, 70, 5, 16, 16), (2, 4, 4, 128, 0), (6, 3, 2, 1, 0), (2, 2, 2, 1024, 6), (300, 8, 2, 128, 64), (1, 33, 1, 34, 34), (4500, 3, 1, 32, 32),
          (17, 6, 2, 72, 36)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,nq,nk,dim,rot", SHAPES)
def test_every_type_and_layout(dec, t, nq, nk, dim, rot, interleaved):
    print("rope", t, nq, nk, dim, rot, interleaved, flush=True)
    for kind in TYPES:
        for y_type in TYPES:
            near(dec, kind, y_type, t, nq, nk, dim, rot, interleaved, start=t * 1000)
    if rot:
        near(dec, ffi.F16, ffi.F32, t, nq, nk, dim, rot, interleaved, norm=False)
        near(dec, ffi.BF16, ffi.BF16, t, nq, nk, dim, rot, interleaved, norm="q", rest=5, gaps=3)


@pytest.mark.parametrize("scaling", [ffi.ROPE_PLAIN, ffi.ROPE_LINEAR, ffi.ROPE_BANDS, ffi.ROPE_RAMP])
def test_far_positions_and_scaled_frequencies(dec, scaling):
    near(dec, ffi.F32, ffi.F32, 5, 4, 2, 128, 128, scaling=scaling, pos=[0, 1, 100003, 2**31 - 1, -7])
    near(dec, ffi.F32, ffi.F32, 5, 4, 2, 96, 32, True, scaling=scaling, pos=[2**31 - 1, -2**31, 999999, 5, 5])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,rot,off", [(128, 128, 0), (80, 20, 2), (7, 4, 6), (66, 66, 2)])
def test_in_place_with_the_rest_of_the_row_left(dec, kind, dim, rot, off):
    off = off * 2 if kind == ffi.F32 else off
    for interleaved in (False, True):
        near(dec, kind, kind, 37, 5, 2, dim, rot, interleaved, rest=9, in_place=True, off=off)


def test_element_alignment_and_gaps(dec):
    for kind, y_type, off in ((ffi.F16, ffi.F16, 2), (ffi.BF16, ffi.F16, 6), (ffi.F32, ffi.F32, 4), (ffi.F16, ffi.BF16, 10)):
        near(dec, kind, y_type, 11, 3, 2, 128, 64, off=off, gaps=5, rest=3)
        near(dec, kind, y_type, 11, 3, 2, 128, 64, True, off=off, gaps=1, rest=1, norm=False)


def test_heads_of_zeros_and_of_no_number_stay_alone(dec):
    t, nq, nk, dim = 4, 3, 2, 64
    x = np.random.default_rng(0).standard_normal((t, 5 * dim)).astype(np.float32)
    x[0, :dim] = 0
    x[1, dim + 3] = np.nan
    x[2, 3 * dim + 63] = np.inf
    x[3] *= np.float32(1e15)
    x[0, 4 * dim:] *= np.float32(1e-18)
    (q, wq, sq), (k, wk, sk) = run(dec, ffi.F32, ffi.F32, t, nq, nk, dim, 64, x=x)
    assert not q[0, 0].any() and np.isnan(q[1, 1]).any() and np.isnan(k[2, 0]).any()
    for got, want, space, skip in ((q, wq, sq, (1, 1)), (k, wk, sk, (2, 0))):
        got, want, space = (a.copy() for a in (got, want, space))
        for a in (got, want, space):
            a[skip] = 0
        f8_ref.near(got, want, space, ffi.F32)
    # infinity behind the turned part, without a norm: its element alone
    x = np.ones((1, 3 * dim), np.float32)
    x[0, 50], x[0, dim + 20], x[0, 2 * dim + 49] = np.inf, np.nan, -np.inf
    for interleaved in (False, True):
        (q, _, _), (k, _, _) = run(dec, ffi.F32, ffi.F32, 1, 2, 1, dim, 40, interleaved, norm=False, x=x)
        assert np.isfinite(np.delete(q[0, 0], 50)).all() and q[0, 0, 50] == np.inf and np.isfinite(np.delete(k[0, 0], 49)).all() and k[0, 0, 49] == -np.inf
        assert (~np.isfinite(q[0, 1])).sum() == 2


def test_turning_back_gives_what_was_there(dec):
    """A rotation by a position and one by its negative: the element, to twice the room of one."""
    t, dim = 9, 64
    r = np.random.default_rng(5)
    x = r.standard_normal((t, 2 * dim)).astype(np.float32)
    freqs, _ = ops.rope_freqs(dim, 10000.0)
    pos = r.integers(0, 10**6, t).astype(np.int32)
    cc = dec.cc
    with w8.Buffers(cc) as b:
        dx, df = b.put(x), b.put(freqs)
        for p in (pos, -pos):
            dec.qk_norm_rope(dx, dx, dx + dim * 4, b.put(p), df, t, 1, 1, dim, dim, x_type=ffi.F32, y_type=ffi.F32, ldx=2 * dim, ldq=2 * dim, ldk=2 * dim)
        got = cc.d2h(dx, (t, 2, 2, dim // 2), np.float32)
    want = x.reshape(t, 2, 2, dim // 2)
    size = np.abs(want).sum(2, keepdims=True)
    assert (np.abs(got - want) <= 2 * np.sqrt(2) * size * (1.9e-7 + 7 * U)).all()


def test_more_rows_than_a_launch_has(dec):
    """Rows of two elements, 2^26 and more of them: four to a workgroup."""
    cc, t = dec.cc, 2**26 + 77
    x = np.random.default_rng(1).standard_normal((t, 2), dtype=np.float32).astype(np.float16)
    freqs = np.array([0.7])
    pos = (np.arange(t, dtype=np.int64) % 1000).astype(np.int32)
    with w8.Buffers(cc) as b:
        dx = b.put(x)
        dec.qk_norm_rope(dx, dx, 0, b.put(pos), b.put(freqs), t, 1, 0, 2, 2, x_type=ffi.F16, y_type=ffi.F16)
        got = cc.d2h(dx, (t, 2), np.float16)
    for at in (slice(0, 1000), slice(2**26 - 600, t)):
        v, a = x[at].astype(np.float64), pos[at] * 0.7
        want = np.stack([v[:, 0] * np.cos(a) - v[:, 1] * np.sin(a), v[:, 1] * np.cos(a) + v[:, 0] * np.sin(a)], 1)
        f8_ref.near(got[at].astype(np.float32), want, np.abs(v).sum(1, keepdims=True) * (1.9e-7 + 7 * U), ffi.F16)


def test_offsets_beyond_32_bits(dec):
    cc, ld, dim = dec.cc, 1_100_000_000, 64
    x = np.random.default_rng(2).standard_normal((3, 2 * dim)).astype(np.float32)
    freqs, _ = ops.rope_freqs(dim, 10000.0)
    pos = np.array([5, 6, 7], np.int32)
    with w8.Buffers(cc) as b:
        wide = cc.alloc(4 * (2 * ld + 2 * dim))
        try:
            for i in range(3):
                cc.h2d(wide + 4 * i * ld, x[i])
            dec.qk_norm_rope(wide, wide, wide + dim * 4, b.put(pos), b.put(freqs), 3, 1, 1, dim, dim, x_type=ffi.F32, y_type=ffi.F32, ldx=ld, ldq=ld, ldk=ld)
            for i in range(3):
                want, space = plain(x[i:i + 1], 1, 2, dim, None, 0, pos[i:i + 1], freqs, 1.0, False)
                f8_ref.near(cc.d2h(wide + 4 * i * ld, (1, 2, dim), np.float32), want, space, ffi.F32)
        finally:
            cc.free(wide)


def test_captured_call_replays_on_new_rows(dec):
    cc, t, dim = dec.cc, 6, 128
    r = np.random.default_rng(3)
    freqs, _ = ops.rope_freqs(dim, 10000.0)
    with w8.Buffers(cc) as b:
        dx, dp, q, k, df, w = b.filled(t * 3 * dim * 2), b.filled(t * 4), b.filled(t * 2 * dim * 2), b.filled(t * dim * 2), b.put(freqs), b.put(np.ones(dim, np.float32))

        def step():
            dec.qk_norm_rope(dx, q, k, dp, df, t, 2, 1, dim, dim, qw_dev=w, kw_dev=w)

        step()
        cc.capture_begin()
        step()
        graph = cc.capture_end()
        for i in range(3):
            cc.h2d(dx, r.standard_normal((t, 3 * dim)).astype(np.float16))
            cc.h2d(dp, r.integers(0, 9999, t).astype(np.int32))
            graph.launch()
            replay = cc.d2h(q, (t, 2 * dim), np.uint16), cc.d2h(k, (t, dim), np.uint16)
            cc.h2d(q, np.zeros((t, 2 * dim), np.uint16))
            step()
            assert np.array_equal(replay[0], cc.d2h(q, (t, 2 * dim), np.uint16)) and np.array_equal(replay[1], cc.d2h(k, (t, dim), np.uint16))
        graph.destroy()


def refused(code, words, call):
    with pytest.raises(ops.W4a16Error) as e:
        call()
    assert e.value.code == code and words in e.value.message, e.value.message


def test_refusals(dec):
    def f(x=256, q=256, k=256, pos=256, freqs=256, t=1, nq=1, nk=1, dim=8, rot=8, **more):
        return lambda: dec.qk_norm_rope(x, q, k, pos, freqs, t, nq, nk, dim, rot, **more)

    for words, code, call in (("null operand", ffi.ERR_ARG, f(x=0)), ("null operand", ffi.ERR_ARG, f(q=0)), ("null operand", ffi.ERR_ARG, f(k=0)),
                              ("x type 4", ffi.ERR_ARG, f(x_type=4)), ("result type 3", ffi.ERR_ARG, f(y_type=3)), ("t=0", ffi.ERR_SHAPE, f(t=0)),
                              ("not both 0", ffi.ERR_SHAPE, f(nq=0, nk=0)), ("head_dim=0", ffi.ERR_SHAPE, f(dim=0, rot=0)), ("head_dim=1025", ffi.ERR_SHAPE, f(dim=1025)),
                              ("rot_dim=3", ffi.ERR_SHAPE, f(rot=3)), ("rot_dim=10", ffi.ERR_SHAPE, f(rot=10)), ("positions", ffi.ERR_ARG, f(pos=0)),
                              ("positions", ffi.ERR_ARG, f(freqs=0)), ("neither", ffi.ERR_ARG, f(rot=0)), ("eps", ffi.ERR_ARG, f(qw_dev=256, eps=-1.0)),
                              ("eps", ffi.ERR_ARG, f(qw_dev=256, eps=float("nan"))), ("ldx=15", ffi.ERR_SHAPE, f(ldx=15)), ("ldq=7", ffi.ERR_SHAPE, f(ldq=7)),
                              ("ldk=7", ffi.ERR_SHAPE, f(ldk=7)), ("aligned", ffi.ERR_ARG, f(x=257)), ("aligned", ffi.ERR_ARG, f(q=258, y_type=ffi.F32)),
                              ("aligned", ffi.ERR_ARG, f(freqs=260)), ("aligned", ffi.ERR_ARG, f(kw_dev=258))):
        refused(code, words, call)
