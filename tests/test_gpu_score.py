"""Scoring of logits on the GPU against the formulas in 64 bits.

Room for the f32 results, in units of u = 2^-24: a term 2^(z L - r) carries the rounding of its exponent (|z - max| / ln 2 u, times ln 2),
of L (as much again, at most) and of the power itself (2 u); the sum of a thread's elements one rounding each, those of the joins less than 64.  So log S is
known to (elements per thread + 2 |z - max| + 70) u in the mean over the terms, weighted by p, where |z - max| p is below 1; an
exponent of its own adds 3 |z - max| u to a log probability, and the final product and difference 2 u of its size.  The entropy is a quotient of
two such sums: twice that, times 1 + U / S."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import w8a8_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0**-24


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


def call(dec, b, bits, t, v, kind, targets, top, ld=0, off=0):
    o = [b.filled(max(1, t * m) * 4) for m in (1, 1, max(top, 1), max(top, 1))]
    dec.token_logprobs(b.put(bits, off), t, v, logits_type=kind, ld=ld, targets_dev=b.put(np.asarray(targets, np.int32)), logp_dev=o[0], entropy_dev=o[1],
                       top_k=top, top_idx_dev=o[2] if top else 0, top_logp_dev=o[3] if top else 0)
    cc = dec.cc
    return cc.d2h(o[0], (t,), np.float32), cc.d2h(o[1], (t,), np.float32), cc.d2h(o[2], (t, max(top, 1)), np.int32)[:, :top], \
        cc.d2h(o[3], (t, max(top, 1)), np.float32)[:, :top]


def near(got, want, room):
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    assert (np.abs(got[fine].astype(np.float64) - want[fine]) <= np.broadcast_to(room, want.shape)[fine]).all(), np.abs(got[fine] - want[fine]).max()


def check(got, z, targets, top):
    logp, ent, idx, lp = ref.scores(z, targets, top)
    v = z.shape[1]
    base = (v / 256 + 64 + 70 + 2) * U
    with np.errstate(invalid="ignore"):
        near(got[0], logp, base + 6 * np.abs(np.nan_to_num(logp, posinf=0, neginf=0)) * U)
        near(got[1], ent, 2 * base * (1 + np.abs(ent)))
        near(got[3], lp, base + 6 * np.abs(np.nan_to_num(lp, posinf=0, neginf=0)) * U)
    assert np.array_equal(got[2], idx)


CASES = [(1, 1, 1), (1, 2, 2), (3, 31, 31), (1, 32, 32), (2, 100, 5), (1, 1023, 20), (5, 1024, 1), (2, 1025, 32), (1, 4096, 32), (1, 4097, 20), (7, 8191, 8),
         (1, 32000, 5), (64, 5000, 20), (1, 100003, 32), (2, 131072, 20), (300, 1500, 3), (1100, 300, 2), (1030, 4200, 32), (1, 262144, 0), (1, 1100000, 32)]


@pytest.mark.parametrize("kind", [ffi.F32, ffi.F16, ffi.BF16])
@pytest.mark.parametrize("t,v,top", CASES)
def test_scores(dec, t, v, top, kind):
    print("score", t, v, top, kind, flush=True)
    r = np.random.default_rng(v + t)
    bits, z = ref.narrow((r.standard_normal((t, v)) * 3).astype(np.float32), kind)
    targets = r.integers(-1, v, t)
    with ref.Buffers(dec.cc) as b:
        check(call(dec, b, bits, t, v, kind, targets, top), z, targets, top)


@pytest.mark.parametrize("kind", [ffi.F32, ffi.F16, ffi.BF16])
@pytest.mark.parametrize("v", [40, 3000, 20000])
def test_masks_ties_and_what_is_no_number(dec, v, kind):
    rows, r = [], np.random.default_rng(v)
    base = (r.standard_normal(v) * 2).astype(np.float32)

    def row(**at):
        z = base.copy()
        for a in at.get("sets", ()):
            z[a[0]] = a[1]
        rows.append(z)

    row()
    row(sets=[(slice(None), -np.inf)])                      # a mask that leaves nothing
    row(sets=[(slice(None), -np.inf), (v - 1, 1.5)])        # one token
    row(sets=[(slice(0, v - 7), -np.inf)])                  # fewer tokens than alternatives
    row(sets=[(slice(v // 2, None), -np.inf)])
    row(sets=[(slice(None), 0.0)])                          # all alike
    row(sets=[(slice(None), np.float32(-3.4e38) if kind != ffi.F16 else -65504.0)])  # the type's lowest value everywhere
    row(sets=[(slice(0, v // 2), np.float32(-3.3e38) if kind != ffi.F16 else -65504.0)])
    row(sets=[(slice(None, None, 2), 0.0), (slice(1, None, 2), -0.0)])               # -0 is 0
    row(sets=[(slice(None, None, 3), 4.0)])                 # a third alike, on top
    row(sets=[(v // 3, np.nan)])
    row(sets=[(0, np.nan), (v - 1, np.nan), (5, np.inf)])
    row(sets=[(v - 2, np.inf)])
    row(sets=[(slice(None), np.inf)])
    row(sets=[(slice(None), np.nan)])
    row(sets=[(3, 200.0)])                                  # one token has it all
    rows.append(np.sort(base))                              # every element is better than all before
    rows.append(np.sort(base)[::-1].copy())
    rows.append(np.full(v, -np.inf, np.float32))
    rows.append((base * 1000).astype(np.float32))
    with np.errstate(over="ignore"):
        bits, z = ref.narrow(np.stack(rows), ffi.F32)
        if kind != ffi.F32:
            z = np.stack(rows)
            nan = np.isnan(z)
            if kind == ffi.F16:
                bits = np.clip(z, -65504, 65504).astype(np.float16)
                bits[np.isinf(z)] = z[np.isinf(z)].astype(np.float16)
                z = bits.astype(np.float32)
            else:
                bits = ref.to_bf16(np.where(nan, 0, z))
                bits[nan] = 0x7FC0
                z = ref.from_bf16(bits)
    t = len(rows)
    targets = np.array([(i * 7919) % v for i in range(t)])
    targets[2], targets[3], targets[0] = v - 1, 0, -5
    for top in (1, 8, 32):
        with ref.Buffers(dec.cc) as b:
            got = call(dec, b, bits, t, v, kind, targets, top)
            check(got, z, targets, top)
        # the rows by themselves: other launches, the same bits
        for i in (0, 3, 10, t - 4):
            with ref.Buffers(dec.cc) as b:
                one = call(dec, b, bits[i:i + 1], 1, v, kind, targets[i:i + 1], top)
            check(one, z[i:i + 1], targets[i:i + 1], top)


@pytest.mark.parametrize("kind", [ffi.F32, ffi.BF16])
@pytest.mark.parametrize("v", [40, 5000, 20000])
def test_finite_masks_and_logits_of_any_size(dec, v, kind):
    """Masks far below the logits that are not the type's lowest value, and logits where a step of the type passes one: every magnitude up to 3e38.
    The differences of such logits are rounded once more, |z - max| p u in the mean over the terms, less than one; the joins, of which there are at most
    20 levels, leave room for it."""
    r = np.random.default_rng(v + 1)
    base = (r.standard_normal(v) * 2).astype(np.float32)
    few = r.permutation(v)[:20]
    rows = []
    for mask in (-2e6, -1e8, -1e9, -2e9, -1e10, -1e12, -1e20, -1e30, -5e37, -2e38):
        z = np.full(v, mask, np.float32)
        rows.append(z.copy())            # nothing is left
        z[few] = base[few]
        rows.append(z.copy())            # twenty tokens are
        z = base.copy()
        z[:v // 2] = mask
        rows.append(z)                   # whole stretches are masked
    for top in (1e6, 3e7, 1e9, 1.45e9, 5e9, 1e12, 1e30, 3e38):
        z = base.copy()
        z[v // 3] = top
        rows.append(z)                   # one token has it all
        rows.append(np.where(np.arange(v) % 3 == 0, np.float32(top), base))
        for sign in (1, -1):             # steps of the type apart, around the size
            rows.append(np.float32(sign * top) + np.float32(np.spacing(np.float32(top))) * np.rint(base))
    for size in (2.0**19, 2.0**20, 2.0**21, 2.0**23, 2.0**30):
        for sign in (1, -1):             # on both sides of a power of two, in one row
            rows.append((np.float64(sign * size) + base).astype(np.float32))
    rows.append((base * 1e36).astype(np.float32))
    bits, z = ref.narrow(np.stack(rows).astype(np.float32), kind)
    assert np.isfinite(z).all()
    t = len(rows)
    targets = np.where(np.arange(t) % 2 == 0, few[0], (np.arange(t) * 7919) % v)
    for top in (0, 20):
        with ref.Buffers(dec.cc) as b:
            got = call(dec, b, bits, t, v, kind, targets, top)
            check(got, z, targets, top)
    for i in (0, 1, 2, 13, 14, 31, 40, t - 1):  # alone: segments and their records
        with ref.Buffers(dec.cc) as b:
            check(call(dec, b, bits[i:i + 1], 1, v, kind, targets[i:i + 1], 20), z[i:i + 1], targets[i:i + 1], 20)

@pytest.mark.parametrize("kind,off,ld", [(ffi.F16, 2, 5003), (ffi.BF16, 6, 5010), (ffi.F32, 4, 5001), (ffi.F16, 14, 6000)])
def test_any_alignment_and_stride(dec, kind, off, ld):
    t, v, top = 9, 5000, 20
    bits, z = ref.narrow((np.random.default_rng(ld).standard_normal((t, ld)) * 3).astype(np.float32), kind)
    bits[:, v:] = 0x7C00 if kind == ffi.F16 else 0x7F80 if kind == ffi.BF16 else np.inf  # never read as logits
    if kind == ffi.F16:
        bits = bits.astype(np.float16)
        bits[:, v:] = np.inf
    targets = np.arange(t) * 500
    with ref.Buffers(dec.cc) as b:
        got = call(dec, b, bits.reshape(-1)[:(t - 1) * ld + v], t, v, kind, targets, top, ld, off)
    check(got, z[:, :v], targets, top)


def test_targets_outside_and_results_left_out(dec):
    t, v = 4, 6000
    z = np.random.default_rng(1).standard_normal((t, v)).astype(np.float32)
    targets = np.array([-1, v, -2**31, 2**31 - 1])
    with ref.Buffers(dec.cc) as b:
        got = call(dec, b, z, t, v, ffi.F32, targets, 3)
        assert got[0][0] == 0 and np.isnan(got[0][1]) and got[0][2] == 0 and np.isnan(got[0][3])
        dz, e, i = b.put(z), b.filled(t * 4), b.filled(t * 12)
        dec.token_logprobs(dz, t, v, entropy_dev=e)
        assert np.array_equal(dec.cc.d2h(e, (t,), np.uint32), got[1].view(np.uint32))
        dec.token_logprobs(dz, t, v, top_k=3, top_idx_dev=i)
        assert np.array_equal(dec.cc.d2h(i, (t, 3), np.int32), got[2])


def test_one_row_or_many_give_the_same_alternatives_and_a_second_call_the_same_bits(dec):
    t, v, top = 40, 70001, 20
    bits, z = ref.narrow((np.random.default_rng(2).standard_normal((t, v)) * 2).astype(np.float32), ffi.BF16)
    targets = np.arange(t)
    with ref.Buffers(dec.cc) as b:
        first, again = (call(dec, b, bits, t, v, ffi.BF16, targets, top) for _ in range(2))
    for x, y in zip(first, again):
        assert x.tobytes() == y.tobytes()
    check(first, z, targets, top)


def test_rows_beyond_32_bits(dec):
    v, ld, cc = 5000, 2_200_000_001, dec.cc
    bits, z = ref.narrow(np.random.default_rng(2).standard_normal((2, v)).astype(np.float32) * 3, ffi.F16)
    wide = cc.alloc(2 * (ld + v))
    try:
        with ref.Buffers(cc) as b:
            for i in range(2):
                cc.h2d(wide + 2 * i * ld, bits[i])
            o = [b.filled(n * 4) for n in (2, 2, 64, 64)]
            dec.token_logprobs(wide, 2, v, logits_type=ffi.F16, ld=ld, targets_dev=b.put(np.array([7, 4999], np.int32)), logp_dev=o[0], entropy_dev=o[1],
                               top_k=32, top_idx_dev=o[2], top_logp_dev=o[3])
            got = [cc.d2h(p, s, d) for p, s, d in zip(o, ((2,), (2,), (2, 32), (2, 32)), (np.float32, np.float32, np.int32, np.float32))]
    finally:
        cc.free(wide)
    check(got, z, [7, 4999], 32)


def test_capture_and_replay(dec):
    """A head and its scoring in one graph: tickets are back at zero after every replay, new logits give new results."""
    cc, v, k, t, top = dec.cc, 9000, 256, 3, 10
    w, sb, _ = ref.weights(4, v, k)
    dec.upload_lin_w8a8("head", w, sb, v, k)
    x = np.random.default_rng(8).standard_normal((t, k)).astype(np.float32)
    with ref.Buffers(cc) as b:
        dx, z, tg = b.put(x), b.filled(t * v * 4), b.put(np.array([1, -1, 8999], np.int32))
        o = [b.filled(t * m * 4) for m in (1, 1, top, top)]

        def step():
            dec.lin_forward_w8a8("head", dx, z, t, x_type=ffi.F32, y_type=ffi.F32)
            dec.token_logprobs(z, t, v, targets_dev=tg, logp_dev=o[0], entropy_dev=o[1], top_k=top, top_idx_dev=o[2], top_logp_dev=o[3])

        def read():
            return [cc.d2h(p, (t, m), np.uint32) for p, m in zip(o, (1, 1, top, top))]

        step()
        first = read()
        logits = cc.d2h(z, (t, v), np.float32)
        check([a.view(np.float32) if i != 2 else a.view(np.int32) for i, a in enumerate([first[0][:, 0], first[1][:, 0], first[2], first[3]])], logits,
              np.array([1, -1, 8999]), top)
        cc.capture_begin()
        step()
        graph = cc.capture_end()
        for i in range(4):
            cc.h2d(dx, x * np.float32(1 + i))
            graph.launch()
            replay = read()
            step()
            assert all(np.array_equal(p, q) for p, q in zip(replay, read()))
            cc.sync()
        graph.destroy()


def test_refusals(dec):
    def refused(code, words, **kw):
        a = dict(t=2, n_vocab=100, entropy_dev=256)
        a.update(kw)
        with pytest.raises(ops.W4a16Error) as e:
            dec.token_logprobs(a.pop("logits_dev", 256), **a)
        assert e.value.code == code and words in e.value.message, e.value.message

    refused(ffi.ERR_ARG, "null operand", logits_dev=0)
    refused(ffi.ERR_ARG, "type 3", logits_type=ffi.Q8)
    refused(ffi.ERR_SHAPE, "t=0", t=0)
    refused(ffi.ERR_SHAPE, "n_vocab=0", n_vocab=0)
    refused(ffi.ERR_SHAPE, "ld=99", ld=99)
    refused(ffi.ERR_SHAPE, "top_k=33", top_k=33, top_idx_dev=256)
    refused(ffi.ERR_SHAPE, "top_k=20", n_vocab=19, top_k=20, top_idx_dev=256)
    refused(ffi.ERR_ARG, "come together", targets_dev=256)
    refused(ffi.ERR_ARG, "come together", logp_dev=256)
    refused(ffi.ERR_ARG, "come together", top_k=3)
    refused(ffi.ERR_ARG, "come together", top_idx_dev=256)
    refused(ffi.ERR_ARG, "no result", entropy_dev=0)
    refused(ffi.ERR_ARG, "aligned", logits_dev=258)
    refused(ffi.ERR_ARG, "aligned", entropy_dev=258)
