"""Verification of drafted tokens on the GPU against the definition in 64 bits.  Both sides hold what draws to 10^-11 and better, so that of the some 10^5 draws here the
chance that one lies between their borders is V * 10^-11 each, 10^-1 in 10^3 runs of all; decisions to 10^-6, of some 10^4 here.  Their inputs are fixed, as are the results of both sides:
tokens and counts are equal."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import verify_ref as ref
from tests import w8a8_ref as w8

pytestmark = pytest.mark.gpu
TYPES = [ffi.F32, ffi.F16, ffi.BF16]


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


def rows_of(drafts):
    return np.concatenate([[0], np.cumsum(drafts)]).astype(np.int32)


def call(dec, b, bits, draft, row0, drafted, u, temps, kind, v, ld=0, ldd=0, off=0, alias=False):
    """(tokens [t], accepted) and 8 words behind each"""
    cc, t, n = dec.cc, len(drafted), len(row0) - 1
    dd = b.put(np.asarray(drafted, np.int32), off * 2)
    tokens, accepted = dd if alias else b.filled(t * 4 + 32, offset=off * 2), b.filled(n * 4 + 32)
    dec.verify_drafts(b.put(bits, off), dd, b.put(row0), b.put(np.asarray(u, np.float32)), tokens, accepted, t, n, v, logits_type=kind, ld=ld,
                      draft_dev=b.put(draft, off) if draft is not None else 0, ld_draft=ldd, temps_dev=b.put(np.asarray(temps, np.float32)) if temps is not None else 0)
    got, acc = cc.d2h(tokens, (t + 8,), np.int32), cc.d2h(accepted, (n + 8,), np.int32)
    assert (acc[n:].view(np.uint8) == 0xA5).all() and (alias or (got[t:].view(np.uint8) == 0xA5).all())
    return got[:t], acc[:n]


def check(dec, bits, z, dbits, d, row0, drafted, u, temps, kind, **more):
    t, v = z.shape
    n = len(row0) - 1
    with w8.Buffers(dec.cc) as b:
        got = call(dec, b, bits, dbits, row0, drafted, u, temps, kind, v, **more)
    before = np.asarray(drafted, np.int32) if more.get("alias") else np.full(t, -1515870811, np.int32)  # 0xA5A5A5A5
    want = ref.verified(z, d, row0, drafted, u, np.ones(n) if temps is None else temps, before)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0]), (got, want)
    return got


def problem(seed, drafts, v, kind, spread=2.5, apart=0.7, greedy=0.0):
    """(bits, z, draft bits, d, row0, drafted, u, temps): drafted tokens are drawn from the draft's distribution"""
    r = np.random.default_rng(seed)
    row0 = rows_of(drafts)
    t, n = int(row0[-1]), len(drafts)
    z = r.standard_normal((t, v)) * spread
    z[np.arange(t), r.integers(0, v, t)] += 4
    d = z + r.standard_normal((t, v)) * apart
    temps = r.uniform(0.5, 1.5, n).astype(np.float32)
    temps[r.random(n) < greedy] = 0
    bits, z = w8.narrow(z.astype(np.float32), kind)
    dbits, d = w8.narrow(d.astype(np.float32), kind)
    seq = np.repeat(np.arange(n), drafts)
    per = np.where(temps == 0, 0.1, temps)[seq][:, None]
    drafted = (d / per - np.log(-np.log(r.uniform(1e-12, 1, (t, v))))).argmax(1).astype(np.int32)
    return bits, z, dbits, d, row0, drafted, r.random(t, dtype=np.float32), temps


SHAPES = [([1], 1), ([1], 7), ([2], 2), ([3, 1, 4], 31), ([5], 100), ([2] * 20, 1000), ([1] * 64, 333), ([0, 3, 0, 0, 2, 1, 0], 5000), ([4, 9, 1], 4096), ([3, 3], 4097),
          ([5, 1], 8192), ([2, 2], 8193), ([5], 32000), ([5, 2, 1], 50021), ([3] * 300, 200), ([70, 1, 130], 64), ([2] * 70, 40000), ([1], 262144)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("drafts,v", SHAPES)
def test_tokens_and_counts(dec, drafts, v, kind):
    print("verify", drafts[:8], len(drafts), v, kind, flush=True)
    bits, z, dbits, d, row0, drafted, u, temps = problem(len(drafts) * 7 + v, drafts, v, kind, greedy=0.2)
    check(dec, bits, z, dbits, d, row0, drafted, u, temps, kind)        # drafts with their logits
    check(dec, bits, z, None, None, row0, drafted, u, temps, kind)      # certain ones
    check(dec, bits, z, dbits, d, row0, drafted, u, None, kind)         # temperature 1
    check(dec, bits, z, dbits, d, row0, drafted, u, np.zeros(len(drafts), np.float32), kind, alias=True)
    check(dec, bits, z, dbits, d, row0, drafted, u, temps, kind, alias=True)


@pytest.mark.parametrize("certain", [False, True])
def test_many_segments_of_a_vocabulary(dec, certain):
    """More segments than a workgroup looks at in one go (256), and draws from all of them."""
    v, drafts = 1_300_000, [1, 2, 2, 1]
    for spread in (0.0, 1.0):
        bits, z, dbits, d, row0, drafted, u, temps = problem(5, drafts, v, ffi.F32, spread=spread, apart=0.05 + spread)
        u[[0, 2, 4, 5]] = [0.9995, 0.5, 0.02, 0.99999]
        got = check(dec, bits, z, None if certain else dbits, None if certain else d, row0, drafted, u, temps, ffi.F32)
        assert spread or (got[0][0] > 1_290_000 and got[0][5] > 1_290_000)


def test_drafts_equal_to_the_target_are_all_accepted(dec):
    """p = q: every u below one accepts, also the largest there is, and the token that follows is the target's."""
    for kind in TYPES:
        bits, z, _, _, row0, drafted, u, temps = problem(3, [6] * 30, 3000, kind)
        u[:] = np.float32(1 - 2.0**-24)
        got = check(dec, bits, z, bits, z, row0, drafted, u, temps, kind)
        assert (got[1] == 5).all()


def test_the_numbers_at_the_ends(dec):
    """u = 0 accepts what is possible at all and draws the first possible token; the largest u draws one of the last."""
    v, kind = 1000, ffi.F32
    bits, z, dbits, d, row0, drafted, u, temps = problem(4, [1, 3, 2, 4], v, kind)
    z[:, :5] = -np.inf
    z[:, -7:] = -np.inf
    for top in (0.0, np.float32(1 - 2.0**-24)):
        u[:] = top
        for drafts in ((dbits, d), (None, None)):
            got = check(dec, z, z, *drafts, row0, drafted, u, temps, kind)
        if top == 0.0:
            assert got[0][0] == 5


def test_masks_rows_of_nothing_and_of_no_number(dec):
    r = np.random.default_rng(9)
    for kind in TYPES:
        for v in (40, 9000):
            low = -65504.0 if kind == ffi.F16 else -3.3e38
            sets = [lambda z: None, lambda z: z.fill(-np.inf), lambda z: z.__setitem__(3, np.nan), lambda z: z.__setitem__(v - 1, np.inf), lambda z: z.fill(low),
                    lambda z: z.__setitem__(slice(0, v - 2), -np.inf), lambda z: z.__setitem__(slice(1, None), low), lambda z: z.fill(0.0), lambda z: z.__imul__(0.0),
                    lambda z: z.__setitem__(slice(None), np.nan), lambda z: z.__setitem__(slice(None), np.inf), lambda z: z.__setitem__(slice(None, None, 2), -np.inf)]
            pairs = [(i, j) for i in range(len(sets)) for j in range(len(sets))]
            drafts = [2] * len(pairs)
            bits, z, dbits, d, row0, drafted, u, temps = problem(v, drafts, v, kind, greedy=0.3)
            z, d = z.copy(), d.copy()
            for n, (i, j) in enumerate(pairs):  # the target's row that judges, and the draft's; the row behind as the target's
                sets[i](z[2 * n]), sets[j](d[2 * n]), sets[j](z[2 * n + 1])
            drafted[::14] = -1
            drafted[2::22] = v
            drafted[4::26] = 2**31 - 1
            bits, z = narrowed(z, kind)
            dbits, d = narrowed(d, kind)
            check(dec, bits, z, dbits, d, row0, drafted, u, temps, kind)
            check(dec, bits, z, None, None, row0, drafted, u, temps, kind)
            check(dec, bits, z, dbits, d, row0, drafted, u, np.where(temps > 0, r.choice([1e-30, 1e-3, 1e4, 1e30], len(temps)), [np.nan, -1.0][v % 2]), kind)


def narrowed(z, kind):
    """Infinities and NaN kept."""
    if kind == ffi.F32:
        return z.astype(np.float32), z.astype(np.float32)
    if kind == ffi.F16:
        h = np.where(np.isinf(z), z, np.clip(z, -65504, 65504)).astype(np.float16)
        return h, h.astype(np.float32)
    b = w8.to_bf16(np.where(np.isfinite(z), z, 0).astype(np.float32))
    b[np.isnan(z)], b[z == np.inf], b[z == -np.inf] = 0x7fc0, 0x7f80, 0xff80
    return b, w8.from_bf16(b)


def test_ties_go_to_the_lowest_token(dec):
    for kind in TYPES:
        v, n = 20000, 12
        z = np.zeros((2 * n, v), np.float32)
        for i in range(n):
            z[2 * i, [19999, 700 * i + 3, 12345]] = 5
            z[2 * i + 1, 1::2] = -0.0
        bits, z = w8.narrow(z, kind)
        drafted = np.repeat(np.arange(n) * 700 + 3, 2).astype(np.int32)
        drafted[::6] = 19999
        got = check(dec, bits, z, None, None, rows_of([2] * n), drafted, np.full(2 * n, 0.5), np.zeros(n, np.float32), kind)
        assert (got[0][1::2][got[1] == 1] == 0).all() and got[1].sum() == n - 4


def test_what_comes_out_is_distributed_as_the_target_says(dec):
    """The first token of 200000 sequences, whatever the draft: counts within five standard deviations of the target's probabilities."""
    v, n = 11, 200_000
    r = np.random.default_rng(12)
    z, d = r.standard_normal(v) * 1.5, r.standard_normal(v) * 1.5
    p, q = (np.exp(a) / np.exp(a).sum() for a in (z, d))
    rows = np.repeat(z[None].astype(np.float32), 2 * n, 0)
    draws = np.repeat(d[None].astype(np.float32), 2 * n, 0)
    drafted = r.choice(v, 2 * n, p=q).astype(np.int32)
    for certain in (False, True):
        with w8.Buffers(dec.cc) as b:
            tokens, accepted = call(dec, b, rows, None if certain else draws, rows_of([2] * n), drafted, r.random(2 * n, dtype=np.float32), None, ffi.F32, v)
        count = np.bincount(tokens[::2], minlength=v)
        assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()
        rate = (np.minimum(p, q).sum() if not certain else (p * q).sum())
        assert abs(accepted.mean() - rate) <= 5 * np.sqrt(rate * (1 - rate) / n)
        second = np.bincount(tokens[1::2][accepted == 1], minlength=v)
        assert (np.abs(second - second.sum() * p) <= 5 * np.sqrt(second.sum() * p * (1 - p)) + 1).all()


@pytest.mark.parametrize("kind,v,ld,ldd,off", [(ffi.F16, 777, 801, 779, 2), (ffi.BF16, 5003, 5003, 6001, 6), (ffi.F32, 4097, 4099, 0, 4)])
def test_strides_and_alignment(dec, kind, v, ld, ldd, off):
    drafts = [3, 1, 2, 5]
    bits, z, dbits, d, row0, drafted, u, temps = problem(v, drafts, v, kind)
    t = len(drafted)
    wide = [np.full((t, w), 0x7fff if a.dtype == np.uint16 else np.nan, a.dtype) for a, w in ((bits, ld), (dbits, ldd or v))]
    wide[0][:, :v], wide[1][:, :v] = bits, dbits
    flat = [w.reshape(-1)[:(t - 1) * w.shape[1] + v] for w in wide]
    with w8.Buffers(dec.cc) as b:
        got = call(dec, b, flat[0], flat[1], row0, drafted, u, temps, kind, v, ld=ld, ldd=ldd, off=off)
    want = ref.verified(z, d, row0, drafted, u, temps, np.full(t, -1, np.int32))
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("kind", TYPES)
def test_temperatures_of_any_size(dec, kind):
    """Above all logits' sizes every token that is not ruled out is as likely; far below them the largest is certain."""
    bits, z, dbits, d, row0, drafted, u, _ = problem(9, [3] * 12, 700, kind)
    for rows in (z, d):
        rows[:, 100:400] = -np.inf
    (bits, z), (dbits, d) = w8.narrow(z, kind), w8.narrow(d, kind)
    drafted = np.where((drafted >= 100) & (drafted < 400), 5, drafted)
    for temp in (np.inf, 3e38, 1e30, 1e-6, 1e-30, 1e-38):
        temps = np.full(12, temp, np.float32)
        check(dec, bits, z, dbits, d, row0, drafted, u, temps, kind)
        check(dec, bits, z, None, None, row0, drafted, u, temps, kind)


def test_rows_of_no_sequence_stay_as_they_are(dec):
    bits, z, dbits, d, row0, drafted, u, temps = problem(1, [3, 2, 4, 3], 500, ffi.F32)
    row0 = np.array([3, 5, 9], np.int32)  # of 12 rows
    got = check(dec, bits, z, dbits, d, row0, drafted, u, temps[:2], ffi.F32)
    assert (got[0][:3] == -1515870811).all() and (got[0][9:] == -1515870811).all()


def test_starts_that_are_none_write_nothing_outside(dec):
    """Not ascending, below zero, beyond the rows: results mean nothing, but lie within the buffers; the context's next call is right."""
    bits, z, dbits, d, row0, drafted, u, temps = problem(2, [3, 3, 3, 3], 300, ffi.F32)
    for bad in ([-5, 3, 2**31 - 1, 6, 12], [12, 9, 6, 3, 0], [-2**31, -1, -1, 40, 50], [4, 4, 2, 100, 12]):
        with w8.Buffers(dec.cc) as b:
            call(dec, b, bits, dbits, np.array(bad, np.int32), drafted, u, temps, ffi.F32, 300)
        check(dec, bits, z, dbits, d, row0, drafted, u, temps, ffi.F32)


def test_more_rows_than_a_launch_has(dec):
    """Sequences of one row, two tokens: the second is drawn where u is p of the first or more."""
    cc, t, v = dec.cc, 2**24 + 77, 2  # workgroups of 256 threads
    r = np.random.default_rng(3)
    z = (r.standard_normal((t, v), dtype=np.float32) * 3).astype(np.float16)
    u = r.random(t, dtype=np.float32)
    with w8.Buffers(cc) as b:
        got = call(dec, b, z, None, np.arange(t + 1, dtype=np.int32), np.zeros(t, np.int32), u, None, ffi.F16, v)
    d = z[:, 1].astype(np.float64) - z[:, 0]
    p = 1 / (1 + np.exp(d))
    near = np.abs(u - p) < 1e-10
    assert near.sum() < 5 and not got[1].any() and np.array_equal(got[0][~near], (u >= p).astype(np.int32)[~near])


def test_offsets_beyond_32_bits(dec):
    """Rows 2.2e9 elements apart."""
    cc, v, ld = dec.cc, 1000, 2_200_000_000
    bits, z, dbits, d, row0, drafted, u, temps = problem(8, [2, 1], v, ffi.F16)
    with w8.Buffers(cc) as b:
        wide = cc.alloc(2 * (2 * ld + v))
        try:
            for i in range(3):
                cc.h2d(wide + 2 * i * ld, bits[i])
            tokens, accepted = b.filled(12), b.filled(8)
            dec.verify_drafts(wide, b.put(drafted), b.put(row0), b.put(u), tokens, accepted, 3, 2, v, logits_type=ffi.F16, ld=ld, draft_dev=b.put(dbits), temps_dev=b.put(temps))
            want = ref.verified(z, d, row0, drafted, u, temps, np.zeros(3, np.int32))
            assert np.array_equal(cc.d2h(tokens, (3,), np.int32), want[0]) and np.array_equal(cc.d2h(accepted, (2,), np.int32), want[1])
        finally:
            cc.free(wide)


def test_captured_calls_replay_on_new_numbers(dec):
    """Graphs of two sizes that share the scratch, and eager calls between them."""
    cc = dec.cc
    big, small = problem(1, [4, 2, 5], 20000, ffi.BF16), problem(2, [3] * 40, 700, ffi.BF16)
    r = np.random.default_rng(0)
    with w8.Buffers(cc) as b:
        sides = []
        for bits, z, dbits, d, row0, drafted, u, temps in (big, small):
            t, n, v = len(drafted), len(row0) - 1, z.shape[1]
            held = [b.put(a) for a in (bits, drafted, row0, u, dbits, temps)] + [b.filled(t * 4), b.filled(n * 4)]

            def step(h=held, t=t, n=n, v=v):
                dec.verify_drafts(h[0], h[1], h[2], h[3], h[6], h[7], t, n, v, logits_type=ffi.BF16, draft_dev=h[4], temps_dev=h[5])

            step()
            sides.append((held, step, (z, d, row0, drafted, temps), t, n))
        graphs = []
        for held, step, _, _, _ in sides:
            cc.capture_begin()
            step()
            graphs.append(cc.capture_end())
        for turn in range(4):
            for (held, step, (z, d, row0, drafted, temps), t, n), graph in zip(sides, graphs):
                u = r.random(t, dtype=np.float32)
                cc.h2d(held[3], u)
                want = ref.verified(z, d, row0, drafted, u, temps, np.zeros(t, np.int32))
                for run in (graph.launch, step):
                    cc.h2d(held[6], np.zeros(t, np.int32))
                    run()
                    assert np.array_equal(cc.d2h(held[6], (t,), np.int32), want[0]) and np.array_equal(cc.d2h(held[7], (n,), np.int32), want[1])
        for graph in graphs:
            graph.destroy()


def refused(code, words, call_):
    with pytest.raises(ops.W4a16Error) as e:
        call_()
    assert e.value.code == code and words in e.value.message, e.value.message


def test_refusals(dec):
    def f(*ptrs, t=1, n=1, v=8, **more):
        args = list(ptrs) + [256] * (6 - len(ptrs))
        return lambda: dec.verify_drafts(*args, t, n, v, **more)

    for i in range(6):
        refused(ffi.ERR_ARG, "null operand", f(*([256] * i + [0])))
    refused(ffi.ERR_ARG, "logits type 3", f(logits_type=3))
    refused(ffi.ERR_SHAPE, "t=0", f(t=0))
    refused(ffi.ERR_SHAPE, "seqs=0", f(n=0))
    refused(ffi.ERR_SHAPE, "n_vocab=0", f(v=0))
    refused(ffi.ERR_SHAPE, "n_vocab=1073741824", f(v=2**30))
    refused(ffi.ERR_SHAPE, "ld=7", f(ld=7))
    refused(ffi.ERR_SHAPE, "ld_draft=7", f(ld_draft=7))
    refused(ffi.ERR_ARG, "aligned", f(257, logits_type=ffi.F16))
    refused(ffi.ERR_ARG, "aligned", f(draft_dev=258))
    refused(ffi.ERR_ARG, "aligned", f(256, 258))
    refused(ffi.ERR_ARG, "aligned", f(temps_dev=257))
    fresh = ops.W4a16Dec()
    try:
        fresh.cc.capture_begin()
        refused(ffi.ERR_ARG, "capture", lambda: fresh.verify_drafts(256, 256, 256, 256, 256, 256, 1, 1, 8))
        with pytest.raises(ops.W4a16Error):
            fresh.cc.capture_end()  # nothing was launched
    finally:
        fresh.cc.close()
