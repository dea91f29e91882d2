"""A verifying step over drafted tokens, its operators one after the other as they are used: a norm that quantises, the FP8 linears (attention itself is left out: the output projection
reads the turned queries), the norm and rotation of queries and keys, the gated FFN, the head, the verification.  Each operator against its plain form on what the device gave the one before
it, with that operator's own room; then the whole step captured and replayed."""
import numpy as np
import pytest

from llm170_amd import ffi, ops
from tests import f8_ref as ref
from tests import verify_ref
from tests import w8a8_ref as w8
from tests.test_gpu_rope import plain as rotated

pytestmark = pytest.mark.gpu
HIDDEN, NQ, NK, DIM, FF, VOCAB = 384, 4, 2, 64, 256, 1003
QKV, K = (NQ + 2 * NK) * DIM, NQ * DIM


@pytest.fixture(scope="module")
def dec():
    d = ops.W4a16Dec()
    yield d
    d.cc.close()


class Step:
    def __init__(self, dec, b, lens):
        self.dec, self.cc, r = dec, dec.cc, np.random.default_rng(7)
        self.row0 = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.t, self.seqs = int(self.row0[-1]), len(lens)
        self.w = {}
        for i, (name, n, k) in enumerate((("qkv", QKV, HIDDEN), ("o", HIDDEN, K), ("gu", 2 * FF, HIDDEN), ("down", HIDDEN, FF), ("head", VOCAB, HIDDEN))):
            w, sb, sv = ref.weights(i, n, k)
            dec.upload_lin_f8("step." + name, w, sb * np.float32(0.1), n, k)
            self.w[name] = (w, sv * np.float32(0.1), n, k)
        t = self.t
        self.nw = (1 + 0.2 * r.standard_normal((3, HIDDEN))).astype(np.float32)
        self.qw, self.kw = ((1 + 0.3 * r.standard_normal(DIM)).astype(np.float32) for _ in range(2))
        self.pos = np.concatenate([900 * i + np.arange(n) for i, n in enumerate(lens)]).astype(np.int32)
        self.freqs, self.amp = ops.rope_freqs(DIM, 10000.0, ffi.ROPE_PLAIN, 1.0, 4096.0, 1.0, 32.0)
        self.drafted = r.integers(0, VOCAB, t).astype(np.int32)
        self.u = r.random(t, dtype=np.float32)
        self.dbits = (r.standard_normal((t, VOCAB)) * 2).astype(np.float16)
        self.temps = np.where(np.arange(self.seqs) % 3 == 2, 0, 0.8).astype(np.float32)
        put = b.put
        self.p = {name: put(v) for name, v in (("nw", self.nw), ("qw", self.qw), ("kw", self.kw), ("pos", self.pos), ("freqs", self.freqs), ("row0", self.row0), ("drafted", self.drafted),
                                               ("u", self.u), ("draft", self.dbits), ("temps", self.temps))}
        for name, size in (("x", HIDDEN * 4), ("ab", HIDDEN * 4), ("ab2", HIDDEN * 4), ("ab3", HIDDEN * 4), ("y", QKV * 2), ("ff", FF * 2), ("logits", VOCAB * 2), ("tokens", 4), ("norm", HIDDEN * 4)):
            self.p[name] = b.filled(t * size)
        self.p["accepted"] = b.filled(self.seqs * 4)
        self.p["q"], self.p["s"] = b.filled(ops.q8_bytes(t, HIDDEN)), b.filled(t * 4 * 3)

    def stages(self):
        d, p, t = self.dec, self.p, self.t
        norm = lambda i, ab: lambda: d.norm_resid_f8(p["x"], p["nw"], p[ab], p["q"], p["s"], t, HIDDEN, w_off=i * HIDDEN)  # noqa: E731
        return [("norm", norm(0, "ab")),
                ("qkv", lambda: d.lin_forward_f8("step.qkv", p["q"], p["y"], t, x_type=ffi.F8, xs_dev=p["s"], y_type=ffi.F16)),
                ("rope", lambda: d.qk_norm_rope(p["y"], p["y"], p["y"] + K * 2, p["pos"], p["freqs"], t, NQ, NK, DIM, DIM, ldx=QKV, ldq=QKV, ldk=QKV, qw_dev=p["qw"], kw_dev=p["kw"], amp=self.amp)),
                ("o", lambda: d.lin_forward_f8("step.o", p["y"], p["ab2"], t, x_type=ffi.F16, ldx=QKV, y_type=ffi.F32)),
                ("norm", norm(1, "ab2")),
                ("gu", lambda: d.lin_forward_f8_glu("step.gu", p["q"], p["ff"], t, x_type=ffi.F8, xs_dev=p["s"], y_type=ffi.F16)),
                ("down", lambda: d.lin_forward_f8("step.down", p["ff"], p["ab3"], t, x_type=ffi.F16, y_type=ffi.F32)),
                ("norm", norm(2, "ab3")),
                ("head", lambda: d.lin_forward_f8("step.head", p["q"], p["logits"], t, x_type=ffi.F8, xs_dev=p["s"], y_type=ffi.F16)),
                ("verify", lambda: d.verify_drafts(p["logits"], p["drafted"], p["row0"], p["u"], p["tokens"], p["accepted"], t, self.seqs, VOCAB, logits_type=ffi.F16, draft_dev=p["draft"],
                                                   temps_dev=p["temps"]))]

    def start(self, seed):
        r = np.random.default_rng(seed)
        for name in ("x", "ab"):
            self.cc.h2d(self.p[name], r.standard_normal((self.t, HIDDEN)).astype(np.float32))
        self.cc.h2d(self.p["tokens"], np.full(self.t, -7, np.int32))

    def get(self, name, shape, kind):
        return self.cc.d2h(self.p[name], shape, kind)

    def results(self):
        t = self.t
        return [self.get("x", (t, HIDDEN), np.uint32), self.get("y", (t, QKV), np.uint16), self.get("logits", (t, VOCAB), np.uint16), self.get("tokens", (t,), np.int32),
                self.get("accepted", (self.seqs,), np.int32)]

    def linear(self, name, x=None):
        """(want, room) of a linear from the quantised rows that are there, or of x"""
        w, sv, n, k = self.w[name]
        q, s = ref.quantised(x) if x is not None else (ops.unpack_q8(self.get("q", (ops.q8_bytes(self.t, k),), np.uint8), self.t, k).view(np.uint8), self.get("s", (-(-k // 128), self.t), np.float32))
        want, a, most = ref.product(q, s, w, sv)
        return want, ref.room(a, most, "f8_tiled", -(-k // 128))  # whichever kernel it was


@pytest.mark.parametrize("lens", [[5], [5, 1, 3], [4] * 30], ids=["t5", "t9", "t120"])
def test_a_step_stage_by_stage_and_replayed(dec, lens):
    with w8.Buffers(dec.cc) as b:
        st = Step(dec, b, lens)
        t, cc = st.t, dec.cc
        st.start(1)
        norms = 0
        for name, go in st.stages():
            print("step", lens[:3], name, flush=True)
            if name == "norm":  # the bits of the norm and of its result's quantisation
                ab = ("ab", "ab2", "ab3")[norms]
                x2 = b.put(st.get("x", (t, HIDDEN), np.float32))
                dec.norm_resid(x2, st.p["nw"], st.p[ab], st.p["norm"], t, HIDDEN, w_off=norms * HIDDEN)
                norms += 1
                q, s = ref.quantised(st.get("norm", (t, HIDDEN), np.float32))
            elif name in ("qkv", "head"):
                want, space = st.linear(name)
            elif name == "rope":
                y = st.get("y", (t, QKV), np.uint16)
            elif name == "o":
                want, space = st.linear("o", st.get("y", (t, QKV), np.float16)[:, :K].astype(np.float32))
            elif name == "down":
                want, space = st.linear("down", st.get("ff", (t, FF), np.float16).astype(np.float32))
            elif name == "gu":
                want, space = st.linear("gu")
            go()
            if name == "norm":
                assert np.array_equal(ops.unpack_q8(st.get("q", (ops.q8_bytes(t, HIDDEN),), np.uint8), t, HIDDEN).view(np.uint8), q) and np.array_equal(st.get("s", (3, t), np.float32), s)
                assert np.array_equal(st.get("x", (t, HIDDEN), np.uint32), cc.d2h(x2, (t, HIDDEN), np.uint32))
            elif name == "qkv":
                ref.near(st.get("y", (t, QKV), np.float16), want, space, ffi.F16)
            elif name == "head":
                ref.near(st.get("logits", (t, VOCAB), np.float16), want, space, ffi.F16)
            elif name in ("o", "down"):
                ref.near(st.get("ab2" if name == "o" else "ab3", (t, HIDDEN), np.float32), want, space, ffi.F32)
            elif name == "gu":
                g, v = want[:, :FF], want[:, FF:]
                act = g / (1 + np.exp(-g))
                # silu's slope is 1.1 at most, and 2^-20 of its value for its own arithmetic
                ref.near(st.get("ff", (t, FF), np.float16), act * v, 1.1 * space[:, :FF] * (np.abs(v) + space[:, FF:]) + np.abs(act) * (space[:, FF:] + 2.0**-20 * np.abs(v)), ffi.F16)
            elif name == "rope":
                got, before = st.get("y", (t, QKV), np.float16), y.view(np.float16).astype(np.float32)
                for first, heads, w in ((0, NQ, st.qw), (K, NK, st.kw)):
                    cols = slice(first, first + heads * DIM)
                    want, space = rotated(before[:, cols], t, heads, DIM, w, 1e-6, st.pos, st.freqs, st.amp, False)
                    ref.near(got[:, cols].reshape(t, heads, DIM), want, space, ffi.F16)
                assert np.array_equal(got[:, K + NK * DIM:].view(np.uint16), y[:, K + NK * DIM:])  # values stay
            else:
                want = verify_ref.verified(st.get("logits", (t, VOCAB), np.float16).astype(np.float32), st.dbits.astype(np.float32), st.row0, st.drafted, st.u, st.temps, np.full(t, -7, np.int32))
                assert np.array_equal(st.get("tokens", (t,), np.int32), want[0]) and np.array_equal(st.get("accepted", (st.seqs,), np.int32), want[1])
        eager = {}
        for seed in (1, 2, 3):
            st.start(seed)
            for _, go in st.stages():
                go()
            eager[seed] = st.results()
        cc.capture_begin()
        for _, go in st.stages():
            go()
        graph = cc.capture_end()
        for seed in (2, 3, 1, 1, 2):
            st.start(seed)
            graph.launch()
            cc.sync()
            assert all(np.array_equal(a, c) for a, c in zip(st.results(), eager[seed])), seed
            dec.quant_rows_f8(st.p["ab"], st.p["q"], st.p["s"], t, HIDDEN, x_type=ffi.F32)  # eager work between them
        graph.destroy()


def test_two_contexts_and_two_graphs_at_once(dec):
    """Launches of two contexts without a wait between them, and two graphs over one scratch: the results of one after the other."""
    other = ops.W4a16Dec()
    try:
        with w8.Buffers(dec.cc) as b0, w8.Buffers(other.cc) as b1:
            steps = [Step(dec, b0, [5, 2]), Step(other, b1, [3] * 9)]
            want = []
            for st in steps:
                per = []
                for seed in (11, 12):
                    st.start(seed)
                    for _, go in st.stages():
                        go()
                    per.append(st.results())
                want.append(per)
            for at, seed in enumerate((11, 12)):
                for st in steps:
                    st.start(seed)
                for (_, a), (_, c) in zip(steps[0].stages(), steps[1].stages()):  # in turns
                    a()
                    c()
                for st, per in zip(steps, want):
                    st.cc.sync()
                    assert all(np.array_equal(x, y) for x, y in zip(st.results(), per[at]))
            more = Step(dec, b0, [4, 4, 1])
            more.start(13)
            for _, go in more.stages():
                go()
            alone = more.results()
            graphs = []
            for st in (steps[0], more):
                st.cc.capture_begin()
                for _, go in st.stages():
                    go()
                graphs.append(st.cc.capture_end())
            for _ in range(3):
                steps[0].start(12)
                more.start(13)
                for g in graphs:
                    g.launch()
                dec.cc.sync()
                assert all(np.array_equal(x, y) for x, y in zip(steps[0].results(), want[0][1])) and all(np.array_equal(x, y) for x, y in zip(more.results(), alone))
            for g in graphs:
                g.destroy()
    finally:
        other.cc.close()
