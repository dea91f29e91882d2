"""Linears in 8-bit floating point with a scale for each block of 128, the norm of queries and keys with the rotation by position, and the
verification of drafted tokens: what a model's pass over a few drafted tokens takes beside the operators that are here, and what each computes.

A case is a dict of plain values:
  kind "linear"  `layers` times: a token row block x [t][k] (x_type f16 | f32 | bf16) through a linear [n][k].  parts = 1: the
                 linear quantises x itself; parts > 1: x is quantised once and read by so many linears, as q, k and v do.
                 glu: rows 0..n/2 are a gate and n/2..n its values, the result is silu(gate) * value, [t][n/2]
  kind "mlp"     `layers` times: residual add, RMS norm and quantisation, the gated projection, the down projection
  kind "qk"      rows of a QKV projection [t][(n_q + n_k) * dim + rest]: every head's norm (norm: with weights, one set for queries and one for keys)
                 and the rotation of its first `rot` elements by the row's position; pairs are (c, c + rot / 2), or (2 c, 2 c + 1) where
                 interleaved.  scaling: of the frequencies, for contexts longer than trained on
  kind "verify"  `seqs` sequences with up to `most` drafted tokens each (exactly so many, or ragged: 0 to `most`): target logits for every drafted token
                 and for the one behind them; drafts: with the draft's own logits, else each drafted token was certain to its draft.
                 greedy: the share of sequences at temperature 0

Definitions.  A block of 128 of a row is quantised in steps of s = 2^max(-126, ceil(log2(max |x| / 448))), 0 for zeros; q is the e4m3 number nearest to x / s
(halves to the even one).  A linear gives sum over blocks b of sx[m][b] * sw[row / 128][b] * sum_k q[m][k] * w[row][k].  A head becomes
v / sqrt(mean v^2 + 1e-6) * weight, then (a cos - b sin, b cos + a sin) for each pair, both times `amp`, angle = position * frequency.  Drafted token j of a
sequence, x, is accepted while u_j q_j(x) < p_j(x), p and q the softmax of target and draft logits over the temperature.  Behind the last one
accepted comes one token more: of max(0, p - q) where a draft was rejected, of p behind the last draft, the first whose running sum exceeds the sequence's
last u times the whole sum.  At temperature 0 a draft is accepted if it is the most likely token (of equal ones the lowest), which is the token behind, too.
"""
import math
import weakref

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# Layer shapes of the repository's benchmark and tests (n, k): the 27B dense layer (QKV, O, gate|up, down) and an 8B-like one
DENSE = [(7168, 5120), (5120, 5120), (34816, 5120), (5120, 17408), (6144, 4096), (4096, 4096), (22016, 4096), (4096, 11008)]


def listed():
    return [
        # one token through square linears of a small layer: latency and launches of a decode step of one sequence
        {"name": "linear_t1_4096", "kind": "linear", "n": 4096, "k": 4096, "t": 1, "x_type": "f16", "y_type": "f16", "glu": False,
         "parts": 1, "layers": 4},
        # five rows, a token and four drafted ones, through the widest projection of the 27B layer: the weight stream of a verifying step
        {"name": "glu_t5_27b", "kind": "linear", "n": 34816, "k": 5120, "t": 5, "x_type": "f16", "y_type": "f16", "glu": True,
         "parts": 1, "layers": 1},
        # sixteen rows, the down projection: few output rows, a long k
        {"name": "linear_t16_down_27b", "kind": "linear", "n": 5120, "k": 17408, "t": 16, "x_type": "f16", "y_type": "f32",
         "glu": False, "parts": 1, "layers": 2},
        # an odd batch through two linears of odd sizes that share their input
        {"name": "shared_t37_odd", "kind": "linear", "n": 5003, "k": 2051, "t": 37, "x_type": "bf16", "y_type": "bf16", "glu": False,
         "parts": 2, "layers": 2},
        # a short prompt of ragged length, or 60 sequences of five rows, through the 27B layer's FFN
        {"name": "mlp_t300_27b", "kind": "mlp", "hidden": 5120, "n_ff": 17408, "t": 300, "layers": 1},
        # a long prompt chunk through the widest projection: the largest call
        {"name": "glu_t4096_27b", "kind": "linear", "n": 34816, "k": 5120, "t": 4096, "x_type": "f16", "y_type": "f16", "glu": True,
         "parts": 1, "layers": 1},
        # one token's queries and keys of the 27B layer's QKV projection, far into a long context
        {"name": "qk_t1_27b", "kind": "qk", "n_q": 40, "n_k": 8, "dim": 128, "rot": 128, "rest": 1024, "t": 1, "x_type": "f32", "y_type": "f16",
         "norm": True, "interleaved": False, "scaling": "ramp", "from": 100000},
        # rows of odd heads, a part of them turned, neighbours as pairs, no norm
        {"name": "qk_t333_part", "kind": "qk", "n_q": 13, "n_k": 3, "dim": 80, "rot": 20, "rest": 7, "t": 333, "x_type": "bf16", "y_type": "bf16",
         "norm": False, "interleaved": True, "scaling": "plain", "from": 0},
        # a long prompt chunk of the 27B layer
        {"name": "qk_t8192_27b", "kind": "qk", "n_q": 40, "n_k": 8, "dim": 128, "rot": 128, "rest": 1024, "t": 8192, "x_type": "f16", "y_type": "f16",
         "norm": True, "interleaved": False, "scaling": "bands", "from": 0},
        # one sequence, four tokens drafted by a lookup in what was said before: no draft logits
        {"name": "verify_b1_32000", "kind": "verify", "seqs": 1, "most": 4, "ragged": False, "vocab": 32000, "type": "f32", "drafts": False,
         "masked": False, "greedy": 0.0},
        # a serving batch, up to four drafts each with their logits, a quarter of the sequences greedy
        {"name": "verify_b64_131072", "kind": "verify", "seqs": 64, "most": 4, "ragged": True, "vocab": 131072, "type": "bf16", "drafts": True,
         "masked": False, "greedy": 0.25},
        # a vocabulary of odd size under a grammar's mask, one draft each
        {"name": "verify_b200_odd", "kind": "verify", "seqs": 200, "most": 1, "ragged": False, "vocab": 100003, "type": "f16", "drafts": True,
         "masked": True, "greedy": 0.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "mlp", "qk", "qk", "verify", "verify"])
    if kind == "linear":
        if rng.random() < 0.4:
            n, k = rng.choice(DENSE)
        else:
            n, k = _log_int(rng, 16, 40000), _log_int(rng, 64, 17408)
            if rng.random() < 0.6:
                k = max(128, k // 128 * 128)
        glu = rng.random() < 0.3
        if not glu and rng.random() < 0.5:
            n = max(16, n // 16 * 16)
        n = min(n, 34816 * 5120 // k)
        n = max(256, n // 256 * 256) if glu else n
        t = _log_int(rng, 1, 4096)
        while 2.0 * t * n * k > 1.4e12:
            t = (t * 3) // 4
        parts = 1 if glu else rng.choice([1, 1, 1, 2, 3])
        layers = 1 if t > 256 or n * k * parts > 3e7 else 2
        while parts > 1 and parts * (2.0 * t * n * k) > 1.4e12:
            parts -= 1
        return {"kind": kind, "n": n, "k": k, "t": t, "x_type": rng.choice(["f16", "f16", "f32", "bf16"]),
                "y_type": rng.choice(["f16", "f32", "bf16"]), "glu": glu, "parts": parts, "layers": layers}
    if kind == "mlp":
        hidden, n_ff = rng.choice([(5120, 17408), (4096, 11008), (2560, 6912), (2048, 5632)])
        t = _log_int(rng, 1, 1000)
        return {"kind": kind, "hidden": hidden, "n_ff": n_ff, "t": t, "layers": 2 if t <= 64 and hidden < 5000 else 1}
    if kind == "qk":
        dim = rng.choice([64, 80, 96, 128, 128, 128, 256, 2 * rng.randint(8, 128)])
        rot = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        n_q = _log_int(rng, 1, 64)
        n_k, t, rest = rng.randint(1, min(n_q, 16)), _log_int(rng, 1, 8192), rng.choice([0, 0, 7, 1024])
        while t > 1 and t * (n_q + n_k) * dim > 8192 * 48 * 128:
            t = t * 3 // 4
        return {"kind": kind, "n_q": n_q, "n_k": n_k, "dim": dim, "rot": rot, "rest": rest, "t": t, "x_type": rng.choice(["f32", "f16", "bf16"]),
                "y_type": rng.choice(["f32", "f16", "bf16"]), "norm": rng.random() < 0.7, "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(["plain", "linear", "bands", "ramp"]), "from": rng.choice([0, rng.randint(0, 1000000)])}
    vocab, kt = _log_int(rng, 200, 260000), rng.choice(["f32", "f16", "bf16"])
    if rng.random() < 0.5:
        vocab = max(200, vocab // 64 * 64)
    most, drafts = rng.choice([0, 1, 2, 4, 7]), rng.random() < 0.6
    seqs = _log_int(rng, 1, 256)
    while seqs > 1 and seqs * (most + 1) * vocab > 320 * 131072:
        seqs = seqs * 3 // 4
    return {"kind": kind, "seqs": seqs, "most": most, "ragged": rng.random() < 0.5, "vocab": vocab, "type": kt, "drafts": drafts,
            "masked": rng.random() < 0.3, "greedy": rng.choice([0.0, 0.0, 0.3, 1.0])}


class _Program:
    """A program's one library context, shared by every state that is alive, and the name slots its models use."""

    def __init__(self):
        from llm170_amd import ops

        self.dec = ops.W4a16Dec()
        self.slots = []
        self.taken = 0

    def slot(self):
        if self.slots:
            return self.slots.pop()
        self.taken += 1
        return self.taken - 1


_live = weakref.WeakValueDictionary()


class _State:
    """What a program holds: weights (registered with the library where it is used), inputs and result buffers."""

    def __init__(self, case):
        self.case, self.program, self.prefix = case, None, ""
        if own:
            self.program = _live.get("program")
            if self.program is None:
                self.program = _live["program"] = _Program()
            slot = self.program.slot()
            self.prefix = "f%d" % slot
            weakref.finalize(self, self.program.slots.append, slot)  # the names are used again by the next model

    def linear(self, g, name, n, k):
        """Weights of one linear: e4m3 [n][k], f32 scales for each block of 128 x 128."""
        nb, kb = (n + 127) // 128, (k + 127) // 128
        w = (torch.randn((n, k), device="cuda", generator=g) * 140).clamp(-448, 448).to(torch.float8_e4m3fn)
        ws = (torch.rand((nb, kb), device="cuda", generator=g) * 1.5 + 0.5) / (140 * math.sqrt(k))
        if own:
            self.program.dec.upload_lin_f8(name, w.view(torch.uint8).cpu().numpy(), ws.cpu().numpy(), n, k)
        return _Lin(name, w, ws)


class _Lin:
    def __init__(self, name, w, ws):
        self.name, self.w, self.ws = name, w, ws


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _empty(*shape, dtype=torch.float32):
    return torch.empty(shape, device="cuda", dtype=dtype)


def _q8(t, k):
    """Room for t quantised rows of k, in whole tiles."""
    return _empty((t + 15) // 16 * 16, (k + 127) // 128 * 128, dtype=torch.uint8)


def _scales(t, k):
    return _empty((k + 127) // 128, t)


# What a context of 32768 positions is stretched by, and its bounds: turns within the trained length (ramp), parts of it as wavelengths (bands)
SCALING = {"plain": {}, "linear": {"factor": 4.0}, "bands": {"factor": 8.0, "low": 1.0, "high": 4.0}, "ramp": {"factor": 4.0, "low": 1.0, "high": 32.0}}
BASE, TRAINED = 1000000.0, 32768.0


def _frequencies(rot, scaling):
    """(radians per position of each pair in 64 bits, amplitude)"""
    c = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    f, p = BASE ** (-2 * c / rot), SCALING[scaling]
    if scaling == "linear":
        return f / p["factor"], 1.0
    if scaling == "bands":
        share = ((TRAINED * f / (2 * math.pi) - p["low"]) / (p["high"] - p["low"])).clamp(0, 1)
        return f * ((1 - share) / p["factor"] + share), 1.0
    if scaling == "ramp":
        at = lambda turns: rot * math.log(TRAINED / (2 * math.pi * turns)) / (2 * math.log(BASE))  # noqa: E731
        lo, hi = max(math.floor(at(p["high"])), 0), min(math.ceil(at(p["low"])), rot - 1)
        ramp = ((c - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * ((1 - ramp) + ramp / p["factor"]), 0.1 * math.log(p["factor"]) + 1
    return f, 1.0


def _drafted(c):
    """Drafted tokens of each sequence; ragged: 0 to `most` in turn."""
    i = torch.arange(c["seqs"])
    return (7 * i + 3) % (c["most"] + 1) if c["ragged"] else torch.full_like(i, c["most"])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, c = _State(case), case
    if c["kind"] == "linear":
        t, n, k, y = c["t"], c["n"], c["k"], TYPES[c["y_type"]]
        s.lins = [[s.linear(g, "%s.%d.%d" % (s.prefix, i, p), n, k) for p in range(c["parts"])] for i in range(c["layers"])]
        s.x = [_randn(g, t, k, dtype=TYPES[c["x_type"]]) for _ in s.lins]
        s.y = [[_empty(t, n // 2 if c["glu"] else n, dtype=y) for _ in parts] for parts in s.lins]
        s.q, s.s = _q8(t, k), _scales(t, k)
    elif c["kind"] == "mlp":
        t, h, f = c["t"], c["hidden"], c["n_ff"]
        s.lins = [[s.linear(g, "%s.%d.gate_up" % (s.prefix, i), 2 * f, h), s.linear(g, "%s.%d.down" % (s.prefix, i), h, f)] for i in range(c["layers"])]
        s.x, s.ab = [_randn(g, t, h) * 4 for _ in s.lins], [_randn(g, t, h) for _ in s.lins]
        s.nw = [1 + 0.1 * _randn(g, h) for _ in s.lins]
        s.q, s.s, s.a = _q8(t, h), _scales(t, h), _empty(t, f, dtype=torch.float16)
        s.y = [_empty(t, h, dtype=torch.float16) for _ in s.lins]
    elif c["kind"] == "qk":
        t, d, y = c["t"], c["dim"], TYPES[c["y_type"]]
        s.x = (_randn(g, t, (c["n_q"] + c["n_k"]) * d + c["rest"]) * 1.7).to(TYPES[c["x_type"]])
        s.qw, s.kw = (1 + 0.2 * _randn(g, d), 1 + 0.2 * _randn(g, d)) if c["norm"] else (None, None)
        s.pos = torch.arange(c["from"], c["from"] + t, dtype=torch.int32, device="cuda")
        s.freqs, s.amp = _frequencies(c["rot"], c["scaling"])
        if own:
            from llm170_amd import ffi, ops

            kinds = {"plain": ffi.ROPE_PLAIN, "linear": ffi.ROPE_LINEAR, "bands": ffi.ROPE_BANDS, "ramp": ffi.ROPE_RAMP}
            freqs, s.amp = ops.rope_freqs(c["rot"], BASE, kinds[c["scaling"]], trained=TRAINED, **SCALING[c["scaling"]])
            s.freqs = torch.from_numpy(freqs).cuda()
        s.q, s.k = _empty(t, c["n_q"] * d, dtype=y), _empty(t, c["n_k"] * d, dtype=y)
    else:
        b, v = c["seqs"], c["vocab"]
        drafted = _drafted(c)
        s.row0 = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(drafted + 1, 0)]).to(torch.int32).cuda()
        t = s.t = int(drafted.sum()) + b
        s.temps = torch.rand(b, device="cuda", generator=g) * 0.6 + 0.6
        s.temps[torch.rand(b, device="cuda", generator=g) < c["greedy"]] = 0.0
        z = _randn(g, t, v) * 2.5
        z.scatter_add_(1, torch.randint(0, v, (t, 3), device="cuda", generator=g), torch.full((t, 3), 9.0, device="cuda"))
        d = z + _randn(g, t, v) * 0.5
        if c["masked"]:
            z[torch.rand(t, v, device="cuda", generator=g) < 0.7] = -math.inf
        s.logits, d = z.to(TYPES[c["type"]]), d.to(TYPES[c["type"]])
        s.draft = d if c["drafts"] else None
        noise = -torch.log(torch.rand((t, v), device="cuda", generator=g).clamp(min=1e-30))
        s.drafted = (d.float() - torch.log(noise.clamp(min=1e-30))).argmax(1).to(torch.int32)
        s.u = torch.rand(t, device="cuda", generator=g)
        s.tokens, s.accepted = _empty(t, dtype=torch.int32), _empty(b, dtype=torch.int32)
    torch.cuda.synchronize()  # the library launches on a stream of its own
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _e4m3(v):
    """The e4m3 number nearest to each v, halves to the even one; |v| <= 448."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6)))) / 8  # three bits behind the leading one; from 2^-6 down all alike
    return torch.round(v / step) * step


def _quantised(x):
    """(x in steps, steps [t][blocks]), x padded to whole blocks.  The steps are powers of two: every quotient is exact."""
    x = x.float()
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 128)).reshape(x.shape[0], -1, 128)
    most = x.abs().amax(2)
    s = torch.exp2(torch.ceil(torch.log2(most.double() / 448)).clamp(min=-126)).float()
    q = torch.where((most > 0)[:, :, None], _e4m3(x / s[:, :, None]), torch.zeros_like(x))
    return q, torch.where(most > 0, s, torch.zeros_like(s))


def _product(q, s, lin):
    n, k = lin.w.shape
    x = (q * s[:, :, None]).reshape(q.shape[0], -1)[:, :k]
    w = lin.w.float() * lin.ws.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ w.T


def _silu_mul(g, u):
    return g / (1 + torch.exp(-g)) * u


def _gated(y):
    f = y.shape[1] // 2
    return _silu_mul(y[:, :f], y[:, f:])


def _turned(x, weight, s, interleaved):
    """x [t][heads][dim]"""
    x = x.float()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-6) * weight
    rot = 2 * len(s.freqs)
    angle = s.pos.double()[:, None] * s.freqs  # far positions: in 64 bits
    cos, sin = (torch.cos(angle) * s.amp).float()[:, None], (torch.sin(angle) * s.amp).float()[:, None]
    part = x[:, :, :rot]
    a, b = (part[:, :, 0::2], part[:, :, 1::2]) if interleaved else (part[:, :, : rot // 2], part[:, :, rot // 2 :])
    both = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(both, 3).flatten(2) if interleaved else torch.cat(both, 2)
    return torch.cat([turned, x[:, :, rot:]], 2).flatten(1)


def _verified(s):
    """In 64 bits: running sums over a vocabulary, and numbers next to a border."""
    c, v = s.case, s.case["vocab"]
    rows, row0 = torch.arange(s.t, device="cuda"), s.row0.long()
    seq = torch.searchsorted(row0, rows, right=True) - 1
    last = rows == row0[seq + 1] - 1
    temp = s.temps.double()[seq][:, None]
    greedy = temp[:, 0] == 0
    temp = torch.where(temp == 0, torch.ones_like(temp), temp)
    z = s.logits.double()
    x = s.drafted.long()[:, None]
    p = torch.softmax((z - z.amax(1, keepdim=True)) / temp, 1)
    if c["drafts"]:
        d = s.draft.double()
        q = torch.softmax((d - d.amax(1, keepdim=True)) / temp, 1)
    else:
        q = torch.zeros_like(p).scatter_(1, x, 1.0)
    best = z.argmax(1)
    best = torch.where(z == z.amax(1, keepdim=True), torch.arange(v, device="cuda"), v).amin(1)
    fine = torch.where(greedy, best == x[:, 0], s.u.double() * q.gather(1, x)[:, 0] < p.gather(1, x)[:, 0]) & ~last
    # rows up to which all before are accepted: the first that is not, of each sequence
    stop = torch.full((c["seqs"],), s.t, device="cuda").scatter_reduce_(0, seq, torch.where(fine, s.t, rows), "amin")
    p, q = p[stop], torch.where(last[stop][:, None], torch.zeros_like(q[stop]), q[stop])
    r = (p - q).clamp(min=0)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
    run = torch.cumsum(r, 1)
    at = (run <= s.u.double()[row0[1:] - 1][:, None] * run[:, -1:]).sum(1)
    token = torch.where(s.temps == 0, best[stop], at.clamp(max=v - 1))
    tokens = torch.where(rows < stop[seq], x[:, 0], torch.where(rows == stop[seq], token[seq], -1))
    return tokens.to(torch.int32), (stop - row0[:-1]).to(torch.int32)


def _run_plain(s):
    c = s.case
    if c["kind"] == "linear":
        got = []
        for x, parts in zip(s.x, s.lins):
            q, sx = _quantised(x)
            y = [_product(q, sx, lin) for lin in parts]
            got.append([(_gated(v) if c["glu"] else v).to(TYPES[c["y_type"]]) for v in y])
        return got
    if c["kind"] == "mlp":
        got = []
        for x, ab, nw, (gate_up, down) in zip(s.x, s.ab, s.nw, s.lins):
            x += ab
            q, sx = _quantised(x * (1 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)) * nw)
            q, sx = _quantised(_gated(_product(q, sx, gate_up)).half())
            got.append(_product(q, sx, down).half())
        return s.x, got
    if c["kind"] == "qk":
        d, nq, y = c["dim"], c["n_q"], TYPES[c["y_type"]]
        heads = s.x[:, : (nq + c["n_k"]) * d].reshape(c["t"], -1, d)
        return [_turned(heads[:, :nq], s.qw, s, c["interleaved"]).to(y), _turned(heads[:, nq:], s.kw, s, c["interleaved"]).to(y)]
    return _verified(s)


# ---------------------------------------------------------------------------------------------- the library's calls
def _run_own(s):
    from llm170_amd import ffi

    c, dec = s.case, s.program.dec
    code = {"f32": ffi.F32, "f16": ffi.F16, "bf16": ffi.BF16}
    if c["kind"] == "linear":
        t = c["t"]
        for x, parts, ys in zip(s.x, s.lins, s.y):
            if c["parts"] > 1:
                dec.quant_rows_f8(x.data_ptr(), s.q.data_ptr(), s.s.data_ptr(), t, c["k"], x_type=code[c["x_type"]])
            for lin, y in zip(parts, ys):
                if c["parts"] > 1:
                    dec.lin_forward_f8(lin.name, s.q.data_ptr(), y.data_ptr(), t, x_type=ffi.F8, xs_dev=s.s.data_ptr(), y_type=code[c["y_type"]])
                elif c["glu"]:
                    dec.lin_forward_f8_glu(lin.name, x.data_ptr(), y.data_ptr(), t, x_type=code[c["x_type"]], y_type=code[c["y_type"]])
                else:
                    dec.lin_forward_f8(lin.name, x.data_ptr(), y.data_ptr(), t, x_type=code[c["x_type"]], y_type=code[c["y_type"]])
        return s.y
    if c["kind"] == "mlp":
        t = c["t"]
        for x, ab, nw, (gate_up, down), y in zip(s.x, s.ab, s.nw, s.lins, s.y):
            dec.norm_resid_f8(x.data_ptr(), nw.data_ptr(), ab.data_ptr(), s.q.data_ptr(), s.s.data_ptr(), t, c["hidden"])
            dec.lin_forward_f8_glu(gate_up.name, s.q.data_ptr(), s.a.data_ptr(), t, x_type=ffi.F8, xs_dev=s.s.data_ptr(), y_type=ffi.F16)
            dec.lin_forward_f8(down.name, s.a.data_ptr(), y.data_ptr(), t, x_type=ffi.F16, y_type=ffi.F16)
        return s.x, s.y
    if c["kind"] == "qk":
        dec.qk_norm_rope(s.x.data_ptr(), s.q.data_ptr(), s.k.data_ptr(), s.pos.data_ptr(), s.freqs.data_ptr(), c["t"], c["n_q"], c["n_k"], c["dim"],
                         c["rot"], x_type=code[c["x_type"]], ldx=s.x.shape[1], y_type=code[c["y_type"]], qw_dev=s.qw.data_ptr() if c["norm"] else 0,
                         kw_dev=s.kw.data_ptr() if c["norm"] else 0, amp=s.amp, interleaved=c["interleaved"])
        return [s.q, s.k]
    dec.verify_drafts(s.logits.data_ptr(), s.drafted.data_ptr(), s.row0.data_ptr(), s.u.data_ptr(), s.tokens.data_ptr(), s.accepted.data_ptr(), s.t,
                      c["seqs"], c["vocab"], logits_type=code[c["type"]], draft_dev=s.draft.data_ptr() if c["drafts"] else 0, temps_dev=s.temps.data_ptr())
    return s.tokens, s.accepted


def run(s):
    return _run_own(s) if own else _run_plain(s)


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    scales = lambda n, k: 4 * ((n + 127) // 128) * ((k + 127) // 128)  # noqa: E731
    if c["kind"] == "linear":
        t, n, k, out = c["t"], c["n"], c["k"], c["n"] // 2 if c["glu"] else c["n"]
        return {"bytes": c["layers"] * (t * k * size[c["x_type"]] + c["parts"] * (n * k + scales(n, k) + t * out * size[c["y_type"]])),
                "flops": 2.0 * c["layers"] * c["parts"] * t * n * k}
    if c["kind"] == "mlp":
        t, h, f = c["t"], c["hidden"], c["n_ff"]
        return {"bytes": c["layers"] * (3 * f * h + scales(2 * f, h) + scales(h, f) + 4 * h + t * h * (3 * 4 + 2)), "flops": 2.0 * c["layers"] * t * 3 * f * h}
    if c["kind"] == "qk":
        heads = c["n_q"] + c["n_k"]
        return {"bytes": c["t"] * (heads * c["dim"] * (size[c["x_type"]] + size[c["y_type"]]) + 4) + 4 * c["rot"] + (8 * c["dim"] if c["norm"] else 0),
                "flops": c["t"] * heads * (4.0 * c["dim"] + 3.0 * c["rot"])}
    drafted = int(_drafted(c).sum())  # a row each, judged, and one more for each sequence
    # sampled sequences read the draft's rows beside the target's
    rows = drafted + c["seqs"] + (drafted * (1 - c["greedy"]) if c["drafts"] else 0)
    return {"bytes": int(rows * c["vocab"] * size[c["type"]] + (drafted + c["seqs"]) * 12 + c["seqs"] * 12), "flops": 3.0 * rows * c["vocab"]}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["kind"] == "verify":
        return None  # whole numbers
    s, c = prepare(case, seed), case

    def through(x, lin):  # rows of 64-bit values, block by block
        n, k = lin.w.shape
        y = torch.zeros(len(x), n, dtype=torch.float64, device="cuda")
        for at in range(0, k, 128):
            block = x[:, at : at + 128]
            exponent = torch.frexp(block.abs().amax(1, keepdim=True) / 448)
            up = exponent.exponent - (exponent.mantissa == 0.5).int()  # the least power of two that is no smaller
            size = torch.ldexp(torch.ones_like(block[:, :1]), up.clamp(min=-126))
            q = (block / size).to(torch.float32)
            lead = (torch.frexp(q).exponent - 1).clamp(min=-6)  # three bits behind the leading one
            q = torch.ldexp(torch.round(torch.ldexp(q, 3 - lead)), lead - 3).double()
            scale = lin.ws[:, at // 128].double()[torch.arange(n, device="cuda") // 128]
            y += (q * size) @ (lin.w[:, at : at + 128].to(torch.float64).t()) * scale
        return y

    def gate(y):
        a, b = y.chunk(2, dim=1)
        return a * torch.special.expit(a) * b

    if c["kind"] == "linear":
        got = [[through(x.to(torch.float64), lin) for lin in parts] for x, parts in zip(s.x, s.lins)]
        return [[gate(y) for y in ys] for ys in got] if c["glu"] else got
    if c["kind"] == "mlp":
        xs, ys = [], []
        for x, ab, nw, (gate_up, down) in zip(s.x, s.ab, s.nw, s.lins):
            v = x.to(torch.float64) + ab.to(torch.float64)
            xs.append(v)
            v = v.to(torch.float32).double()  # the residual stream is held in 32 bits
            normed = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6) * nw.to(torch.float64)
            ys.append(through(gate(through(normed, gate_up)).to(torch.float16).double(), down))
        return xs, ys

    half = c["rot"] // 2
    wheel = torch.polar(torch.full((c["t"], half), float(s.amp), dtype=torch.float64, device="cuda"), torch.outer(s.pos.double(), s.freqs))[:, None]
    at = torch.arange(c["rot"], device="cuda")
    order = torch.stack([at[0::2], at[1::2]]) if c["interleaved"] else at.reshape(2, half)

    def heads(first, count, weight):
        v = s.x[:, first * c["dim"] : (first + count) * c["dim"]].double().unflatten(1, (count, c["dim"]))
        if weight is not None:
            v = v * torch.rsqrt(v.square().mean(2, keepdim=True) + 1e-6) * weight.double()
        else:
            v = v.clone()
        turned = torch.complex(v[:, :, order[0]], v[:, :, order[1]]) * wheel
        v[:, :, order[0]], v[:, :, order[1]] = turned.real, turned.imag
        return v.flatten(1)

    return [heads(0, c["n_q"], s.qw), heads(c["n_q"], c["n_k"], s.kw)]
