"""W8A8 linears (8-bit weights with a scale per output channel, activations quantised per token) and the scoring of
the logits that a head made of one gives: what these operators compute and what a pass through them takes.

A case is a dict of plain values:
  kind "linear"  `layers` times: a token row block x [t][k] (x_type f16 | f32 | bf16) through a linear [n][k].  parts = 1: the
                 linear quantises x itself; parts > 1: x is quantised once and read by so many linears, as q, k and v do.
                 glu: rows 0..n/2 are a gate and n/2..n its values, the result is silu(gate) * value, [t][n/2]
  kind "mlp"     `layers` times: residual add, RMS norm and quantisation, the gated projection, the down projection
  kind "score"   for every row of logits [t][vocab] the log probability of a given token (-1: none is asked for), the
                 entropy of the distribution and the `top` most likely tokens.  masked: some tokens are ruled out (-inf)
  kind "head"    hidden states through a linear to the vocabulary, and the scoring of its logits

Definitions.  A row is quantised as s = fl32(max |x| / 127), q = the whole number nearest to x / s (halves to the even
one), both 0 where s < 2^-126.  A linear gives (sum_k q[m][k] * w[n][k]) * s[m] * ws[n].  Of logits z the log
probability of token j is z_j - log(sum exp z), the entropy is -sum p log p, and of equal logits the lower token comes first.
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
        # one token, three projections that share their input: quantised once
        {"name": "shared_t1_5120", "kind": "linear", "n": 7168, "k": 5120, "t": 1, "x_type": "f32", "y_type": "f32", "glu": False,
         "parts": 3, "layers": 1},
        # one token through the widest projection of the 27B layer: the weight stream of a decode step
        {"name": "glu_t1_27b", "kind": "linear", "n": 34816, "k": 5120, "t": 1, "x_type": "f16", "y_type": "f16", "glu": True,
         "parts": 1, "layers": 1},
        # sixteen sequences, the down projection: few output rows, a long k
        {"name": "linear_t16_down_27b", "kind": "linear", "n": 5120, "k": 17408, "t": 16, "x_type": "f16", "y_type": "f32",
         "glu": False, "parts": 1, "layers": 2},
        # an odd batch through two linears of odd sizes that share their input
        {"name": "shared_t37_odd", "kind": "linear", "n": 5003, "k": 2051, "t": 37, "x_type": "bf16", "y_type": "bf16", "glu": False,
         "parts": 2, "layers": 2},
        # a decode step of four sequences through a layer's gated FFN, norm to down projection
        {"name": "mlp_t4_8b", "kind": "mlp", "hidden": 4096, "n_ff": 11008, "t": 4, "layers": 2},
        # a short prompt of ragged length through the 27B layer's FFN
        {"name": "mlp_t300_27b", "kind": "mlp", "hidden": 5120, "n_ff": 17408, "t": 300, "layers": 1},
        # a long prompt chunk through the widest projection: the largest call
        {"name": "glu_t4096_27b", "kind": "linear", "n": 34816, "k": 5120, "t": 4096, "x_type": "f16", "y_type": "f16", "glu": True,
         "parts": 1, "layers": 1},
        # one token's logits, five alternatives: what a served decode step returns
        {"name": "score_t1_32000", "kind": "score", "vocab": 32000, "t": 1, "type": "f32", "top": 5, "masked": False},
        # a serving batch under a grammar's mask, twenty alternatives
        {"name": "score_t64_131072", "kind": "score", "vocab": 131072, "t": 64, "type": "bf16", "top": 20, "masked": True},
        # a prompt's tokens scored, a vocabulary of odd size
        {"name": "score_t2048_odd", "kind": "score", "vocab": 100003, "t": 2048, "type": "f16", "top": 1, "masked": False},
        # the head of a decode step of four sequences and its scoring
        {"name": "head_t4_131072", "kind": "head", "vocab": 131072, "k": 5120, "t": 4, "top": 20},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "mlp", "score", "score", "head"])
    if kind == "linear":
        if rng.random() < 0.4:
            n, k = rng.choice(DENSE)
        else:
            n, k = _log_int(rng, 16, 40000), _log_int(rng, 64, 17408)
            if rng.random() < 0.6:
                k = max(64, k // 64 * 64)
        glu = rng.random() < 0.3
        if glu:
            n = max(32, n // 32 * 32)
        elif rng.random() < 0.5:
            n = max(16, n // 16 * 16)
        n = min(n, 34816 * 5120 // k)
        n = max(32, n // 32 * 32) if glu else n
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
    if kind == "score":
        vocab, kt = _log_int(rng, 200, 260000), rng.choice(["f32", "f16", "bf16"])
        if rng.random() < 0.5:
            vocab = max(200, vocab // 64 * 64)
        t = min(_log_int(rng, 1, 4096), int(4e8 / (vocab * (4 if kt == "f32" else 2))))
        return {"kind": kind, "vocab": vocab, "t": t, "type": kt, "top": rng.choice([0, 1, 5, 20, 32]), "masked": rng.random() < 0.3}
    return {"kind": kind, "vocab": _log_int(rng, 4000, 131072), "k": rng.choice([1024, 2048, 4096, 5120]), "t": _log_int(rng, 1, 24),
            "top": rng.choice([1, 5, 20])}


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
            self.prefix = "w%d" % slot
            weakref.finalize(self, self.program.slots.append, slot)  # the names are used again by the next model

    def linear(self, g, name, n, k):
        """Weights of one linear: int8 [n][k], f32 [n]."""
        w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
        ws = (torch.rand(n, device="cuda", generator=g) * 1.5 + 0.5) / (73.3 * math.sqrt(k))
        if own:
            self.program.dec.upload_lin_w8a8(name, w.cpu().numpy(), ws.cpu().numpy(), n, k)
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
    return _empty((t + 15) // 16 * 16, (k + 127) // 128 * 128, dtype=torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s, c, t = _State(case), case, case["t"]
    if c["kind"] == "linear":
        n, k, y = c["n"], c["k"], TYPES[c["y_type"]]
        s.lins = [[s.linear(g, "%s.%d.%d" % (s.prefix, i, p), n, k) for p in range(c["parts"])] for i in range(c["layers"])]
        s.x = [_randn(g, t, k, dtype=TYPES[c["x_type"]]) for _ in s.lins]
        s.y = [[_empty(t, n // 2 if c["glu"] else n, dtype=y) for _ in parts] for parts in s.lins]
        s.q, s.s = _q8(t, k), _empty(t)
    elif c["kind"] == "mlp":
        h, f = c["hidden"], c["n_ff"]
        s.lins = [[s.linear(g, "%s.%d.gate_up" % (s.prefix, i), 2 * f, h), s.linear(g, "%s.%d.down" % (s.prefix, i), h, f)] for i in range(c["layers"])]
        s.x, s.ab = [_randn(g, t, h) * 4 for _ in s.lins], [_randn(g, t, h) for _ in s.lins]
        s.nw = [1 + 0.1 * _randn(g, h) for _ in s.lins]
        s.q, s.s, s.a = _q8(t, h), _empty(t), _empty(t, f, dtype=torch.float16)
        s.y = [_empty(t, h, dtype=torch.float16) for _ in s.lins]
    else:
        v = c["vocab"]
        s.target = torch.randint(0, v, (t,), dtype=torch.int32, device="cuda", generator=g)
        s.target[5::7] = -1  # rows of a padded batch
        s.logp, s.entropy = _empty(t), _empty(t)
        s.top_idx, s.top_logp = _empty(t, c["top"], dtype=torch.int32), _empty(t, c["top"])
        if c["kind"] == "head":
            s.lin = s.linear(g, s.prefix + ".head", v, c["k"])
            s.x, s.logits = _randn(g, t, c["k"], dtype=torch.float16), _empty(t, v)
        else:
            z = _randn(g, t, v) * 2.5
            z[torch.arange(t, device="cuda"), torch.randint(0, v, (t,), device="cuda", generator=g)] += 6.0
            if c["masked"]:
                z[torch.rand(t, v, device="cuda", generator=g) < 0.7] = -math.inf
            s.logits = z.to(TYPES[c["type"]])
    torch.cuda.synchronize()  # the library launches on a stream of its own
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _quantised(x):
    """(q as f32, s): the quotient in 64 bits, where a value next to a border between two steps falls on its side."""
    s = (x.float().abs().amax(1, keepdim=True).double() / 127).float()
    s = torch.where(s < 2.0**-126, torch.zeros_like(s), s)
    q = torch.round(x.double() / torch.where(s == 0, torch.ones_like(s), s).double())
    return torch.where(s == 0, torch.zeros_like(q), q).float(), s


def _product(q, s, lin):
    return (q @ lin.w.float().T) * s * lin.ws


def _silu_mul(g, u):
    return g / (1 + torch.exp(-g)) * u


def _gated(y):
    f = y.shape[1] // 2
    return _silu_mul(y[:, :f], y[:, f:])


def _scores(z, target, top):
    z = z.float()
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    logp = z - m - torch.log(total)
    p = e / total
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    at = target.clamp(min=0).long()
    chosen = torch.where(target < 0, torch.zeros_like(m[:, 0]), logp.gather(1, at[:, None])[:, 0])
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    return chosen, entropy, order.to(torch.int32), logp.gather(1, order)


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
    if c["kind"] == "head":
        q, sx = _quantised(s.x)
        # whole sums, in 64 bits: in 32 they lose the digits that order neighbouring alternatives
        logits = (q.double() @ s.lin.w.double().T).float() * sx * s.lin.ws
        return (logits,) + _scores(logits, s.target, c["top"])
    return _scores(s.logits, s.target, c["top"])


# ---------------------------------------------------------------------------------------------- the library's calls
def _run_own(s):
    from llm170_amd import ffi

    c, t, dec = s.case, s.case["t"], s.program.dec
    code = {"f32": ffi.F32, "f16": ffi.F16, "bf16": ffi.BF16}
    if c["kind"] == "linear":
        for x, parts, ys in zip(s.x, s.lins, s.y):
            if c["parts"] > 1:
                dec.quant_rows(x.data_ptr(), s.q.data_ptr(), s.s.data_ptr(), t, c["k"], x_type=code[c["x_type"]])
            for lin, y in zip(parts, ys):
                if c["parts"] > 1:
                    dec.lin_forward_w8a8(lin.name, s.q.data_ptr(), y.data_ptr(), t, x_type=ffi.Q8, xs_dev=s.s.data_ptr(), y_type=code[c["y_type"]])
                elif c["glu"]:
                    dec.lin_forward_w8a8_glu(lin.name, x.data_ptr(), y.data_ptr(), t, x_type=code[c["x_type"]], y_type=code[c["y_type"]])
                else:
                    dec.lin_forward_w8a8(lin.name, x.data_ptr(), y.data_ptr(), t, x_type=code[c["x_type"]], y_type=code[c["y_type"]])
        return s.y
    if c["kind"] == "mlp":
        for x, ab, nw, (gate_up, down), y in zip(s.x, s.ab, s.nw, s.lins, s.y):
            dec.norm_resid_q8(x.data_ptr(), nw.data_ptr(), ab.data_ptr(), s.q.data_ptr(), s.s.data_ptr(), t, c["hidden"])
            dec.lin_forward_w8a8_glu(gate_up.name, s.q.data_ptr(), s.a.data_ptr(), t, x_type=ffi.Q8, xs_dev=s.s.data_ptr(), y_type=ffi.F16)
            dec.lin_forward_w8a8(down.name, s.a.data_ptr(), y.data_ptr(), t, x_type=ffi.F16, y_type=ffi.F16)
        return s.x, s.y
    if c["kind"] == "head":
        dec.lin_forward_w8a8(s.lin.name, s.x.data_ptr(), s.logits.data_ptr(), t, x_type=ffi.F16, y_type=ffi.F32)
    dec.token_logprobs(s.logits.data_ptr(), t, c["vocab"], logits_type=code[c.get("type", "f32")], targets_dev=s.target.data_ptr(),
                       logp_dev=s.logp.data_ptr(), entropy_dev=s.entropy.data_ptr(), top_k=c["top"], top_idx_dev=s.top_idx.data_ptr() if c["top"] else 0,
                       top_logp_dev=s.top_logp.data_ptr() if c["top"] else 0)
    scores = s.logp, s.entropy, s.top_idx, s.top_logp
    return (s.logits,) + scores if c["kind"] == "head" else scores


def run(s):
    return _run_own(s) if own else _run_plain(s)


def work(case):
    c, t = case, case["t"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "linear":
        n, k, out = c["n"], c["k"], c["n"] // 2 if c["glu"] else c["n"]
        return {"bytes": c["layers"] * (t * k * size[c["x_type"]] + c["parts"] * (n * k + 4 * n + t * out * size[c["y_type"]])),
                "flops": 2.0 * c["layers"] * c["parts"] * t * n * k}
    if c["kind"] == "mlp":
        h, f = c["hidden"], c["n_ff"]
        return {"bytes": c["layers"] * (3 * f * h + 4 * (2 * f + 2 * h) + t * h * (3 * 4 + 2)), "flops": 2.0 * c["layers"] * t * 3 * f * h}
    out = t * (4 + 4 + 4 + 8 * c["top"])
    if c["kind"] == "head":
        v, k = c["vocab"], c["k"]
        return {"bytes": v * k + 4 * v + 2 * t * k + 4 * t * v + out, "flops": 2.0 * t * v * k}
    return {"bytes": t * c["vocab"] * size[c["type"]] + out, "flops": 6.0 * t * c["vocab"]}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case

    def steps(x):  # rows of 64-bit values -> whole steps and their size, an f32 number
        size = torch.div(torch.linalg.vector_norm(x, float("inf"), dim=1), 127.0).to(torch.float32).double()[:, None]
        size[size < 2.0**-126] = 0.0
        return torch.nan_to_num(x / size, nan=0.0).round(), size

    def through(x, lin):
        q, size = steps(x)
        return torch.mm(q, lin.w.to(torch.float64).t()).mul(size).mul(lin.ws.to(torch.float64)[None, :])

    def gate(y):
        a, b = y.chunk(2, dim=1)
        return a * torch.special.expit(a) * b

    def scores(z):
        z = z.to(torch.float64)
        lse = torch.special.logsumexp if hasattr(torch.special, "logsumexp") else torch.logsumexp
        lp = z - lse(z, 1)[:, None]
        entropy = torch.special.entr(torch.exp(lp)).sum(1)
        chosen = lp[torch.arange(len(z), device=z.device), s.target.long() % z.shape[1]].masked_fill(s.target < 0, 0.0)
        best = torch.topk(lp, c["top"], dim=1).values
        return chosen, entropy, None, best

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
    if c["kind"] == "head":
        logits = through(s.x.to(torch.float64), s.lin)
        return (logits,) + scores(logits)
    return scores(s.logits)
