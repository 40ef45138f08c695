"""The operators of a transformer layer, each in its plain form and as the framework's call.

Kinds of case
  rotary     norm of each query and key head and its rotation by the position, both tensors at once (back 0 / 1)
  attention  attention over packed sequences of different lengths, heads that share keys and values (back 0 / 1); with one query a
             sequence it is a step of decoding over the keys and values of what came before
  gated      a gated feed-forward product: both projections, the activation and their product (back 0 / 1; keep 1 is training,
             where the projections are kept for the way back)

`run` with own = False computes the formulas with elementary torch operations in 32 bits; with own = True it calls the C ABI
(deep8_amd.capi).  Lengths of sequences follow from the case, values from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"float32": (torch.float32, 4), "float16": (torch.float16, 2)}
EPSILON = 1e-6


def listed():
    return [
        # decoding, 8 sequences a step: bound by the launch
        {"name": "rotary_decode_f16", "kind": "rotary", "dtype": "float16", "back": 0, "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": 0},
        # a whole prompt
        {"name": "rotary_prompt_f16", "kind": "rotary", "dtype": "float16", "back": 0, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": 0},
        # training in single precision: neighbouring pairs, part of the head, an odd number of tokens
        {"name": "rotary_grad_f32", "kind": "rotary", "dtype": "float32", "back": 1, "tokens": 4099, "heads": 12, "kv_heads": 4, "dim": 96,
         "rotary": 64, "interleaved": 1},
        # one new token for each of 16 sequences of several thousand tokens
        {"name": "attention_decode_f16", "kind": "attention", "dtype": "float16", "back": 0, "sequences": 16, "queries": 16, "keys": 131072,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": 1, "lengths": 1},
        # prompts of different lengths, packed
        {"name": "attention_prompt_f16", "kind": "attention", "dtype": "float16", "back": 0, "sequences": 3, "queries": 16384, "keys": 16384,
         "heads": 16, "kv_heads": 4, "dim": 128, "causal": 1, "lengths": 2},
        # the same in single precision, with a head that is no power of two and odd lengths
        {"name": "attention_odd_f32", "kind": "attention", "dtype": "float32", "back": 0, "sequences": 5, "queries": 2501, "keys": 2501,
         "heads": 6, "kv_heads": 2, "dim": 80, "causal": 1, "lengths": 3},
        # training on packed sequences
        {"name": "attention_grad_f16", "kind": "attention", "dtype": "float16", "back": 1, "sequences": 3, "queries": 6144, "keys": 6144,
         "heads": 16, "kv_heads": 4, "dim": 128, "causal": 1, "lengths": 4},
        # training an encoder: every position sees every other
        {"name": "attention_grad_f32", "kind": "attention", "dtype": "float32", "back": 1, "sequences": 4, "queries": 2048, "keys": 2048,
         "heads": 8, "kv_heads": 8, "dim": 64, "causal": 0, "lengths": 5},
        # decoding: a few rows against the whole weight
        {"name": "gated_decode_f16", "kind": "gated", "dtype": "float16", "back": 0, "rows": 4, "inner": 4096, "cols": 8192, "act": "silu", "keep": 0},
        # training at an ordinary size, forward and back
        {"name": "gated_train_f16", "kind": "gated", "dtype": "float16", "back": 0, "rows": 8192, "inner": 4096, "cols": 8192, "act": "silu", "keep": 1},
        {"name": "gated_grad_f16", "kind": "gated", "dtype": "float16", "back": 1, "rows": 4096, "inner": 2048, "cols": 5632, "act": "silu", "keep": 1},
        # single precision, odd sizes
        {"name": "gated_odd_f32", "kind": "gated", "dtype": "float32", "back": 0, "rows": 777, "inner": 1000, "cols": 1351, "act": "gelu", "keep": 1},
    ]


# ---- more cases of the same ranges ----------------------------------------------------------------------------------
MOST_BYTES = 6e8
MOST_FLOPS = {"float16": {0: 1.1e12, 1: 4e11}, "float32": {0: 2.5e10, 1: 2.5e10}}
MOST_PAIRS = {0: 2e9, 1: 1.6e9}  # entries of the padded score matrices, all heads


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, grain):
    """a size between lo and hi: mostly multiples of `grain`, some of 8, a few anything"""
    n, r = _log(rng, lo, hi), rng.random()
    g = grain if r < 0.6 else 8 if r < 0.85 else 1
    return max(n // g * g, g if g <= hi else 1, 1)


def _heads(rng):
    kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 8])
    return {"heads": kv * group, "kv_heads": kv}


def _draw_once(rng):
    kind = rng.choice(["rotary", "attention", "attention", "attention", "gated", "gated"])
    dtype, back = rng.choice(["float16", "float16", "float32"]), int(rng.random() < 0.4)
    if kind == "rotary":
        dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128])
        rotary = dim if rng.random() < 0.7 else 2 * rng.randint(1, dim // 2)
        return {"kind": kind, "dtype": dtype, "back": back, "tokens": _size(rng, 64 if back else 1, 8192, 64), **_heads(rng), "dim": dim, "rotary": rotary,
                "interleaved": int(rng.random() < 0.4)}
    if kind == "attention":
        dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128])
        n = _log(rng, 1, 16)
        form = "train" if back else rng.choice(["prompt", "prompt", "decode", "chunk"])
        if form == "decode":
            queries, keys, causal = n, _size(rng, 64 * n, 131072, 64), 1
        elif form == "chunk":  # part of a prompt, or a few tokens at once, over what is there already
            queries = n * _log(rng, 1, 64)
            keys, causal = queries + _log(rng, 64, 16384), 1
        else:
            queries = keys = max(n, _size(rng, 32, 8192, 64))
            causal = int(rng.random() < 0.75)
        return {"kind": kind, "dtype": dtype, "back": back, "sequences": n, "queries": queries, "keys": keys, **_heads(rng), "dim": dim, "causal": causal,
                "lengths": rng.randint(10, 1 << 20)}
    if not back and rng.random() < 0.4:
        return {"kind": kind, "dtype": dtype, "back": 0, "rows": _log(rng, 1, 64), "inner": _size(rng, 256, 4096, 64), "cols": _size(rng, 256, 8192, 64),
                "act": rng.choice(["silu", "silu", "gelu"]), "keep": 0}
    return {"kind": kind, "dtype": dtype, "back": back, "rows": _size(rng, 64, 8192, 64), "inner": _size(rng, 64, 4096, 64), "cols": _size(rng, 64, 8192, 64),
            "act": rng.choice(["silu", "silu", "gelu"]), "keep": 1}


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] > MOST_BYTES or w["flops"] > MOST_FLOPS[case["dtype"]][case["back"]]:
            continue
        if case["kind"] == "attention":
            q, k = _lengths(case)
            if case["sequences"] * case["heads"] * max(q) * max(k) > MOST_PAIRS[case["back"]] or case["sequences"] * max(k) * case["kv_heads"] > 4e6:
                continue
        return case


# ---- sizes ----------------------------------------------------------------------------------------------------------
def _parts(total, n, rng):
    """`total` as n lengths, the longest some times the shortest"""
    share = [0.25 + rng.random() for _ in range(n)]
    ends = [int(total * sum(share[: i + 1]) / sum(share)) for i in range(n)]
    ends[-1] = total
    return [b - a for a, b in zip([0] + ends, ends)]


def _lengths(case):
    """queries and keys of each sequence"""
    n, rng = case["sequences"], random.Random(case["lengths"])
    if case["queries"] == case["keys"]:
        q = _parts(case["queries"], n, rng)
        return q, q
    if case["queries"] == n:
        return [1] * n, _parts(case["keys"], n, rng)
    q = _parts(case["queries"], n, rng)
    return q, [a + b for a, b in zip(q, _parts(case["keys"] - case["queries"], n, rng))]


def _visible(case):
    """pairs of a query and a key that it sees, of one head: causal, query t sees the first t + 1 + k - q keys"""
    if not case["causal"]:
        return sum(q * k for q, k in zip(*_lengths(case)))
    few = [(q, k, max(0, q - k)) for q, k in zip(*_lengths(case))]
    return sum((q - e) * (k - q) + (q * (q + 1) - e * (e + 1)) // 2 for q, k, e in few)


def work(case):
    es = TYPES[case["dtype"]][1]
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": n * es * (3 if case["back"] else 2), "flops": n * (16 if case["back"] else 8)}
    if case["kind"] == "attention":
        q, kv = case["queries"] * case["heads"] * case["dim"], case["keys"] * case["kv_heads"] * case["dim"]
        pairs = _visible(case) * case["heads"] * case["dim"]
        lse = 4 * case["queries"] * case["heads"]
        if case["back"]:
            return {"bytes": es * (4 * q + 4 * kv) + lse, "flops": 10 * pairs}
        return {"bytes": es * (2 * q + 2 * kv) + lse, "flops": 4 * pairs}
    rows, inner, cols = case["rows"], case["inner"], case["cols"]
    if case["back"]:
        return {"bytes": es * (2 * rows * inner + 4 * inner * cols + 3 * rows * cols), "flops": 8 * rows * inner * cols}
    return {"bytes": es * (rows * inner + 2 * inner * cols + rows * cols * (3 if case["keep"] else 1)), "flops": 4 * rows * inner * cols}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(rng, kind, *shape, scale=1.0):
    return (torch.randn(shape, generator=rng, device="cuda") * scale).to(kind)


def _angles(case, longest):
    """cosines and sines of every position and pair, [positions][rotary / 2][2]"""
    half = case["rotary"] // 2
    rate = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(longest, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def prepare(case, seed):
    rng, kind = torch.Generator(device="cuda").manual_seed(seed), TYPES[case["dtype"]][0]
    s = {"case": case}
    if case["kind"] == "rotary":
        T, H, G, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        longest = 16384
        s["q"], s["k"] = _normal(rng, kind, T, H, D, scale=3.0), _normal(rng, kind, T, G, D, scale=3.0)
        s["wq"], s["wk"] = (1 + _normal(rng, torch.float32, 2, D, scale=0.2)).to(kind).unbind(0)
        s["positions"] = torch.randint(longest, (T,), generator=rng, device="cuda", dtype=torch.int32)
        s["table"] = _angles(case, longest)
        if case["back"]:
            s["dq"], s["dk"] = _normal(rng, kind, T, H, D), _normal(rng, kind, T, G, D)
        return s
    if case["kind"] == "attention":
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        s["q"], s["k"], s["v"] = _normal(rng, kind, case["queries"], H, D), _normal(rng, kind, case["keys"], G, D), _normal(rng, kind, case["keys"], G, D)
        q, k = _lengths(case)
        s["longest"] = max(q), max(k)
        s["q_starts"], s["k_starts"] = (torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device="cuda") for n in (q, k))
        if case["back"]:  # what the forward pass left
            s["o"], s["lse"] = _attention(s)
            s["do"] = _normal(rng, kind, case["queries"], H, D)
        return s
    rows, inner, cols = case["rows"], case["inner"], case["cols"]
    s["x"], s["w"] = _normal(rng, kind, rows, inner), _normal(rng, kind, inner, 2 * cols, scale=inner ** -0.5)
    if case["back"]:
        s["pre"] = (s["x"].float() @ s["w"].float()).to(kind)
        s["dh"] = _normal(rng, kind, rows, cols)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _turn(x, table, positions, rotary, interleaved, back):
    """the first `rotary` elements of each head turned by the angles of its token's position (the other way: back)"""
    c, n = table[positions.long()].unbind(-1)
    c, n = c[:, None], -n[:, None] if back else n[:, None]
    part, rest = x[..., :rotary], x[..., rotary:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    a, b = a * c - b * n, a * n + b * c
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), rest], -1)


def _rotary(s):
    c = s["case"]
    return {name: _turn(_unit(s[name].float()) * s["w" + name].float(), s["table"], s["positions"], c["rotary"], c["interleaved"], False).to(s[name].dtype)
            for name in ("q", "k")}


def _unit(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON)


def _rotary_grad_of(s, x, w, dy):
    c, kind = s["case"], x.dtype
    x, w = x.float(), w.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON)
    g = _turn(dy.float(), s["table"], s["positions"], c["rotary"], c["interleaved"], True)
    unit = x * r
    return (r * (w * g - unit * (w * g * unit).mean(-1, keepdim=True))).to(kind), (g * unit).sum((0, 1)).to(kind)


def _rotary_grad(s):
    dq, dwq = _rotary_grad_of(s, s["q"], s["wq"], s["dq"])
    dk, dwk = _rotary_grad_of(s, s["k"], s["wk"], s["dk"])
    return {"dq": dq, "dwq": dwq, "dk": dk, "dwk": dwk}


def _pad(x, starts, longest):
    """packed rows as [sequences][longest] of them, zero where a sequence is shorter"""
    at = torch.arange(longest, device="cuda")
    begin, end = starts[:-1, None].long(), starts[1:, None].long()
    there = begin + at < end
    return x[(begin + at).clamp(max=max(x.shape[0] - 1, 0))].float() * there[..., None, None], there


def _pack(x, starts, rows):
    """[sequences][longest] ... back to packed rows"""
    i = torch.arange(rows, device="cuda")
    which = torch.searchsorted(starts[1:].long(), i, right=True)
    return x[which, i - starts[which].long()]


def _scores(s):
    """queries [n][kv heads][group * longest][dim], keys and values [n][kv heads][longest][dim], probabilities, log sums"""
    c, (lq, lk) = s["case"], s["longest"]
    G, g, D = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    q, k, v = (_pad(s[n], s[b], l)[0] for n, b, l in (("q", "q_starts", lq), ("k", "k_starts", lk), ("v", "k_starts", lk)))
    n = q.shape[0]
    q = q.view(n, lq, G, g, D).permute(0, 2, 3, 1, 4).reshape(n, G, g * lq, D).contiguous()
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    have_q, have_k = s["q_starts"].diff(), s["k_starts"].diff()
    t, j = torch.arange(lq, device="cuda")[:, None], torch.arange(lk, device="cuda")
    seen = (j < have_k[:, None, None]) & (t < have_q[:, None, None])
    if c["causal"]:
        seen = seen & (j <= t + (have_k - have_q)[:, None, None])
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(n, G, g, lq, lk)
    p = p.masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + total.log(), -math.inf)
    p = p.div_(torch.where(total > 0, total, 1.0))
    return q, k, v, p.view(n, G, g * lq, lk), lse[..., 0]


def _attention(s):
    c, (lq, _) = s["case"], s["longest"]
    q, k, v, p, lse = _scores(s)
    n, G, g, D = q.shape[0], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    o = torch.matmul(p, v).view(n, G, g, lq, D).permute(0, 3, 1, 2, 4).reshape(n, lq, G * g, D)
    lse = lse.permute(0, 3, 1, 2).reshape(n, lq, G * g)
    return _pack(o, s["q_starts"], c["queries"]).to(s["q"].dtype), _pack(lse, s["q_starts"], c["queries"]).t().contiguous()


def _attention_grad(s):
    c, (lq, _) = s["case"], s["longest"]
    q, k, v, p, _ = _scores(s)
    kind, n, G, g, D = s["q"].dtype, q.shape[0], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    do = _pad(s["do"], s["q_starts"], lq)[0].view(n, lq, G, g, D).permute(0, 2, 3, 1, 4).reshape(n, G, g * lq, D).contiguous()
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p.mul_(dp.sub_((p * dp).sum(-1, keepdim=True))).mul_(D ** -0.5)
    dq = torch.matmul(ds, k).view(n, G, g, lq, D).permute(0, 3, 1, 2, 4).reshape(n, lq, G * g, D)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    return {"dq": _pack(dq, s["q_starts"], c["queries"]).to(kind), "dk": _pack(dk.transpose(1, 2), s["k_starts"], c["keys"]).to(kind),
            "dv": _pack(dv.transpose(1, 2), s["k_starts"], c["keys"]).to(kind)}


def _activation(a, act):
    return a * torch.sigmoid(a) if act == "silu" else 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))


def _slope(a, act):
    if act == "silu":
        e = torch.sigmoid(a)
        return e * (1 + a * (1 - e))
    return 0.5 * (1 + torch.erf(a * math.sqrt(0.5))) + a * torch.exp(-0.5 * a * a) * (2 * math.pi) ** -0.5


def _gated(s):
    c, kind = s["case"], s["x"].dtype
    pre = torch.matmul(s["x"].float(), s["w"].float())
    gate, up = pre.chunk(2, -1)
    h = (_activation(gate, c["act"]) * up).to(kind)
    return {"h": h, "pre": pre.to(kind)} if c["keep"] else {"h": h}


def _gated_grad(s):
    c, kind = s["case"], s["x"].dtype
    (gate, up), dh = s["pre"].float().chunk(2, -1), s["dh"].float()
    dpre = torch.cat([dh * up * _slope(gate, c["act"]), dh * _activation(gate, c["act"])], -1)
    return {"dx": torch.matmul(dpre, s["w"].float().t()).to(kind), "dw": torch.matmul(s["x"].float().t(), dpre).to(kind)}


# ---- the framework's calls ------------------------------------------------------------------------------------------
class _Calls:
    """what a program lays out once for its tensors: outputs, scratch, the call with its arguments"""

    def __init__(self, s):
        from deep8_amd import capi
        self.capi, self.lib, c = capi, capi.init(), s["case"]
        self.dt = {"float32": capi.FLOAT32, "float16": capi.FLOAT16}[c["dtype"]]
        getattr(self, "_" + c["kind"] + ("_grad" if c["back"] else ""))(s, c)

    def _call(self, name, *args, need=None):
        """tensors stand for their addresses; the element type, the scratch block if there is one and the (default) stream are added"""
        if need is not None:
            self.scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            args += (self.scratch, need)
        self.fn = getattr(self.lib, name)
        kinds = self.fn.argtypes
        self.args = tuple(k(a.data_ptr() if isinstance(a, torch.Tensor) else a) for k, a in zip(kinds, (self.dt,) + args + (None,), strict=True))

    def _rotary(self, s, c):
        out = {"q": torch.empty_like(s["q"]), "k": torch.empty_like(s["k"])}
        H, G, D = c["heads"], c["kv_heads"], c["dim"]
        self._call("d8_head_norm_rotary", s["q"], H * D, H, s["wq"], out["q"], H * D, s["k"], G * D, G, s["wk"], out["k"], G * D, c["tokens"], D, 1, EPSILON,
                   s["positions"], s["table"], s["table"].shape[0], c["rotary"], c["interleaved"])
        self.out = out

    def _rotary_grad(self, s, c):
        out = {"dq": torch.empty_like(s["q"]), "dwq": torch.empty_like(s["wq"]), "dk": torch.empty_like(s["k"]), "dwk": torch.empty_like(s["wk"])}
        T, H, G, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
        need = self.lib.d8_head_norm_rotary_grad_scratch_bytes(self.dt, T, H, G, D)
        self._call("d8_head_norm_rotary_grad", s["q"], H * D, H, s["wq"], s["dq"], H * D, out["dq"], H * D, out["dwq"], s["k"], G * D, G, s["wk"], s["dk"],
                   G * D, out["dk"], G * D, out["dwk"], T, D, 1, EPSILON, s["positions"], s["table"], s["table"].shape[0], c["rotary"], c["interleaved"], 3,
                   need=need)
        self.out = out

    def _sizes(self, c):
        return c["sequences"], c["queries"], c["keys"], c["heads"], c["kv_heads"], c["dim"]

    def _attention(self, s, c):
        H, G, D = c["heads"], c["kv_heads"], c["dim"]
        o, lse = torch.empty_like(s["q"]), torch.empty(H, c["queries"], device="cuda")
        need = self.lib.d8_attention_scratch_bytes(self.dt, 0, *self._sizes(c), c["causal"])
        self._call("d8_attention", s["q"], H * D, s["k"], G * D, s["v"], G * D, o, H * D, lse, s["q_starts"], s["k_starts"], *self._sizes(c), D ** -0.5,
                   c["causal"], need=need)
        self.out = (o, lse)

    def _attention_grad(self, s, c):
        H, G, D = c["heads"], c["kv_heads"], c["dim"]
        out = {"dq": torch.empty_like(s["q"]), "dk": torch.empty_like(s["k"]), "dv": torch.empty_like(s["v"])}
        need = self.lib.d8_attention_scratch_bytes(self.dt, 1, *self._sizes(c), c["causal"])
        self._call("d8_attention_grad", s["q"], H * D, s["k"], G * D, s["v"], G * D, s["o"], H * D, s["lse"], s["do"], H * D, out["dq"], H * D, out["dk"], G * D,
                   out["dv"], G * D, s["q_starts"], s["k_starts"], *self._sizes(c), D ** -0.5, c["causal"], 7, need=need)
        self.out = out

    def _gated(self, s, c):
        rows, inner, cols = c["rows"], c["inner"], c["cols"]
        h = torch.empty(rows, cols, dtype=s["x"].dtype, device="cuda")
        pre = torch.empty(rows, 2 * cols, dtype=s["x"].dtype, device="cuda") if c["keep"] else None
        need = self.lib.d8_matmul_gated_scratch_bytes(self.dt, 0, rows, inner, cols)
        self._call("d8_matmul_gated", s["x"], rows, inner, s["w"], cols, {"silu": 0, "gelu": 1}[c["act"]], pre, h, need=need)
        self.out = {"h": h, "pre": pre} if c["keep"] else {"h": h}

    def _gated_grad(self, s, c):
        rows, inner, cols = c["rows"], c["inner"], c["cols"]
        out = {"dx": torch.empty_like(s["x"]), "dw": torch.empty_like(s["w"])}
        need = self.lib.d8_matmul_gated_scratch_bytes(self.dt, 1, rows, inner, cols)
        self._call("d8_matmul_gated_grad", s["x"], out["dx"], rows, inner, s["w"], out["dw"], cols, {"silu": 0, "gelu": 1}[c["act"]], s["pre"], s["dh"], 3, need=need)
        self.out = out


PLAIN = {"rotary": (_rotary, _rotary_grad), "attention": (_attention, _attention_grad), "gated": (_gated, _gated_grad)}


def run(state):
    if not own:
        return PLAIN[state["case"]["kind"]][state["case"]["back"]](state)
    calls = state.get("calls")
    if calls is None:
        calls = state["calls"] = _Calls(state)
    rc = calls.fn(*calls.args)
    if rc:
        calls.capi.check(rc)
    return calls.out


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_rotary(s, c):
    """token by token and head by head as products of complex numbers: a pair is x + iy, its rotation a factor"""
    R, half = c["rotary"], c["rotary"] // 2
    first = torch.arange(0, R, 2, device="cuda") if c["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if c["interleaved"] else half)
    factor = torch.view_as_complex(s["table"].double())[s["positions"].long()][:, None]

    def turned(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        x = x.clone()
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = {}
    for name in ("q", "k"):
        x, w = s[name].double(), s["w" + name].double()
        length = (x.pow(2).sum(-1, keepdim=True) / c["dim"] + EPSILON).sqrt()
        if not c["back"]:
            out[name] = turned(x / length * w, factor)
            continue
        g = turned(s["d" + name].double(), factor.conj())
        gw = g * w
        out["d" + name] = gw / length - x * (gw * x).sum(-1, keepdim=True) / (c["dim"] * length.pow(3))
        out["dw" + name] = (g * x / length).flatten(0, 1).sum(0)
    return out


def _exact_attention(s, c):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o, lse = torch.zeros_like(q), torch.full((H, c["queries"]), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    qa = ka = 0
    for nq, nk in zip(*_lengths(c)):
        qs, ks = slice(qa, qa + nq), slice(ka, ka + nk)
        qa, ka = qa + nq, ka + nk
        if not nq or not nk:
            continue
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1) if c["causal"] else None
        for h in range(H):
            e = h * G // H
            t = (q[qs, h] @ k[ks, e].t()) / math.sqrt(D)
            if hidden is not None:
                t[hidden] = -math.inf
            z = torch.logsumexp(t, -1, keepdim=True)
            p = torch.nan_to_num(torch.exp(t - z), nan=0.0)
            if not c["back"]:
                o[qs, h], lse[h, qs] = p @ v[ks, e], z[:, 0]
                continue
            g = s["do"][qs, h].double()
            dv[ks, e] += p.t() @ g
            w = g @ v[ks, e].t()
            w = p * (w - (g * (p @ v[ks, e])).sum(-1, keepdim=True)) / math.sqrt(D)
            dq[qs, h] = w @ k[ks, e]
            dk[ks, e] += w.t() @ q[qs, h]
    return {"dq": dq, "dk": dk, "dv": dv} if c["back"] else (o, lse)


def _exact_gated(s, c):
    n, act = c["cols"], {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[c["act"]]
    x, w = s["x"].double(), s["w"].double()
    if not c["back"]:
        a, b = x @ w[:, :n].contiguous(), x @ w[:, n:].contiguous()
        return {"h": act(a) * b, "pre": torch.cat([a, b], 1)} if c["keep"] else {"h": act(a) * b}
    pre = s["pre"].double().requires_grad_()
    (act(pre[:, :n]) * pre[:, n:]).backward(s["dh"].double())
    return {"dx": pre.grad @ w.t().contiguous(), "dw": x.t().contiguous() @ pre.grad}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "gated": _exact_gated}[case["kind"]](s, case)
