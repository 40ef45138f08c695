"""A layer's norm and its serving in 8 bits, each operator in its plain form and as the framework's call.

Kinds of case
  norm    norm of whole rows, mean and spread, with weight and bias (back 0 / 1: the gradients of rows, weight and bias)
  int8    a product with a weight held in 8-bit integers, a scale for each of its columns: the rows of x are brought to 8-bit integers with a
          scale each, then multiplied
  append  new tokens' keys and values written into a cache of 8-bit pages (64 tokens a page, a scale for each page and head), and what the
          pages they reached then hold, read back
  attend  attention over such a cache; with one query a sequence it is a step of decoding, causal 0 is attention to another sequence's states

`run` with own = False computes the formulas with elementary torch operations in 32 bits; with own = True it calls the C ABI
(deep8_amd.capi).  Lengths of sequences follow from the case, values from the seed.
"""
import math
import random

import torch

own = False

TYPES = {"float32": (torch.float32, 4), "float16": (torch.float16, 2)}
EPSILON = 1e-5
PAGE = 64            # tokens of a page
SMALLEST = 2.0 ** -100  # the least scale


def listed():
    return [
        # decoding, 8 sequences a step: bound by the launch
        {"name": "norm_decode_f16", "kind": "norm", "dtype": "float16", "back": 0, "rows": 8, "cols": 4096},
        # training, forward and back
        {"name": "norm_train_f16", "kind": "norm", "dtype": "float16", "back": 0, "rows": 16384, "cols": 4096},
        {"name": "norm_grad_f16", "kind": "norm", "dtype": "float16", "back": 1, "rows": 8192, "cols": 4096},
        # the same in single precision, an odd number of rows that are no power of two
        {"name": "norm_grad_odd_f32", "kind": "norm", "dtype": "float32", "back": 1, "rows": 4099, "cols": 1000},
        # decoding: a few rows against the whole weight
        {"name": "int8_decode_f16", "kind": "int8", "dtype": "float16", "rows": 4, "inner": 4096, "cols": 8192},
        # a whole prompt
        {"name": "int8_prompt_f16", "kind": "int8", "dtype": "float16", "rows": 8192, "inner": 4096, "cols": 8192},
        # single precision, odd sizes
        {"name": "int8_odd_f32", "kind": "int8", "dtype": "float32", "rows": 777, "inner": 1000, "cols": 1351},
        # prompts of different lengths written to fresh pages
        {"name": "append_prompt_f16", "kind": "append", "dtype": "float16", "sequences": 3, "new": 8192, "old": 0, "kv_heads": 8, "dim": 128, "lengths": 1},
        # a few tokens for each of 16 sequences, onto pages that hold some already, heads that are no power of two
        {"name": "append_few_f32", "kind": "append", "dtype": "float32", "sequences": 16, "new": 40, "old": 5000, "kv_heads": 4, "dim": 80, "lengths": 2},
        # one new token for each of 16 sequences of several thousand tokens
        {"name": "attend_decode_f16", "kind": "attend", "dtype": "float16", "sequences": 16, "queries": 16, "keys": 131072, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": 1, "lengths": 3},
        # the next part of four prompts
        {"name": "attend_chunk_f16", "kind": "attend", "dtype": "float16", "sequences": 4, "queries": 512, "keys": 32768, "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": 1, "lengths": 4},
        # single precision, odd lengths, a head that is no power of two
        {"name": "attend_odd_f32", "kind": "attend", "dtype": "float32", "sequences": 5, "queries": 83, "keys": 9001, "heads": 6, "kv_heads": 2, "dim": 80,
         "causal": 1, "lengths": 5},
    ]


# ---- more cases of the same ranges ----------------------------------------------------------------------------------
MOST_BYTES = {"norm": 2.8e8, "int8": 2e8, "append": 1.7e8, "attend": 2.8e8}
MOST_FLOPS = {"float16": 5.5e11, "float32": 2.5e10}
MOST_PAIRS = 1.2e9  # entries of the padded score matrices, all heads


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi, grain):
    """a size between lo and hi: mostly multiples of `grain`, some of 8, a few anything"""
    n, r = _log(rng, lo, hi), rng.random()
    g = grain if r < 0.6 else 8 if r < 0.85 else 1
    return max(n // g * g, g if g <= hi else 1, 1)


def _draw_once(rng):
    kind = rng.choice(["norm", "int8", "int8", "append", "attend", "attend"])
    dtype = rng.choice(["float16", "float16", "float32"])
    if kind == "norm":
        return {"kind": kind, "dtype": dtype, "back": int(rng.random() < 0.5), "rows": _size(rng, 1, 16384, 64), "cols": _size(rng, 64, 8192, 64)}
    if kind == "int8":
        rows = _log(rng, 1, 64) if rng.random() < 0.4 else _size(rng, 64, 8192, 64)
        return {"kind": kind, "dtype": dtype, "rows": rows, "inner": _size(rng, 64, 4096, 64), "cols": _size(rng, 64, 8192, 64)}
    n, dim, lengths = _log(rng, 1, 16), rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128]), rng.randint(10, 1 << 20)
    if kind == "append":
        new = n if rng.random() < 0.3 else n * _log(rng, 1, 64) if rng.random() < 0.4 else max(n, _log(rng, 64, 8192))
        old = 0 if rng.random() < 0.3 else _log(rng, n, 32768)
        return {"kind": kind, "dtype": dtype, "sequences": n, "new": new, "old": old, "kv_heads": rng.choice([1, 2, 3, 4, 8]), "dim": dim, "lengths": lengths}
    kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 3, 4, 5, 8])
    form = rng.choice(["decode", "decode", "chunk", "cross"])
    queries = n if form == "decode" else n * _log(rng, 1, 128)
    keys = _size(rng, PAGE * n, 131072, 64) if form != "chunk" else queries + _log(rng, 64, 32768)
    return {"kind": kind, "dtype": dtype, "sequences": n, "queries": queries, "keys": keys, "heads": kv * group, "kv_heads": kv, "dim": dim,
            "causal": int(form != "cross"), "lengths": lengths}


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] > MOST_BYTES[case["kind"]] or w["flops"] > MOST_FLOPS[case["dtype"]]:
            continue
        if case["kind"] == "attend":
            q, k = _lengths(case)
            if case["sequences"] * case["heads"] * max(q) * max(k) > MOST_PAIRS or case["sequences"] * max(k) * case["kv_heads"] > 4e6:
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
    """tokens that a call brings, and tokens that the cache then holds, of each sequence"""
    n, rng = case["sequences"], random.Random(case["lengths"])
    if case["kind"] == "append":
        new = [1] * n if case["new"] == n else _parts(case["new"], n, rng)
        return new, [a + b for a, b in zip(new, _parts(case["old"], n, rng))]
    q = [1] * n if case["queries"] == n else _parts(case["queries"], n, rng)
    if not case["causal"] or case["queries"] == n:
        return q, _parts(case["keys"], n, rng)
    return q, [a + b for a, b in zip(q, _parts(case["keys"] - case["queries"], n, rng))]


def _back(case):
    """append: tokens that are read back of each sequence, from the first page that was written to"""
    return [have - (have - new) // PAGE * PAGE if new else 0 for new, have in zip(*_lengths(case))]


def _visible(case):
    """pairs of a query and a key that it sees, of one head: causal, query t sees the first t + 1 + k - q keys"""
    if not case["causal"]:
        return sum(q * k for q, k in zip(*_lengths(case)))
    few = [(q, k, max(0, q - k)) for q, k in zip(*_lengths(case))]
    return sum((q - e) * (k - q) + (q * (q + 1) - e * (e + 1)) // 2 for q, k, e in few)


def work(case):
    es = TYPES[case["dtype"]][1]
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": es * (n * (3 if case["back"] else 2) + (3 if case["back"] else 2) * case["cols"]), "flops": n * (16 if case["back"] else 8)}
    if case["kind"] == "int8":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        return {"bytes": es * (rows * inner + rows * cols) + inner * cols + 4 * cols, "flops": 2 * rows * inner * cols}
    width = case["kv_heads"] * case["dim"]
    if case["kind"] == "append":
        new, back = case["new"], sum(_back(case))
        # new rows read, tokens that the pages held already read, the pages' tokens written in 8 bits, and once more as values
        return {"bytes": 2 * width * (es * new + (back - new) + back + es * back), "flops": 4 * width * back}
    q = case["queries"] * case["heads"] * case["dim"]
    pages = sum(-(-k // PAGE) for k in _lengths(case)[1])
    return {"bytes": 2 * es * q + 2 * case["keys"] * width + 8 * pages * case["kv_heads"] + 4 * case["queries"] * case["heads"],
            "flops": 4 * _visible(case) * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(rng, kind, *shape, scale=1.0):
    return (torch.randn(shape, generator=rng, device="cuda") * scale).to(kind)


def _starts(lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")


def _pages_of(lengths, rng):
    """a page table with pages in no order, -1 where a sequence has none, and the number of pages"""
    need = [-(-n // PAGE) for n in lengths]
    order, width = torch.randperm(sum(need), generator=rng, device="cuda").int().tolist(), max(need) + 1
    at = [sum(need[:i]) for i in range(len(need))]
    return torch.tensor([order[a : a + n] + [-1] * (width - n) for a, n in zip(at, need)], dtype=torch.int32, device="cuda"), sum(need)


def _up(n, to):
    return -(-n // to) * to


def _cache(case, s, rng):
    """pages of tokens that are there already: heads of different sizes, each page's scale what its largest value asks for"""
    G, D, pitch = case["kv_heads"], case["dim"], _up(case["dim"], 16)
    new, have = _lengths(case)
    s["table"], pages = _pages_of(have, rng)
    size = torch.exp2(torch.randint(-2, 3, (G, 1, 1), generator=rng, device="cuda").float())
    for name in ("k", "v"):
        x = torch.randn((pages, G, PAGE, D), generator=rng, device="cuda") * size
        scale = _scale_of(x.abs().amax((2, 3)))
        codes = torch.zeros((pages, G, PAGE, pitch), dtype=torch.int8, device="cuda")
        codes[..., :D] = torch.round(x / scale[..., None, None]).to(torch.int8)
        s[name + "_codes"] = codes if name == "k" else codes.transpose(2, 3).contiguous()
        s[name + "_scales"] = scale
    s["starts"], s["lengths"] = _starts(new), torch.tensor(have, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    rng, kind = torch.Generator(device="cuda").manual_seed(seed), TYPES[case["dtype"]][0]
    s = {"case": case}
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = (_normal(rng, torch.float32, rows, cols, scale=2.0) + _normal(rng, torch.float32, rows, 1)).to(kind)
        s["w"], s["b"] = (1 + _normal(rng, torch.float32, cols, scale=0.2)).to(kind), _normal(rng, kind, cols, scale=0.2)
        if case["back"]:
            s["dy"] = _normal(rng, kind, rows, cols)
    elif case["kind"] == "int8":
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        # some columns of what a layer passes on are several times the others
        wide = 1 + 7 * (torch.rand(inner, generator=rng, device="cuda") < 0.01)
        s["x"] = (_normal(rng, torch.float32, rows, inner) * wide).to(kind)
        w = _normal(rng, torch.float32, cols, inner, scale=inner ** -0.5)
        s["w_scales"] = w.abs().amax(1) / 127
        s["w"] = torch.zeros((cols, _up(inner, 128)), dtype=torch.int8, device="cuda")  # the framework's layout: a column's codes in a row, zeros behind
        s["w"][:, :inner] = torch.round(w / s["w_scales"][:, None]).to(torch.int8)
    else:
        _cache(case, s, rng)
        G, D = case["kv_heads"], case["dim"]
        if case["kind"] == "append":
            s["k"], s["v"] = _normal(rng, kind, case["new"], G, D), _normal(rng, kind, case["new"], G, D, scale=0.5)
            s["back"] = _starts(_back(case))
            # the pages that the call reaches, and how many tokens each holds before it: a program that keeps the lengths knows them
            spans = [(i, n - b, n - m) for i, (m, n, b) in enumerate(zip(*_lengths(case), _back(case))) if m]
            reached = [(i, p, old - p) for i, first, old in spans for p in range(first, _lengths(case)[1][i], PAGE)]
            s["reached"] = torch.stack([s["table"][i, p // PAGE] for i, p, _ in reached]).long()
            s["held"] = torch.tensor([max(0, n) for _, _, n in reached], device="cuda")
        else:
            s["q"] = _normal(rng, kind, case["queries"], case["heads"], D)
            s["longest"] = tuple(max(n) for n in _lengths(case))
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _norm(s):
    x = s["x"].float()
    x = x - x.mean(1, keepdim=True)
    return (x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPSILON) * s["w"].float() + s["b"].float()).to(s["x"].dtype)


def _norm_grad(s):
    x, g, kind = s["x"].float(), s["dy"].float(), s["x"].dtype
    x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt(x.square().mean(1, keepdim=True) + EPSILON)
    x = x * r
    wg = g * s["w"].float()
    dx = r * (wg - wg.mean(1, keepdim=True) - x * (wg * x).mean(1, keepdim=True))
    return {"dx": dx.to(kind), "dw": (g * x).sum(0).to(kind), "db": g.sum(0).to(kind)}


def _int8(s):
    x = s["x"].float()
    scale = (x.abs().amax(1, keepdim=True) / 127).clamp(min=SMALLEST)
    codes = torch.round(x.double() / scale.double()).float()  # in 64 bits: quotients next to a half
    z = torch.matmul(codes, s["w"][:, : x.shape[1]].float().t())
    return (z * (scale * s["w_scales"])).to(s["x"].dtype)


def _scale_of(largest):
    """the least power of two of which 127 reach `largest`"""
    m, e = torch.frexp(largest)
    return torch.exp2((e - 7 + (m > 127 / 128).int()).clamp(min=-100).float())


def _token_of(starts, lengths, rows):
    """sequence and place in it of each row of a call: the last rows of what the cache holds"""
    i = torch.arange(rows, device="cuda")
    which = torch.searchsorted(starts[1:].long(), i, right=True)
    return which, lengths[which].long() - starts[which + 1].long() + i


def _append(s):
    c, D, pages, held = s["case"], s["case"]["dim"], s["reached"], s["held"]
    which, place = _token_of(s["starts"], s["lengths"], c["new"])
    page, slot = s["table"][which, place // PAGE].long(), place % PAGE
    keep = (torch.arange(PAGE, device="cuda") < held[:, None])[:, None, :, None]
    for name in ("k", "v"):
        x, scales = s[name].float(), s[name + "_scales"]
        codes = s[name + "_codes"] if name == "k" else s[name + "_codes"].transpose(2, 3)
        largest = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, scales.shape[1]), x.abs().amax(2), "amax")[pages]
        before = torch.where((held > 0)[:, None], scales[pages], 0.0)
        scale = torch.maximum(before, _scale_of(largest))
        old = codes[pages]
        codes[pages] = torch.where(keep, torch.round(old.float() * (before / scale)[..., None, None]).to(torch.int8), old)
        scales[pages] = scale
        codes[page, :, slot, :D] = torch.round(x / scales[page][..., None]).to(torch.int8)
    which, place = _token_of(s["back"], s["lengths"], sum(_back(c)))
    page, slot = s["table"][which, place // PAGE].long(), place % PAGE
    k = s["k_codes"][page, :, slot, :D].float() * s["k_scales"][page][..., None]
    v = s["v_codes"][page, :, :D, slot].float() * s["v_scales"][page][..., None]
    return {"k": k.to(s["k"].dtype), "v": v.to(s["v"].dtype), "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def _attend(s):
    c, (lq, lk) = s["case"], s["longest"]
    G, g, D, n = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["sequences"]
    pages = s["table"][:, : -(-lk // PAGE)].long().clamp(min=0)
    P = pages.shape[1]
    k = (s["k_codes"][pages][..., :D].float() * s["k_scales"][pages][..., None, None]).transpose(1, 2).reshape(n, G, P * PAGE, D)
    v = (s["v_codes"][pages][..., :D, :].float() * s["v_scales"][pages][..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, G, P * PAGE, D)
    t, j = torch.arange(lq, device="cuda")[:, None], torch.arange(P * PAGE, device="cuda")
    begin, have_q, have_k = s["starts"][:-1, None].long(), s["starts"].diff()[:, None, None], s["lengths"][:, None, None]
    at = (begin + torch.arange(lq, device="cuda")).clamp(max=c["queries"] - 1)
    q = s["q"][at].float().view(n, lq, G, g, D).permute(0, 2, 3, 1, 4).reshape(n, G, g * lq, D).contiguous()
    seen = (j < have_k) & (t < have_q)
    if c["causal"]:
        seen = seen & (j <= t + have_k - have_q)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).view(n, G, g, lq, P * PAGE).masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + total.log(), -math.inf)[..., 0].permute(0, 3, 1, 2).reshape(n, lq, G * g)
    p = p.div_(torch.where(total > 0, total, 1.0)).view(n, G, g * lq, P * PAGE)
    o = torch.matmul(p, v).view(n, G, g, lq, D).permute(0, 3, 1, 2, 4).reshape(n, lq, G * g, D)
    which = torch.searchsorted(s["starts"][1:].long(), torch.arange(c["queries"], device="cuda"), right=True)
    place = torch.arange(c["queries"], device="cuda") - s["starts"][which].long()
    return {"o": o[which, place].to(s["q"].dtype), "lse": lse[which, place].t().contiguous()}


# ---- the framework's calls ------------------------------------------------------------------------------------------
class _Calls:
    """what a program lays out once for its tensors: outputs, scratch, the calls with their arguments"""

    def __init__(self, s):
        from deep8_amd import capi
        self.capi, self.lib, c = capi, capi.init(), s["case"]
        self.dt = {"float32": capi.FLOAT32, "float16": capi.FLOAT16}[c["dtype"]]
        self.calls = []
        getattr(self, "_" + c["kind"] + ("_grad" if c.get("back") else ""))(s, c)

    def _call(self, name, *args, need=None):
        """tensors stand for their addresses; the element type, the scratch block if there is one and the (default) stream are added"""
        if need is not None:
            self.scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            args += (self.scratch, need)
        fn = getattr(self.lib, name)
        self.calls.append((fn, tuple(k(a.data_ptr() if isinstance(a, torch.Tensor) else a) for k, a in zip(fn.argtypes, (self.dt,) + args + (None,), strict=True))))

    def _norm(self, s, c):
        self.out = torch.empty_like(s["x"])
        self._call("d8_layer_norm", s["x"], c["cols"], s["w"], s["b"], self.out, c["cols"], c["rows"], c["cols"], EPSILON)

    def _norm_grad(self, s, c):
        rows, cols = c["rows"], c["cols"]
        self.out = {"dx": torch.empty_like(s["x"]), "dw": torch.empty_like(s["w"]), "db": torch.empty_like(s["b"])}
        need = self.lib.d8_layer_norm_grad_scratch_bytes(self.dt, rows, cols)
        self._call("d8_layer_norm_grad", s["x"], cols, s["w"], s["dy"], cols, self.out["dx"], cols, self.out["dw"], self.out["db"], rows, cols, EPSILON, 3, need=need)

    def _int8(self, s, c):
        rows, inner, cols = c["rows"], c["inner"], c["cols"]
        self.out = torch.empty((rows, cols), dtype=s["x"].dtype, device="cuda")
        self.codes = torch.empty((rows, self.lib.d8_int8_pitch(inner)), dtype=torch.int8, device="cuda")
        self.scales = torch.empty(rows, device="cuda")
        self._call("d8_quantize_rows", s["x"], inner, rows, inner, self.codes, self.scales)
        self._call("d8_matmul_int8", self.codes, self.scales, rows, inner, s["w"], s["w_scales"], cols, self.out, cols,
                   need=self.lib.d8_matmul_int8_scratch_bytes(rows, inner, cols))

    def _where(self, s, c, starts, rows):
        return starts, s["lengths"], s["table"], c["sequences"], rows, s["table"].shape[1], s["k_scales"].shape[0]

    def _pages(self, s):
        return s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]

    def _append(self, s, c):
        G, D, row, back = c["kv_heads"], c["dim"], c["kv_heads"] * c["dim"], sum(_back(c))
        k, v = (torch.empty((back, G, D), dtype=s["k"].dtype, device="cuda") for _ in range(2))
        self._call("d8_cache_append", s["k"], row, s["v"], row, *self._pages(s), *self._where(s, c, s["starts"], c["new"]), G, D)
        self._call("d8_cache_read", k, row, v, row, *self._pages(s), *self._where(s, c, s["back"], back), G, D)
        self.out = {"k": k, "v": v, "k_scales": s["k_scales"], "v_scales": s["v_scales"]}

    def _attend(self, s, c):
        H, G, D, n = c["heads"], c["kv_heads"], c["dim"], c["queries"]
        self.out = {"o": torch.empty_like(s["q"]), "lse": torch.empty((H, n), device="cuda")}
        need = self.lib.d8_attention_cache_scratch_bytes(self.dt, c["sequences"], n, s["table"].shape[1], H, G, D)
        self._call("d8_attention_cache", s["q"], H * D, *self._pages(s), self.out["o"], H * D, self.out["lse"], *self._where(s, c, s["starts"], n), H, G, D,
                   D ** -0.5, c["causal"], need=need)


PLAIN = {"norm": (_norm, _norm_grad), "int8": (_int8,), "append": (_append,), "attend": (_attend,)}


def run(state):
    if not own:
        return PLAIN[state["case"]["kind"]][state["case"].get("back", 0)](state)
    calls = state.get("calls")
    if calls is None:
        calls = state["calls"] = _Calls(state)
    for fn, args in calls.calls:
        rc = fn(*args)
        if rc:
            calls.capi.check(rc)
    return calls.out


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_norm(s, c):
    x, w, b = (s[n].double().requires_grad_() for n in ("x", "w", "b"))
    y = torch.nn.functional.layer_norm(x, (c["cols"],), w, b, EPSILON)
    if not c["back"]:
        return y.detach()
    y.backward(s["dy"].double())
    return {"dx": x.grad, "dw": w.grad, "db": b.grad}


def _exact_int8(s, c):
    # scales are numbers of 32 bits by definition, codes the whole numbers nearest to the exact quotients
    step = torch.clamp((s["x"].double().abs().max(dim=1, keepdim=True).values / 127).float().double(), min=SMALLEST)
    codes = torch.round(s["x"].double() / step)
    w = s["w"][:, : c["inner"]].double().t().contiguous() * s["w_scales"].double()
    return (codes @ w) * step


def _exact_append(s, c):
    """sequence by sequence and page by page"""
    out = {"k": [], "v": []}
    for name in ("k", "v"):
        scales = s[name + "_scales"].double().clone()
        first, rows = 0, s[name].double()
        for i, (new, have, back) in enumerate(zip(*_lengths(c), _back(c))):
            page_at = have - back
            while page_at < have and new:
                page, end = int(s["table"][i, page_at // PAGE]), min(page_at + PAGE, have)
                held = max(0, have - new - page_at)
                fresh = rows[first + page_at + held - (have - new) : first + end - (have - new)]
                old = s[name + "_codes"][page]
                old = (old if name == "k" else old.transpose(1, 2))[:, :held, : c["dim"]].double()
                need = torch.exp2(torch.ceil(torch.log2(fresh.abs().amax((0, 2)) / 127)).clamp(min=-100))
                need = torch.where(fresh.abs().amax((0, 2)) > 127 * need, 2 * need, need)
                if held:
                    need = torch.maximum(need, scales[page])
                    old = torch.round(old * (scales[page] / need)[:, None, None])
                scales[page] = need
                fresh = torch.round(fresh / need[:, None])
                out[name].append(torch.cat([old.transpose(0, 1), fresh]) * need[:, None])
                page_at = end
            first += new
        out[name + "_scales"] = scales
    return {**out, "k": torch.cat(out["k"]), "v": torch.cat(out["v"])}


def _exact_attend(s, c):
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    o, lse = torch.zeros(c["queries"], H, D, dtype=torch.float64, device="cuda"), torch.full((H, c["queries"]), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for i, (nq, nk) in enumerate(zip(*_lengths(c))):
        rows = slice(first, first + nq)
        first += nq
        if not nq or not nk:
            continue
        pages = s["table"][i, : -(-nk // PAGE)].long()
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1) if c["causal"] else None
        for h in range(G):
            k = (s["k_codes"][pages, h, :, :D].double() * s["k_scales"][pages, h].double()[:, None, None]).flatten(0, 1)[:nk]
            v = (s["v_codes"][pages, h, :D].double() * s["v_scales"][pages, h].double()[:, None, None]).transpose(1, 2).flatten(0, 1)[:nk]
            for e in range(h * H // G, (h + 1) * H // G):
                t = (s["q"][rows, e].double() @ k.t().contiguous()) / math.sqrt(D)
                if hidden is not None:
                    t[hidden] = -math.inf
                z = torch.logsumexp(t, -1, keepdim=True)
                o[rows, e], lse[e, rows] = torch.nan_to_num(torch.exp(t - z), nan=0.0) @ v, z[:, 0]
    return {"o": o, "lse": lse}


def exact(case, seed):
    return {"norm": _exact_norm, "int8": _exact_int8, "append": _exact_append, "attend": _exact_attend}[case["kind"]](prepare(case, seed), case)
