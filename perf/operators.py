"""Performance cases of the operators around the head and the draw: the norm in front of them, the
matrix product of draft heads and unquantised heads, and the logits' adjustment before a draw.

`run` computes an operator in its plain form (elementary torch operations in 32 bits) where `own` is
false, and calls the package (`SamplerScratch.add_rms_norm`, `.linear`, `.adjust_logits`) where it is
true. Handles and output buffers are made once, as a decode loop makes them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
ELEMENT = {"f32": 4, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
LEAST_MAX = 2.0 ** -64  # the least largest value that a row's 8-bit scale is taken from
EPS = 1e-6


def listed():
    """The cases of everyday use, an operator at a time, smallest to largest."""
    return [
        # One interactive user, one token: the norm in front of the head. Latency.
        {"name": "norm 1 token", "kind": "norm", "tokens": 1, "hidden": 2048, "dtype": "bf16", "residual": True,
         "out": "bf16"},
        # A full decode batch in front of a projection that takes 8 bits.
        {"name": "norm 64 tokens, 8 bits", "kind": "norm", "tokens": 64, "hidden": 4096, "dtype": "bf16",
         "residual": True, "out": "e4m3"},
        # A ragged prompt kept in f32, of a width that no vector divides.
        {"name": "norm 777 tokens, ragged", "kind": "norm", "tokens": 777, "hidden": 5001, "dtype": "f32",
         "residual": False, "out": "f32"},
        # A long prompt, in front of a projection that takes 8 bits.
        {"name": "norm 16384 tokens, 8 bits", "kind": "norm", "tokens": 16384, "hidden": 4096, "dtype": "bf16",
         "residual": True, "out": "e4m3"},
        # A draft head's block, x + silu(W x + b), for one user's last token. Latency.
        {"name": "draft block 1 token", "kind": "linear", "tokens": 1, "in": 2048, "outs": 2048, "dtype": "bf16",
         "out": "bf16", "act": "silu", "bias": True, "residual": True},
        # The same in 8 bits for a batch of requests.
        {"name": "draft block 24 tokens, 8 bits", "kind": "linear", "tokens": 24, "in": 4096, "outs": 4096,
         "dtype": "e4m3", "out": "bf16", "act": "silu", "bias": True, "residual": True},
        # An unquantised head of an odd vocabulary: the logits that a draw reads.
        {"name": "ragged head 37 tokens", "kind": "linear", "tokens": 37, "in": 2048, "outs": 50257, "dtype": "bf16",
         "out": "f32", "act": "none", "bias": False, "residual": False},
        # A prompt through a projection with everything in its epilogue; the last tile is ragged.
        {"name": "prompt 4099 tokens", "kind": "linear", "tokens": 4099, "in": 4096, "outs": 4096, "dtype": "bf16",
         "out": "bf16", "act": "gelu", "bias": True, "residual": True},
        # A long prompt in 8 bits, widening.
        {"name": "prompt 8192 tokens, 8 bits", "kind": "linear", "tokens": 8192, "in": 4096, "outs": 8192,
         "dtype": "e4m3", "out": "bf16", "act": "none", "bias": False, "residual": False},
        # One request that has to answer in a grammar: few ids are allowed. In place. Latency.
        {"name": "grammar 1 row", "kind": "adjust", "rows": 1, "vocab": 32768, "dtype": "f32", "history": 0, "lists": 0,
         "mask": "tight", "in_place": True, "frequency": False, "shards": 1},
        # A few requests with everything on, of an odd vocabulary.
        {"name": "adjust 4 rows, all lists", "kind": "adjust", "rows": 4, "vocab": 50257, "dtype": "f32", "history": 8192,
         "lists": 64, "mask": "loose", "in_place": False, "frequency": True, "shards": 1},
        # The throughput batch: long contexts, half of the requests under a grammar.
        {"name": "adjust 256 rows", "kind": "adjust", "rows": 256, "vocab": 151936, "dtype": "bf16", "history": 32768,
         "lists": 16, "mask": "mixed", "in_place": False, "frequency": True, "shards": 1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed kinds, over the ranges that serving meets."""
    kind = rng.choice(["norm", "linear", "adjust"])
    if kind == "norm":
        hidden = _log(rng, 512, 8192)
        hidden = hidden if rng.random() < 0.3 else hidden // 64 * 64
        tokens = min(_log(rng, 1, 16384), 16384 * 4096 // hidden)
        dtype = rng.choice(["f32", "bf16", "bf16"])
        return {"kind": kind, "tokens": tokens if dtype == "bf16" else max(1, tokens // 2), "hidden": hidden,
                "dtype": dtype, "residual": rng.random() < 0.7, "out": rng.choice([dtype, "e4m3"])}
    if kind == "linear":
        width = 16 * _log(rng, 32, 512)
        outs = _log(rng, 128, 65536)
        outs = outs if rng.random() < 0.3 else outs // 64 * 64
        tokens = _log(rng, 1, 8192)
        dtype = rng.choice(["bf16", "e4m3"])
        most = 4099 * 4096 * 4096 if dtype == "bf16" else 8192 * 4096 * 8192
        return {"kind": kind, "tokens": max(1, min(tokens, most // (width * outs))), "in": width, "outs": outs,
                "dtype": dtype, "out": "f32" if tokens <= 64 and rng.random() < 0.3 else "bf16",
                "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "bias": rng.random() < 0.5,
                "residual": rng.random() < 0.5}
    vocab = _log(rng, 8192, 262144)
    vocab = vocab if rng.random() < 0.5 else vocab // 128 * 128
    rows = min(_log(rng, 1, 256), 256 * 151936 // vocab)
    dtype = rng.choice(["f32", "bf16"])
    rows = rows if dtype == "bf16" else max(1, rows // 2)
    mask = rng.choice(["none", "tight", "loose", "mixed"])
    in_place = mask != "none" and rng.random() < 0.3
    history = 0 if in_place else rng.choice([0, _log(rng, 16, 32768)])
    lists = 0 if in_place else rng.choice([0, rng.randint(1, 128)])
    if mask == "none" and not history and not lists:  # a call with nothing to do is no case
        history = _log(rng, 16, 32768)
    return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "history": history, "lists": lists, "mask": mask,
            "in_place": in_place, "frequency": rng.random() < 0.5, "shards": rng.choice([1, 1, 2, 8])}


# ------------------------------------------------------------------ inputs --


class _Inputs:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device="cuda")

    def ids(self, high, *shape):
        return torch.randint(0, high, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def skewed_ids(self, high, *shape):
        """Token ids as text has them: few are frequent (a power law of exponent 1.3)."""
        u = torch.rand(shape, generator=self.g, device="cuda", dtype=torch.float64).clamp_min(1e-12)
        return (u.pow(-1.0 / 0.3).clamp_max(1e15).long() % high).int()

    def distinct(self, rows, high, n):
        """n ids a row, none of them twice: a step that is prime to `high` from a start of its own."""
        step = max(1, high // (n + 1))
        start = self.ids(high, rows, 1).long()
        return ((start + step * torch.arange(n, device="cuda")) % high).int()

    def quantised(self, x):
        """e4m3 codes of a matrix and one scale a row."""
        scale = x.abs().amax(1).clamp_min(1e-12) / E4M3_MAX
        return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    x = _Inputs(seed)
    state = {"kind": case["kind"]}
    state.update(_PREPARE[case["kind"]](case, x))
    if own:
        import lily_b200 as lily

        # An engine has one handle; norms and products take any of them.
        if case["kind"] == "adjust":
            state["scratch"] = lily.SamplerScratch(state["here"], max_rows=case["rows"], max_history=32768, max_list=128)
        else:
            state["scratch"] = lily.SamplerScratch(1024, max_rows=1, max_history=0)
    return state


def _norm(case, x):
    t, n, dtype = case["tokens"], case["hidden"], DTYPES[case["dtype"]]
    out = DTYPES[case["out"]]
    # Hidden states of real models have a few channels far above the rest.
    loud = 1.0 + 20.0 * (x.uniform(n) < 0.01)
    state = {"x": (x.normal(t, n) * loud).to(dtype), "weight": (1.0 + 0.2 * x.normal(n)).to(torch.bfloat16),
             "residual": (x.normal(t, n) * 2.0 * loud).to(dtype) if case["residual"] else None,
             "sum": torch.empty((t, n), dtype=dtype, device="cuda") if case["residual"] else None,
             "out": torch.empty((t, n), dtype=out, device="cuda"),
             "scales": torch.empty(t, device="cuda") if case["out"] == "e4m3" else None}
    return state


def _linear(case, x):
    t, k, n = case["tokens"], case["in"], case["outs"]
    a, w = x.normal(t, k), x.normal(n, k) / math.sqrt(k)
    state = {"a_scales": None, "w_scales": None, "act": case["act"]}
    if case["dtype"] == "e4m3":
        state["a"], state["a_scales"] = x.quantised(a)
        state["w"], state["w_scales"] = x.quantised(w)
    else:
        state["a"], state["w"] = a.to(torch.bfloat16), w.to(torch.bfloat16)
    dtype = DTYPES[case["out"]]
    state["bias"] = (0.5 * x.normal(n)).to(torch.bfloat16) if case["bias"] else None
    state["residual"] = x.normal(t, n).to(dtype) if case["residual"] else None
    state["out"] = torch.empty((t, n), dtype=dtype, device="cuda")
    return state


def _adjust(case, x):
    rows, v, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    # A vocabulary shard holds the logits of ids [first, first + here) of the v ids that lists and masks speak of.
    here = v // case["shards"]
    first = here * (case["shards"] // 2)
    state = {"logits": (3.0 * x.normal(rows, here)).to(dtype), "first": first, "here": here, "in_place": case["in_place"],
             "history": None, "bias_ids": None, "mask": None, "mask_rows": None, "params": None}
    state["out"] = state["logits"] if case["in_place"] else torch.empty_like(state["logits"])
    if case["history"]:
        h = case["history"]
        state["history"] = x.skewed_ids(v, rows, h)
        state["history_len"] = (h - x.ids(max(1, h // 4), rows)).int()
    pens = [(1.05 + 0.05 * (r % 8), 0.25 * (r % 3), 0.125 * (1 + r % 2) if case["frequency"] else 0.0) for r in range(rows)]
    state["pens"] = torch.tensor(pens, device="cuda") if case["history"] else None
    if own and case["history"]:
        import lily_b200 as lily

        state["params"] = [lily.SamplingParams(temperature=0.8, top_k=40, top_p=0.95, repetition_penalty=p,
                                               presence_penalty=q, frequency_penalty=f) for p, q, f in pens]
    if case["lists"]:
        n = case["lists"]
        state["bias_ids"], state["bias_vals"] = x.distinct(rows, v, n), 10.0 * x.uniform(rows, n) - 5.0
        state["bias_len"] = (n - x.ids(max(1, n // 2), rows)).int()
        state["ban_ids"] = x.distinct(rows, v, n)
        state["ban_len"] = (n - x.ids(max(1, n // 2), rows)).int()
    if case["mask"] != "none":
        # Masks belong to grammars: requests share them, and in a mixed batch some have none (-1).
        masks, words = max(1, rows // 2), (v + 31) // 32
        allowed = x.uniform(masks, words * 32) < {"tight": 0.002, "loose": 0.98, "mixed": 0.02}[case["mask"]]
        if case["mask"] == "mixed":  # half of a grammar's states take most of the vocabulary
            allowed[::2] = x.uniform((masks + 1) // 2, words * 32) < 0.9
        bits = allowed.view(masks, words, 32).long() << torch.arange(32, device="cuda")
        state["mask"] = bits.sum(2).int()  # (the words' 32 bits as they are)
        which = x.ids(masks, rows)
        if case["mask"] == "mixed":
            which = torch.where(torch.arange(rows, device="cuda") % 2 == 0, which, torch.full_like(which, -1))
        state["mask_rows"] = which
    return state


_PREPARE = {"norm": _norm, "linear": _linear, "adjust": _adjust}


# -------------------------------------------------------------- plain forms --


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    got = {}
    if s["residual"] is not None:
        got["sum"] = h.to(s["sum"].dtype)
    if s["scales"] is None:
        got["out"] = y.to(s["out"].dtype)
    else:
        m = y.abs().amax(1, keepdim=True).clamp_min(LEAST_MAX)
        got["out"] = (y * (E4M3_MAX / m)).to(torch.float8_e4m3fn)
        got["scales"] = (m / E4M3_MAX).view(-1)
    return got


def _activated(y, act):
    if act == "relu":
        return y.clamp_min(0.0)
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _product(s, dtype):
    y = s["a"].to(dtype) @ s["w"].to(dtype).t()
    if s["a_scales"] is not None:
        y = y * (s["a_scales"].to(dtype)[:, None] * s["w_scales"].to(dtype))
    if s["bias"] is not None:
        y = y + s["bias"].to(dtype)
    y = _activated(y, s["act"])
    if s["residual"] is not None:
        y = y + s["residual"].to(dtype)
    return y


def _plain_linear(s):
    return {"out": _product(s, torch.float32).to(s["out"].dtype)}


def _listed_ids(s, name):
    """A list's ids as places in the shard, and which of them count: within the list's length and the shard."""
    ids = s[name + ("" if name == "history" else "_ids")].long() - s["first"]
    n = torch.arange(ids.shape[1], device="cuda") < s[name + "_len"][:, None]
    live = n & (ids >= 0) & (ids < s["here"])
    return torch.where(live, ids, torch.zeros_like(ids)), live


def _plain_adjust(s):
    x = s["logits"].float()
    if s["bias_ids"] is not None:
        at, live = _listed_ids(s, "bias")
        x = x.scatter_add(1, at, s["bias_vals"] * live)
    if s["history"] is not None:
        at, live = _listed_ids(s, "history")
        count = torch.zeros_like(x).scatter_add_(1, at, live.float())
        rep, presence, frequency = (s["pens"][:, k:k + 1] for k in range(3))
        lowered = torch.where(x > 0, x / rep, x * rep) - (presence + frequency * count)
        x = torch.where(count > 0, lowered, x)
    if s["bias_ids"] is not None:
        at, live = _listed_ids(s, "ban")
        banned = torch.zeros_like(x).scatter_add_(1, at, live.float()) > 0
        x = torch.where(banned, torch.full_like(x, -math.inf), x)
    if s["mask"] is not None:
        ids = torch.arange(s["first"], s["first"] + s["here"], device="cuda")
        words = s["mask"][s["mask_rows"].long().clamp_min(0)][:, ids >> 5]
        allowed = ((words >> (ids & 31).int()) & 1 > 0) | (s["mask_rows"][:, None] < 0)
        x = torch.where(allowed, x, torch.full_like(x, -math.inf))
    s["out"].copy_(x)
    return {"out": s["out"]}


_PLAIN = {"norm": _plain_norm, "linear": _plain_linear, "adjust": _plain_adjust}


# ------------------------------------------------------------ the framework --


def _own_norm(s):
    s["scratch"].add_rms_norm(s["x"], s["weight"], s["out"], residual=s["residual"], residual_out=s["sum"],
                              out_scales=s["scales"], eps=EPS)
    return {k: s[k] for k in ("sum", "out", "scales") if s[k] is not None}


def _own_linear(s):
    s["scratch"].linear(s["a"], s["w"], s["out"], a_scales=s["a_scales"], weight_scales=s["w_scales"], bias=s["bias"],
                        activation=s["act"], residual=s["residual"])
    return {"out": s["out"]}


def _own_adjust(s):
    kw = {}
    if s["history"] is not None:
        kw.update(history_ids=s["history"], history_len=s["history_len"])
    if s["bias_ids"] is not None:
        kw.update(bias_ids=s["bias_ids"], bias_vals=s["bias_vals"], bias_len=s["bias_len"], ban_ids=s["ban_ids"],
                  ban_len=s["ban_len"])
    if s["mask"] is not None:
        kw.update(mask=s["mask"], mask_rows=s["mask_rows"])
    s["scratch"].adjust_logits(s["logits"], s["params"], s["out"], first_id=s["first"], **kw)
    return {"out": s["out"]}


_OWN = {"norm": _own_norm, "linear": _own_linear, "adjust": _own_adjust}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# -------------------------------------------------------------------- floors --


def work(case):
    """The bytes of every input once and of every output once, and the products' operations."""
    if case["kind"] == "norm":
        values = case["tokens"] * case["hidden"]
        per = ELEMENT[case["dtype"]] * (3 if case["residual"] else 1) + ELEMENT[case["out"]]
        return {"bytes": values * per + 2 * case["hidden"] + (4 * case["tokens"] if case["out"] == "e4m3" else 0),
                "flops": 6 * values}
    if case["kind"] == "linear":
        t, k, n, e = case["tokens"], case["in"], case["outs"], ELEMENT[case["dtype"]]
        scales = 4 * (t + n) if case["dtype"] == "e4m3" else 0
        out = ELEMENT[case["out"]] * t * n
        return {"bytes": (t + n) * k * e + scales + out * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0),
                "flops": 2 * t * k * n}
    rows, e = case["rows"], ELEMENT[case["dtype"]]
    here = case["vocab"] // case["shards"]
    # How many logits a mask takes away: those are written, but need not be read.
    away = {"none": 0.0, "tight": 0.998, "loose": 0.02, "mixed": 0.27}[case["mask"]]
    masks = min(rows, max(1, rows // 2)) if case["mask"] != "none" else 0
    lists = rows * (4 * case["history"] + 12 * case["lists"]) + masks * here // 8
    if case["in_place"]:
        return {"bytes": lists + rows * here * e * away, "flops": rows * here}
    return {"bytes": lists + rows * here * e * (2.0 - away), "flops": rows * here}


# --------------------------------------------------- the definitions, in 64 bits --


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_norm(s):
    h = s["x"].double()
    if s["residual"] is not None:
        h = h + s["residual"].double()
    mean = torch.einsum("tn,tn->t", h, h) / h.shape[1]
    y = (h / torch.sqrt(mean + EPS)[:, None]) * s["weight"].double()
    got = {"sum": h} if s["residual"] is not None else {}
    if s["scales"] is None:
        return {**got, "out": y}
    scale = torch.maximum(y.max(1).values, -y.min(1).values).clamp_min(LEAST_MAX) / E4M3_MAX
    return {**got, "out": y / scale[:, None], "scales": scale}


def _exact_linear(s):
    a, w = s["a"].double(), s["w"].double()
    if s["a_scales"] is not None:
        a, w = a * s["a_scales"].double()[:, None], w * s["w_scales"].double()[:, None]
    y = torch.einsum("tk,nk->tn", a, w)
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["act"] == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif s["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif s["act"] == "gelu":  # y times the normal distribution's integral up to y
        y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
    elif s["act"] == "gelu_tanh":
        y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    return {"out": y if s["residual"] is None else y + s["residual"].double()}


def _exact_adjust(s):
    """Row by row over the whole vocabulary, from the lists as they stand."""
    rows, here, first = s["logits"].shape[0], s["here"], s["first"]
    total = s["mask"].shape[1] * 32 if s["mask"] is not None else first + here
    out = torch.empty((rows, here), dtype=torch.float64, device="cuda")
    for r in range(rows):
        l = torch.zeros(max(total, first + here, 1 << 18), dtype=torch.float64, device="cuda")
        l[first:first + here] = s["logits"][r].double()
        if s["bias_ids"] is not None:
            n = int(s["bias_len"][r])
            l.index_add_(0, s["bias_ids"][r, :n].long(), s["bias_vals"][r, :n].double())
        if s["history"] is not None:
            ids, count = torch.unique(s["history"][r, :int(s["history_len"][r])].long(), return_counts=True)
            rep, presence, frequency = (float(p) for p in s["pens"][r])
            v = l[ids]
            l[ids] = v * torch.where(v > 0, 1.0 / rep, rep) - presence - frequency * count.double()
        if s["bias_ids"] is not None:
            l[s["ban_ids"][r, :int(s["ban_len"][r])].long()] = -math.inf
        if s["mask"] is not None and int(s["mask_rows"][r]) >= 0:
            word = s["mask"][int(s["mask_rows"][r])]
            bits = torch.stack([(word >> b) & 1 for b in range(32)], 1).view(-1)
            l[:bits.numel()][bits == 0] = -math.inf
        out[r] = l[first:first + here]
    return {"out": out}


_EXACT = {"norm": _exact_norm, "linear": _exact_linear, "adjust": _exact_adjust}
