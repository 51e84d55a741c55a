"""More operators of a batched decoder as cases that can be timed, each in its
plain form (elementary torch operations) and as the framework's own kernel.

A server whose sequences are long keeps their keys and values in 8 bits, a
scale for each place and key head, and answers with tokens that it samples:

* ``append``: the new tokens' keys normed per head and rotated, keys and values
  rounded to int8 as they are written to their slots of the paged cache, and the
  cache read back as float32;
* ``read``: places of such a cache as float32, as when a prefix is moved to
  another cache;
* ``attention``: the new tokens' queries over the shared beginning and each
  sequence's own pages of such a cache;
* ``sample``: rows of logits to tokens: temperature, top-k, top-p and min-p,
  from given random numbers.

``run`` takes the plain form where ``own`` is false and the framework's calls
where it is true; ``exact`` states each result in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One chat's token into its cache: the smallest call.
        {"name": "append one token", "kind": "append", "n": 1, "heads": 16, "kv_heads": 8,
         "hd": 128, "page": 16, "pages": 24, "norm": True},
        # The prompts of a batch that is let in at once, an odd number of tokens.
        {"name": "append prompts", "kind": "append", "n": 4093, "heads": 32, "kv_heads": 8,
         "hd": 128, "page": 64, "pages": 66, "norm": True},
        # The last places of a chat, to be written elsewhere.
        {"name": "read a few", "kind": "read", "n": 37, "kv_heads": 2, "hd": 64, "page": 16,
         "pages": 40},
        # A long shared beginning, moved to another cache.
        {"name": "read prefix", "kind": "read", "n": 8191, "kv_heads": 8, "hd": 128, "page": 64,
         "pages": 200},
        # Three short chats without a common beginning, head size 64: latency.
        {"name": "attention short", "kind": "attention", "seqs": 3, "tokens": 1, "prefix": 0,
         "own_low": 33, "own_high": 200, "heads": 8, "kv_heads": 2, "hd": 64, "page": 16,
         "window": 0, "gate": False},
        # A server's decode step: sixty-four chats of unequal lengths under one
        # system prompt.
        {"name": "attention decode", "kind": "attention", "seqs": 64, "tokens": 1, "prefix": 1000,
         "own_low": 128, "own_high": 4096, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64,
         "window": 0, "gate": False},
        # One sequence with a long document behind it: its keys are split.
        {"name": "attention long", "kind": "attention", "seqs": 1, "tokens": 1, "prefix": 0,
         "own_low": 131072, "own_high": 131072, "heads": 32, "kv_heads": 8, "hd": 128,
         "page": 256, "window": 0, "gate": False},
        # Drafted tokens and short prompts together: up to 37 tokens a sequence,
        # three query heads a key head, a sliding window that reaches into the
        # shared beginning, gated heads.
        {"name": "attention drafts window", "kind": "attention", "seqs": 6, "tokens": 37,
         "prefix": 777, "own_low": 40, "own_high": 500, "heads": 12, "kv_heads": 4, "hd": 64,
         "page": 16, "window": 512, "gate": True},
        # The second half of a prompt: as many keys before it as tokens in it.
        {"name": "attention prompt", "kind": "attention", "seqs": 1, "tokens": 2047, "prefix": 0,
         "own_low": 4099, "own_high": 4099, "heads": 16, "kv_heads": 8, "hd": 128, "page": 32,
         "window": 0, "gate": False},
        # One chat's next token, the usual filters: latency.
        {"name": "sample one", "kind": "sample", "rows": 1, "vocab": 128000, "filters": "top"},
        # A server's batch, whose users ask for different things.
        {"name": "sample batch", "kind": "sample", "rows": 64, "vocab": 151936,
         "filters": "mixed"},
        # A smaller vocabulary without filters, an odd size.
        {"name": "sample plain", "kind": "sample", "rows": 13, "vocab": 32003, "filters": "none"},
    ]


def _log(rng, low, high, step=1):
    """A size between low and high, even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "read", "attention", "attention", "sample"])
    if kind == "append":
        n, page = _log(rng, 1, 4000), rng.choice([16, 32, 64])
        return {"kind": kind, "n": n, "heads": 8 * rng.choice([1, 2, 3, 4]),
                "kv_heads": rng.choice([1, 2, 4, 8]), "hd": rng.choice([64, 128]), "page": page,
                "pages": -(-n // page) + rng.randint(1, 8), "norm": rng.random() < 0.6}
    if kind == "read":
        n, page = _log(rng, 1, 8000), rng.choice([16, 32, 64, 128])
        return {"kind": kind, "n": n, "kv_heads": rng.choice([1, 2, 4, 8]),
                "hd": rng.choice([64, 128]), "page": page,
                "pages": -(-n // page) + rng.randint(1, 64)}
    if kind == "attention":
        kv, low = rng.choice([1, 2, 4, 8]), _log(rng, 1, 1000)
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 500)
        return {"kind": kind, "seqs": _log(rng, 1, max(1, min(64, 1000 // tokens))),
                "tokens": tokens, "prefix": 0 if rng.random() < 0.4 else _log(rng, 30, 2000),
                "own_low": low, "own_high": low + _log(rng, 1, 3000),
                "heads": kv * rng.choice([1, 2, 3, 4]), "kv_heads": kv,
                "hd": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
                "window": rng.choice([0, 0, 0, 512]), "gate": rng.random() < 0.3}
    return {"kind": kind, "rows": _log(rng, 1, 60), "vocab": _log(rng, 500, 150000),
            "filters": rng.choice(["top", "mixed", "mixed", "none"])}


# ------------------------------------------------------- what a case amounts to

def _spread(i, low, high):
    """Whole numbers between low and high that the case alone fixes, ragged
    over the sequences (steps of the golden ratio)."""
    return low + int((i * 0.6180339887498949 + 0.5) % 1.0 * (high - low + 1))


def _batch(case):
    """New tokens and own keys (those of the new tokens among them) of each
    sequence; the rows of the batch, padded as a captured step's are."""
    n = [_spread(7 * i + 3, 1, case["tokens"]) for i in range(case["seqs"])]
    lens = [max(_spread(i, case["own_low"], case["own_high"]), n[i]) for i in range(case["seqs"])]
    return n, lens, -(-sum(n) // 8) * 8


def work(case):
    if case["kind"] == "append":
        n, hd, kv = case["n"], case["hd"], case["kv_heads"]
        places = case["pages"] * case["page"]
        new = n * hd * (8 * case["heads"] + 2 * kv * 4) + 4 * n * hd + 8 * n
        back = 2 * places * kv * (hd + 4 + 4 * hd)
        return {"bytes": new + 2 * n * kv * (hd + 4) + back,
                "flops": 8 * n * hd * (case["heads"] + kv) + 2 * places * kv * hd}
    if case["kind"] == "read":
        count = 2 * case["n"] * case["kv_heads"]
        return {"bytes": count * (5 * case["hd"] + 4) + 4 * case["n"],
                "flops": count * case["hd"]}
    if case["kind"] == "attention":
        n, lens, _ = _batch(case)
        window, prefix = case["window"], case["prefix"]
        pairs, seen, first = 0, 0, prefix
        for c, own_len in zip(n, lens):
            spans = [(max(0, p - window + 1) if window else 0, p + 1)
                     for p in range(prefix + own_len - c, prefix + own_len)]
            pairs += sum(b - a for a, b in spans)
            seen += spans[-1][1] - max(prefix, spans[0][0])
            first = min(first, spans[0][0])
        keys = seen + prefix - first
        return {"bytes": keys * 2 * case["kv_heads"] * (case["hd"] + 4)
                + sum(n) * case["heads"] * case["hd"] * 8,
                "flops": 4 * pairs * case["heads"] * case["hd"]}
    count = case["rows"] * case["vocab"]
    return {"bytes": 4 * count + 24 * case["rows"], "flops": 4 * count}


# --------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _x(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    """What a user's program holds before the call; with ``own`` also the
    handles, output buffers and workspaces that it keeps from step to step."""
    state = {"append": _prepare_append, "read": _prepare_read, "attention": _prepare_attention,
             "sample": _prepare_sample}[case["kind"]](case, _gen(seed))
    if own:
        from dianoia_amd import device
        state["D"] = device
        {"append": _keep_append, "read": _keep_read, "attention": _keep_attention,
         "sample": _keep_sample}[case["kind"]](state, case, device)
    return state


def _cache(case, g, pages):
    """Codes [pages][page][kv_heads][hd] and scales [pages][kv_heads][page] as an
    engine leaves them: some channels and some places larger than others."""
    codes, scales = [], []
    for _ in range(2):
        x = _x(g, pages, case["page"], case["kv_heads"], case["hd"])
        x *= torch.exp(0.4 * _x(g, case["kv_heads"], case["hd"]))
        x *= torch.exp(0.3 * _x(g, pages, case["page"], 1, 1))
        top = x.abs().amax(-1)
        codes.append((127 * x / top[..., None]).round_().to(torch.int8))
        scales.append((top / 127).transpose(1, 2).contiguous())
    return {"keys": codes[0], "values": codes[1], "key_scales": scales[0], "value_scales": scales[1]}


def _handle(s, D):
    s["cache"] = D.PagedCache(s["keys"], s["values"], s["key_scales"], s["value_scales"])


def _prepare_append(case, g):
    n, heads, kv, hd = case["n"], case["heads"], case["kv_heads"], case["hd"]
    places = case["pages"] * case["page"]
    # One projection's output holds q, k and v of a token side by side.
    qkv = _x(g, n, (heads + 2 * kv) * hd)
    q = qkv[:, :heads * hd].view(n, heads, hd)
    k = qkv[:, heads * hd:(heads + kv) * hd].view(n, kv, hd)
    v = qkv[:, (heads + kv) * hd:].view(n, kv, hd)
    # The rotation's table, one row a position: [cos(hd / 2), sin(hd / 2)].
    places_max = 8192
    freq = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(places_max, dtype=torch.float64, device="cuda")[:, None] * freq
    return {
        "case": case, "q": q, "k": k, "v": v, **_cache(case, g, case["pages"]),
        "rope": torch.cat([angle.cos(), angle.sin()], 1).float(),
        "positions": torch.randint(0, places_max, (n,), device="cuda", generator=g).int(),
        "slots": torch.randperm(places, device="cuda", generator=g)[:n].int(),
        "all": torch.arange(places, device="cuda").int(),
        "q_norm": 1 + 0.1 * _x(g, hd) if case["norm"] else None,
        "k_norm": 1 + 0.1 * _x(g, hd) if case["norm"] else None,
    }


def _keep_append(s, case, D):
    _handle(s, D)
    s["q_out"] = torch.empty(case["n"], case["heads"], case["hd"], device="cuda")
    s["back"] = [torch.empty(case["pages"] * case["page"], case["kv_heads"], case["hd"],
                             device="cuda") for _ in range(2)]


def _prepare_read(case, g):
    places = case["pages"] * case["page"]
    return {"case": case, **_cache(case, g, case["pages"]),
            "slots": torch.randperm(places, device="cuda", generator=g)[:case["n"]].int()}


def _keep_read(s, case, D):
    _handle(s, D)
    s["back"] = [torch.empty(case["n"], case["kv_heads"], case["hd"], device="cuda")
                 for _ in range(2)]


def _prepare_attention(case, g):
    n, lens, rows = _batch(case)
    page, prefix = case["page"], case["prefix"]
    need = [-(-length // page) for length in lens]
    shared = -(-prefix // page)
    pages = shared + sum(need)
    # A pool that has been in use: every sequence's pages lie anywhere.
    order = torch.randperm(pages, device="cuda", generator=g).int()
    width = max(need)
    ends = [sum(need[:i + 1]) for i in range(len(need))]
    at = torch.tensor([[shared + min(e - c + j, e - 1) for j in range(width)]
                       for e, c in zip(ends, need)], device="cuda")
    return {
        "case": case, **_cache(case, g, pages),
        "q": 2 * _x(g, rows, case["heads"], case["hd"]),
        "gate": _x(g, rows, case["heads"]) if case["gate"] else None,
        "starts": _ints([sum(n[:i]) for i in range(len(n) + 1)]), "lens": _ints(lens),
        "tables": order[at].contiguous(), "shared": order[:shared].contiguous(),
        "max_tokens": max(n), "max_len": max(lens), "rows": rows, "live": sum(n),
    }


def _keep_attention(s, case, D):
    _handle(s, D)
    s["batch"] = D.PagedBatch(s["starts"], s["lens"], s["tables"], s["rows"], s["max_tokens"],
                              s["max_len"], prefix_pages=s["shared"], prefix_len=case["prefix"])
    s["workspace"] = D.paged_attention_workspace(s["cache"], s["batch"], case["heads"])
    s["out"] = torch.zeros(s["rows"], case["heads"], case["hd"], device="cuda")


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    # A model's logits: a broad floor, and some tokens well above it.
    logits = 2.0 * _x(g, rows, vocab)
    some = torch.randint(0, vocab, (rows, 48), device="cuda", generator=g)
    logits.scatter_add_(1, some, 7 + 2.5 * _x(g, rows, 48))

    def column(values, dtype):
        return torch.tensor([values[i % len(values)] for i in range(rows)], dtype=dtype,
                            device="cuda")

    # Each kind of request: top-k 0, top-p 1 and min-p 0 keep everything,
    # temperature 0 is the greedy answer.
    temperature, top_k, top_p, min_p = {
        "none": ([1.0], [0], [1.0], [0.0]),
        "top": ([0.8], [40], [0.95], [0.0]),
        "mixed": ([0.7, 1.0, 0.0, 0.9, 1.3], [0, 50, 0, 20, 0, 1000, 0],
                  [0.9, 1.0, 0.95, 0.8], [0.0, 0.05, 0.0]),
    }[case["filters"]]
    return {"case": case, "logits": logits,
            "u": torch.rand(rows, device="cuda", generator=g),
            "temperature": column(temperature, torch.float32), "top_k": column(top_k, torch.int32),
            "top_p": column(top_p, torch.float32), "min_p": column(min_p, torch.float32)}


def _keep_sample(s, case, D):
    s["out"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
    s["workspace"] = D.sample_workspace(case["rows"], case["vocab"])


# ------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state, state["D"])
    return _PLAIN[state["case"]["kind"]](state)


def _own_append(s, D):
    D.paged_append(s["cache"], s["k"], s["v"], s["positions"], s["slots"], rope=s["rope"],
                   q=s["q"], q_out=s["q_out"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    D.paged_read(s["cache"], s["all"], s["back"][0], s["back"][1])
    return {"q": s["q_out"], "keys": s["back"][0], "values": s["back"][1]}


def _own_read(s, D):
    D.paged_read(s["cache"], s["slots"], s["back"][0], s["back"][1])
    return {"keys": s["back"][0], "values": s["back"][1]}


def _own_attention(s, D):
    D.paged_attention(s["cache"], s["batch"], s["q"], s["out"], s["workspace"],
                      window=s["case"]["window"], gate=s["gate"])
    return s["out"]


def _own_sample(s, D):
    D.sample(s["logits"], s["u"], s["out"], s["workspace"], temperature=s["temperature"],
             top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return s["out"]


def _rotated(x, norm, rope):
    """Per head: RMSNorm, then the rotation of the pairs (j, j + hd / 2)."""
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = rope[:, None, :half], rope[:, None, half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _codes(y):
    """Rows of 64 bits, in which a value next to the border of two codes goes
    to its own, as codes and scales."""
    top = y.abs().amax(-1, keepdim=True)
    code = 127 * y / top
    code = torch.trunc(code + torch.copysign(torch.full_like(code, 0.5), code))
    return code.to(torch.int8), (top[..., 0] / 127).float()


def _read_back(s, pages, rows):
    """Rows of pages of the cache as float32."""
    return [codes[pages, rows].float() * scales[pages, :, rows][..., None]
            for codes, scales in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"]))]


def _plain_append(s):
    c = s["case"]
    page, row = s["slots"].long() // c["page"], s["slots"].long() % c["page"]
    rope = s["rope"][s["positions"]]
    norm = None if s["k_norm"] is None else s["k_norm"].double()
    y = _rotated(s["k"].double(), norm, rope.double())
    s["keys"][page, row], s["key_scales"][page, :, row] = _codes(y)
    s["values"][page, row], s["value_scales"][page, :, row] = _codes(s["v"].double())
    places = s["all"].long()
    keys, values = _read_back(s, places // c["page"], places % c["page"])
    return {"q": _rotated(s["q"], s["q_norm"], rope), "keys": keys, "values": values}


def _plain_read(s):
    slots = s["slots"].long()
    keys, values = _read_back(s, slots // s["case"]["page"], slots % s["case"]["page"])
    return {"keys": keys, "values": values}


def _plain_attention(s):
    c = s["case"]
    kv, hd, page, prefix, window = c["kv_heads"], c["hd"], c["page"], c["prefix"], c["window"]
    group, rows, seqs = c["heads"] // kv, s["rows"], c["seqs"]
    dev = s["q"].device
    scale = 1.0 / math.sqrt(hd)
    n = (s["starts"][1:] - s["starts"][:-1]).long()
    step = torch.arange(s["max_tokens"], device=dev)
    # The queries of each sequence, padded to the most: [seqs][kv][tokens * group][hd].
    token = (s["starts"][:-1, None] + step).long()
    held = step < n[:, None]
    q = s["q"][torch.where(held, token, 0)].view(seqs, -1, kv, group, hd)
    lanes = s["max_tokens"] * group
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kv, lanes, hd)
    place = prefix + s["lens"][:, None].long() - n[:, None] + step

    def keys_at(pages, count):
        at = torch.arange(count, device=dev)
        found = _read_back(s, pages.long()[..., at // page], at % page)
        return [t.transpose(-3, -2) for t in found]

    k1, v1 = keys_at(s["shared"], prefix)             # [kv][prefix][hd]
    k2, v2 = keys_at(s["tables"], s["max_len"])       # [seqs][kv][len][hd]
    all_q = q.transpose(0, 1).reshape(kv, seqs * lanes, hd)
    s1 = (all_q @ k1.transpose(-1, -2)).view(kv, seqs, lanes, prefix).transpose(0, 1)
    s2 = q @ k2.transpose(-1, -2)
    scores = torch.cat([s1, s2], -1) * scale
    key = torch.arange(prefix + s["max_len"], device=dev)
    seen = key <= place[..., None]
    if window:
        seen = seen & (key > place[..., None] - window)
    seen = seen.repeat_interleave(group, 1)[:, None]   # [seqs][1][tokens * group][keys]
    scores = scores.masked_fill(~seen, -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    e1, e2 = e[..., :prefix], e[..., prefix:]
    o1 = (e1.transpose(0, 1).reshape(kv, seqs * lanes, prefix) @ v1).view(kv, seqs, lanes, hd)
    o1 = o1.transpose(0, 1)
    o = (o1 + e2 @ v2) / e.sum(-1, keepdim=True)
    o = o.view(seqs, kv, -1, group, hd).permute(0, 2, 1, 3, 4).reshape(seqs, -1, c["heads"], hd)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"][torch.where(held, token, 0)])[..., None]
    # One more row takes what the padding of the sequences leaves over.
    out = torch.zeros(rows + 1, c["heads"], hd, device=dev)
    out[torch.where(held, token, rows)] = o
    return out[:rows]


def _plain_sample(s):
    # 64 bits: sums of many small weights, and a border that a random number meets.
    l, t = s["logits"].double(), s["temperature"].double()[:, None]
    by_size, order = torch.sort(l, dim=-1, descending=True, stable=True)
    greedy = t <= 0
    w = torch.exp((by_size - by_size[:, :1]) / torch.where(greedy, 1.0, t))
    rank = torch.arange(l.shape[1], device=l.device)
    top_k = s["top_k"].long()[:, None]
    w = torch.where((top_k <= 0) | (rank < top_k), w, 0)
    before = torch.cumsum(w, -1) - w
    top_p = s["top_p"].double()[:, None]
    inside = (top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True))
    inside = inside & (w >= s["min_p"].double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(inside, w, 0))
    upto = torch.cumsum(kept, -1)
    token = (upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(-1)
    return torch.where(greedy[:, 0], order[:, 0], token).int()


_OWN = {"append": _own_append, "read": _own_read, "attention": _own_attention,
        "sample": _own_sample}
_PLAIN = {"append": _plain_append, "read": _plain_read, "attention": _plain_attention,
          "sample": _plain_sample}


# ------------------------------------------------------- the results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attention": _exact_attention,
            "sample": _exact_sample}[case["kind"]](case, s)


def _stored(s, which):
    """The whole cache in 64 bits, [pages][page][kv_heads][hd]."""
    return s[which + "s"].double() * s[which + "_scales"].double().transpose(1, 2)[..., None]


def _exact_append(case, s):
    half = case["hd"] // 2
    turn = torch.complex(*(t.double() for t in s["rope"][s["positions"].long()].split(half, 1)))

    def turned(x, norm):
        x = x.double()
        if norm is not None:
            x = norm.double() * x / (x.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    def rounded(y):
        top = y.abs().max(-1, keepdim=True).values
        return torch.sign(y) * torch.floor(127 * y.abs() / top + 0.5) * (top / 127)

    out = []
    for which, new in (("key", turned(s["k"], s["k_norm"])), ("value", s["v"].double())):
        flat = _stored(s, which).flatten(0, 1)
        flat[s["slots"].long()] = rounded(new)
        out.append(flat)
    return {"q": turned(s["q"], s["q_norm"]), "keys": out[0], "values": out[1]}


def _exact_read(case, s):
    slots = s["slots"].long()
    return {w + "s": _stored(s, w).flatten(0, 1)[slots] for w in ("key", "value")}


def _exact_attention(case, s):
    kv, hd, prefix, window = (case[k] for k in ("kv_heads", "hd", "prefix", "window"))
    group = case["heads"] // kv
    n, lens, rows = _batch(case)
    out = torch.zeros(rows, case["heads"], hd, dtype=torch.float64, device="cuda")

    def listed_keys(pages, count):
        pages = pages.long()
        return [(s[w + "s"][pages].double() * s[w + "_scales"][pages].double().transpose(1, 2)[..., None])
                .flatten(0, 1)[:count].permute(1, 0, 2) for w in ("key", "value")]

    first = listed_keys(s["shared"], prefix)
    t0 = 0
    for b, (count, length) in enumerate(zip(n, lens)):
        mine = listed_keys(s["tables"][b], length)
        k, v = (torch.cat([x, y], 1) for x, y in zip(first, mine))     # [kv][keys][hd]
        for i in range(0, count, 256):
            some = min(256, count - i)
            q = s["q"][t0 + i:t0 + i + some].double().view(some, kv, group, hd).permute(1, 2, 0, 3)
            w = (q.reshape(kv, group * some, hd) @ k.transpose(1, 2)).view(kv, group, some, -1)
            w = w / hd ** 0.5
            p = torch.arange(some, device="cuda")[:, None] + prefix + length - count + i
            j = torch.arange(prefix + length, device="cuda")
            hidden = (j > p) | (j <= p - window if window else torch.zeros_like(j > p))
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            o = (w.reshape(kv, group * some, -1) @ v).view(kv, group, some, hd).permute(2, 0, 1, 3)
            o = o.reshape(some, case["heads"], hd)
            if s["gate"] is not None:
                o = o / (1 + torch.exp(-s["gate"][t0 + i:t0 + i + some].double()))[..., None]
            out[t0 + i:t0 + i + some] = o
        t0 += count
    return out


def _exact_sample(case, s):
    """A row after the other, its tokens in the order of their logits."""
    tokens = []
    rows = zip(s["logits"].double().cpu().numpy(),
               *(s[k].double().cpu().numpy() for k in ("u", "temperature", "top_k", "top_p", "min_p")))
    for l, u, t, k, p, low in rows:
        order = np.lexsort((np.arange(l.size), -l))
        if t <= 0:
            tokens.append(int(order[0]))
            continue
        if k > 0:
            order = order[:int(k)]
        w = np.exp((l[order] - l[order[0]]) / t)
        if p < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1)]
        w = w[:max(1, int((w >= low).sum()))]
        at = np.sort(order[:w.size])
        sums = np.cumsum(np.exp((l[at] - l[order[0]]) / t))
        tokens.append(int(at[np.searchsorted(sums, u * sums[-1], side="right")]))
    return torch.tensor(tokens, dtype=torch.int32, device="cuda")
