"""Operators of a batched decoder as cases that can be timed, each in its
plain form (elementary torch operations) and as the framework's own kernel.

A server that decodes many sequences at once keeps their keys and values in
pages, lets sequences that begin alike share the pages of that beginning, and
runs its projections in 8-bit integers. One layer of such a step is a run of
these operators:

* ``append``: the new tokens' queries and keys normed per head and rotated by
  their positions, keys and values written to their slots of the paged cache;
* ``attention``: every sequence's new tokens over the shared beginning, whose
  keys are read once for all of them, and over the sequence's own pages;
* ``rows``: rows as int8 with one scale a row, the residual's addition and the
  RMSNorm before them or not (also the load-time form of bf16 weights);
* ``product``: int8 rows times int8 weights, exact integer sums, scaled by one
  scale a token and one a weight row.

``run`` takes the plain form where ``own`` is false and the framework's calls
where it is true; ``exact`` states each result in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One sequence's token into a float32 cache: the smallest call.
        {"name": "append one token", "kind": "append", "n": 1, "heads": 16, "kv_heads": 8,
         "hd": 128, "type": "f32", "page": 32, "pages": 160, "norm": True},
        # The prompts of a batch that is let in at once, bf16 pages, an odd
        # number of tokens.
        {"name": "append prompts", "kind": "append", "n": 4093, "heads": 32, "kv_heads": 8,
         "hd": 128, "type": "bf16", "page": 64, "pages": 96, "norm": True},
        # Three short chats without a common beginning, head size 64.
        {"name": "attention short", "kind": "attention", "seqs": 3, "tokens": 1, "prefix": 0,
         "own_low": 33, "own_high": 200, "heads": 8, "kv_heads": 2, "hd": 64, "type": "f32",
         "page": 16, "window": 0, "gate": False},
        # A server's decode step: sixteen chats under one system prompt.
        {"name": "attention shared prompt", "kind": "attention", "seqs": 16, "tokens": 1,
         "prefix": 2048, "own_low": 64, "own_high": 700, "heads": 16, "kv_heads": 8, "hd": 128,
         "type": "f32", "page": 32, "window": 0, "gate": False},
        # Drafted tokens and short prompts together: up to 37 tokens a
        # sequence, three query heads a key head, a sliding window that
        # reaches into the shared beginning, gated heads.
        {"name": "attention drafts window", "kind": "attention", "seqs": 6, "tokens": 37,
         "prefix": 777, "own_low": 40, "own_high": 500, "heads": 12, "kv_heads": 4, "hd": 64,
         "type": "f32", "page": 16, "window": 512, "gate": True},
        # The largest: 64 sequences over a long shared document, bf16 pages.
        {"name": "attention shared document", "kind": "attention", "seqs": 64, "tokens": 1,
         "prefix": 8192, "own_low": 128, "own_high": 2048, "heads": 32, "kv_heads": 8, "hd": 128,
         "type": "bf16", "page": 64, "window": 0, "gate": False},
        # A decode batch's residual, norm and int8 rows: latency.
        {"name": "rows norm decode", "kind": "rows", "rows": 16, "cols": 2048, "norm": True,
         "add": True, "source": "f32"},
        # The same of a long prompt.
        {"name": "rows norm prompt", "kind": "rows", "rows": 4099, "cols": 4096, "norm": True,
         "add": True, "source": "f32"},
        # Loading: a bf16 matrix as int8 with a scale for each output channel.
        {"name": "rows weights bf16", "kind": "rows", "rows": 8192, "cols": 4096, "norm": False,
         "add": False, "source": "bf16"},
        # A decode batch's projection: the weights' bytes are what it costs.
        {"name": "product decode", "kind": "product", "n": 13, "rows": 6144, "cols": 2048},
        # The vision encoder's first projection over its 1024 patches.
        {"name": "product vision", "kind": "product", "n": 1024, "rows": 4304, "cols": 1152},
        # A long prompt's projection.
        {"name": "product prompt", "kind": "product", "n": 2047, "rows": 8192, "cols": 4096},
    ]


def _log(rng, low, high, step=1):
    """A size between low and high, even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "rows", "product"])
    if kind == "append":
        n, page = _log(rng, 1, 4096), rng.choice([16, 32, 64, 128])
        return {"kind": kind, "n": n, "heads": 8 * rng.choice([1, 2, 3, 4]),
                "kv_heads": rng.choice([1, 2, 4, 8]), "hd": rng.choice([64, 128]),
                "type": rng.choice(["f32", "bf16"]), "page": page,
                "pages": -(-n // page) + rng.randint(1, 64), "norm": rng.random() < 0.6}
    if kind == "attention":
        kv, low, kept = rng.choice([1, 2, 4, 8]), _log(rng, 1, 400), rng.choice(["f32", "bf16"])
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 48)
        most = 32 if kept == "f32" else 64
        return {"kind": kind, "seqs": _log(rng, 1, min(most, 400 // tokens)), "tokens": tokens,
                "prefix": 0 if rng.random() < 0.25 else _log(rng, 30, 8192), "own_low": low,
                "own_high": low + _log(rng, 1, 1600), "heads": kv * rng.choice([1, 2, 3, 4]),
                "kv_heads": kv, "hd": rng.choice([64, 128]), "type": kept,
                "page": rng.choice([16, 32, 64, 128, 256]), "window": rng.choice([0, 0, 0, 512]),
                "gate": rng.random() < 0.3}
    if kind == "rows":
        norm = rng.random() < 0.6
        return {"kind": kind, "rows": _log(rng, 1, 4096), "cols": _log(rng, 256, 4096, 4),
                "norm": norm, "add": norm and rng.random() < 0.7,
                "source": "f32" if norm else rng.choice(["f32", "bf16"])}
    return {"kind": kind, "n": _log(rng, 1, 2048), "rows": _log(rng, 200, 8192),
            "cols": _log(rng, 256, 4096, 32)}


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


def _pad32(cols):
    return -(-cols // 32) * 32


def work(case):
    if case["kind"] == "append":
        row, size = case["hd"] * case["n"], {"f32": 4, "bf16": 2}[case["type"]]
        moved = row * (8 * case["heads"] + 2 * case["kv_heads"] * (4 + size)) + 4 * row + 8 * case["n"]
        return {"bytes": moved, "flops": 6 * row * (case["heads"] + case["kv_heads"])}
    if case["kind"] == "attention":
        n, lens, _ = _batch(case)
        size, window, prefix = {"f32": 4, "bf16": 2}[case["type"]], case["window"], case["prefix"]
        pairs, seen, first = 0, 0, prefix
        for c, own_len in zip(n, lens):
            spans = [(max(0, p - window + 1) if window else 0, p + 1)
                     for p in range(prefix + own_len - c, prefix + own_len)]
            pairs += sum(b - a for a, b in spans)
            seen += spans[-1][1] - max(prefix, spans[0][0])
            first = min(first, spans[0][0])
        keys = seen + prefix - first
        return {"bytes": keys * 2 * case["kv_heads"] * case["hd"] * size
                + sum(n) * case["heads"] * case["hd"] * 8,
                "flops": 4 * pairs * case["heads"] * case["hd"]}
    if case["kind"] == "rows":
        count = case["rows"] * case["cols"]
        source = 2 if case["source"] == "bf16" else 4
        return {"bytes": count * (source + (8 if case["add"] else 0)) + case["rows"] * 4
                + case["rows"] * _pad32(case["cols"]) + (4 * case["cols"] if case["norm"] else 0),
                "flops": 4 * count}
    n, rows, cols = case["n"], case["rows"], case["cols"]
    return {"bytes": rows * cols + n * cols + 4 * (n * rows + n + rows), "flops": 2 * n * rows * cols}


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
    state = {"append": _prepare_append, "attention": _prepare_attention, "rows": _prepare_rows,
             "product": _prepare_product}[case["kind"]](case, _gen(seed))
    if own:
        from dianoia_amd import device
        state["D"] = device
        {"append": _keep_append, "attention": _keep_attention, "rows": _keep_rows,
         "product": _keep_product}[case["kind"]](state, case, device)
    return state


def _cache(case, g, pages):
    shape = (pages, case["page"], case["kv_heads"], case["hd"])
    kind = TYPES[case["type"]]
    return _x(g, *shape).to(kind), _x(g, *shape).to(kind)


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
    keys, values = _cache(case, g, case["pages"])
    return {
        "case": case, "q": q, "k": k, "v": v, "keys": keys, "values": values,
        "rope": torch.cat([angle.cos(), angle.sin()], 1).float(),
        "positions": torch.randint(0, places_max, (n,), device="cuda", generator=g).int(),
        "slots": torch.randperm(places, device="cuda", generator=g)[:n].int(),
        "q_norm": 1 + 0.1 * _x(g, hd) if case["norm"] else None,
        "k_norm": 1 + 0.1 * _x(g, hd) if case["norm"] else None,
    }


def _keep_append(s, case, D):
    s["cache"] = D.PagedCache(s["keys"], s["values"])
    s["q_out"] = torch.empty(case["n"], case["heads"], case["hd"], device="cuda")


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
    keys, values = _cache(case, g, pages)
    return {
        "case": case, "keys": keys, "values": values,
        "q": 2 * _x(g, rows, case["heads"], case["hd"]),
        "gate": _x(g, rows, case["heads"]) if case["gate"] else None,
        "starts": _ints([sum(n[:i]) for i in range(len(n) + 1)]), "lens": _ints(lens),
        "tables": order[at].contiguous(), "shared": order[:shared].contiguous(),
        "max_tokens": max(n), "max_len": max(lens), "rows": rows, "live": sum(n),
    }


def _keep_attention(s, case, D):
    s["cache"] = D.PagedCache(s["keys"], s["values"])
    s["batch"] = D.PagedBatch(s["starts"], s["lens"], s["tables"], s["rows"], s["max_tokens"],
                              s["max_len"], prefix_pages=s["shared"], prefix_len=case["prefix"])
    s["workspace"] = D.paged_attention_workspace(s["cache"], s["batch"], case["heads"])
    s["out"] = torch.zeros(s["rows"], case["heads"], case["hd"], device="cuda")


def _prepare_rows(case, g):
    rows, cols = case["rows"], case["cols"]
    source = TYPES[case["source"]]
    size = 1.0 if source == torch.float32 else 0.02   # activations, or weights
    return {"case": case, "x": (size * _x(g, rows, cols)).to(source),
            "m": _x(g, rows, cols) if case["add"] else None,
            "w": 1 + 0.2 * _x(g, cols) if case["norm"] else None}


def _keep_rows(s, case, D):
    rows, cols = case["rows"], case["cols"]
    s["qs"] = torch.empty(rows, _pad32(cols), dtype=torch.int8, device="cuda")
    s["scales"] = torch.empty(rows, 1, device="cuda")
    s["x_out"] = torch.empty(rows, cols, device="cuda") if case["add"] else None


def _codes(g, rows, cols):
    """int8 rows as a quantizer leaves them: bell-shaped, one at least at the end of the range."""
    q = (_x(g, rows, cols) * 36).round_().clamp_(-127, 127)
    q[:, 0] = 127
    return q.to(torch.int8)


def _prepare_product(case, g):
    n, rows, cols = case["n"], case["rows"], case["cols"]
    return {"case": case, "w": _codes(g, rows, cols), "x": _codes(g, n, cols),
            "w_scale": (_x(g, rows).abs() + 0.5) * 1e-3, "x_scale": (_x(g, n).abs() + 0.5) * 1e-2}


def _keep_product(s, case, D):
    s["y"] = torch.empty(case["n"], case["rows"], device="cuda")


# ------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _OWN[state["case"]["kind"]](state, state["D"])
    return _PLAIN[state["case"]["kind"]](state)


def _own_append(s, D):
    D.paged_append(s["cache"], s["k"], s["v"], s["positions"], s["slots"], rope=s["rope"],
                   q=s["q"], q_out=s["q_out"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}


def _own_attention(s, D):
    D.paged_attention(s["cache"], s["batch"], s["q"], s["out"], s["workspace"],
                      window=s["case"]["window"], gate=s["gate"])
    return s["out"]


def _own_rows(s, D):
    c = s["case"]
    rows, cols, pad = c["rows"], c["cols"], _pad32(c["cols"])
    if c["norm"]:
        D.rms_norm_i8r(s["x"], s["w"], s["qs"], s["scales"], rows, cols, pad, EPS, m=s["m"],
                       x_out=s["x_out"])
    elif c["source"] == "bf16":
        D.quantize_i8r_bf16(s["x"], s["qs"], s["scales"], rows, cols, pad)
    else:
        D.quantize_i8r(s["x"], s["qs"], s["scales"], rows, cols, pad)
    return {"values": s["qs"] * s["scales"], "x": s["x_out"]}


def _own_product(s, D):
    c = s["case"]
    D.gemm_i8r(s["w"], s["w_scale"], s["x"], s["x_scale"], s["y"], c["rows"], c["cols"], c["n"])
    return s["y"]


def _rotated(x, norm, rope):
    """Per head: RMSNorm, then the rotation of the pairs (j, j + hd / 2)."""
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = rope[:, None, :half], rope[:, None, half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    rope = s["rope"][s["positions"]]
    keys, values = s["keys"], s["values"]
    keys.view(-1, c["kv_heads"], c["hd"])[s["slots"]] = _rotated(s["k"], s["k_norm"], rope).to(keys.dtype)
    values.view(-1, c["kv_heads"], c["hd"])[s["slots"]] = s["v"].to(values.dtype)
    return {"q": _rotated(s["q"], s["q_norm"], rope), "keys": keys, "values": values}


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
        spot = pages.long()[..., at // page] * page + at % page
        return [t.view(-1, kv, hd)[spot].float().transpose(-3, -2) for t in (s["keys"], s["values"])]

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


def _plain_rows(s):
    c = s["case"]
    x = s["x"].float()
    total = x + s["m"] if s["m"] is not None else x
    # 64 bits: a value next to the border of two codes goes to its own.
    y = total.double()
    if c["norm"]:
        y = y * s["w"].double() * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    top = y.abs().amax(-1, keepdim=True)
    code = 127 * y / top
    code = torch.trunc(code + torch.copysign(torch.full_like(code, 0.5), code))
    code = torch.nn.functional.pad(code, (0, _pad32(c["cols"]) - c["cols"])).to(torch.int8)
    return {"values": code * (top / 127).float(), "x": total if s["m"] is not None else None}


def _plain_product(s):
    # Sums of 8-bit products pass 24 bits: in 64.
    y = s["x"].double() @ s["w"].double().t()
    return (y * s["x_scale"].double()[:, None] * s["w_scale"].double()).float()


_OWN = {"append": _own_append, "attention": _own_attention, "rows": _own_rows,
        "product": _own_product}
_PLAIN = {"append": _plain_append, "attention": _plain_attention, "rows": _plain_rows,
          "product": _plain_product}


# ------------------------------------------------------- the results in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "rows": _exact_rows,
            "product": _exact_product}[case["kind"]](case, s)


def _exact_append(case, s):
    half = case["hd"] // 2
    turn = torch.complex(*(t.double() for t in s["rope"][s["positions"].long()].split(half, 1)))

    def turned(x, norm):
        x = x.double()
        if norm is not None:
            x = norm.double() * x / (x.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    keys, values = s["keys"].double(), s["values"].double()
    page, slot = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    keys[page, slot] = turned(s["k"], s["k_norm"])
    values[page, slot] = s["v"].double()
    return {"q": turned(s["q"], s["q_norm"]), "keys": keys, "values": values}


def _exact_attention(case, s):
    kv, hd, page, prefix, window = (case[k] for k in ("kv_heads", "hd", "page", "prefix", "window"))
    group = case["heads"] // kv
    n, lens, rows = _batch(case)
    out = torch.zeros(rows, case["heads"], hd, dtype=torch.float64, device="cuda")

    def listed_keys(pages, count):
        return [t[pages.long()].flatten(0, 1)[:count].double().permute(1, 0, 2)
                for t in (s["keys"], s["values"])]

    first = listed_keys(s["shared"], prefix)
    t0 = 0
    for b, (count, length) in enumerate(zip(n, lens)):
        mine = listed_keys(s["tables"][b], length)
        k, v = (torch.cat([x, y], 1) for x, y in zip(first, mine))     # [kv][keys][hd]
        q = s["q"][t0:t0 + count].double().view(count, kv, group, hd).permute(1, 2, 0, 3)
        w = (q.reshape(kv, group * count, hd) @ k.transpose(1, 2)).view(kv, group, count, -1) / hd ** 0.5
        p = torch.arange(prefix + length - count, prefix + length, device="cuda")[:, None]
        j = torch.arange(prefix + length, device="cuda")
        hidden = (j > p) | (j <= p - window if window else torch.zeros_like(j > p))
        w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
        o = (w.reshape(kv, group * count, -1) @ v).view(kv, group, count, hd).permute(2, 0, 1, 3)
        o = o.reshape(count, case["heads"], hd)
        if s["gate"] is not None:
            o = o / (1 + torch.exp(-s["gate"][t0:t0 + count].double()))[..., None]
        out[t0:t0 + count] = o
        t0 += count
    return out


def _exact_rows(case, s):
    total = s["x"].float() if s["m"] is None else s["x"] + s["m"]   # the sum is held in float32
    y = total.double()
    if case["norm"]:
        y = s["w"].double() * (y / (y.pow(2).sum(-1, keepdim=True) / case["cols"] + EPS).sqrt())
    top = y.abs().max(-1, keepdim=True).values
    code = torch.sign(y) * torch.floor(127 * y.abs() / top + 0.5)
    values = torch.zeros(case["rows"], _pad32(case["cols"]), dtype=torch.float64, device="cuda")
    values[:, :case["cols"]] = code * (top / 127)
    return {"values": values, "x": total.double() if s["m"] is not None else None}


def _exact_product(case, s):
    y = torch.empty(case["n"], case["rows"], dtype=torch.float64, device="cuda")
    for at in range(0, case["rows"], 1024):   # whole numbers below 2^53: exact
        part = s["w"][at:at + 1024].double() @ s["x"].double().t()
        y[:, at:at + 1024] = (part * s["w_scale"][at:at + 1024, None].double()).t()
    return y * s["x_scale"][:, None].double()
