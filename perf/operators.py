"""The operators of an autoregressive text stage beside the diffusion transformer, as cases that can be timed and compared: rotary
positions whose keys and values go into a paged cache, attention over whole prompts with rules for what a query sees and what its scores
become, and attention of one new token over the paged cache.

A text stage encodes or rewrites the prompt ahead of the denoising loop: prompts come packed or padded, in batches of a few to a few
dozen, and decode one token at a time. Head layouts are those of this package's cases (24 heads of 128, 32 heads on 8 of 64) and the
generic 32 on 8 of 128.
"""

import math

import torch

own = False  # False: plain torch operations; True: this package's kernels

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEVICE = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def _rope(name, tokens, heads, kv_heads, dim, rot, neox, cache, page, far, dtype):
    return dict(name=name, kind="rope", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, neox=neox, cache=cache, page=page,
                far=far, dtype=dtype)


def _ruled(name, batch, sq, sk, docs, heads, kv_heads, dim, causal, window, prefix, cap, bias, dtype):
    return dict(name=name, kind="ruled", batch=batch, sq=sq, sk=sk, docs=docs, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal,
                window=window, prefix=prefix, cap=cap, bias=bias, dtype=dtype)


def _paged(name, batch, least, most, page, heads, kv_heads, dim, window, cap, bias, dtype):
    return dict(name=name, kind="paged", batch=batch, least=least, most=most, page=page, heads=heads, kv_heads=kv_heads, dim=dim,
                window=window, cap=cap, bias=bias, dtype=dtype)


def listed():
    return [
        # one decoding step of 16 sequences: their new tokens' keys and values go to 16 places of the cache
        _rope("rope_step", 16, 32, 8, 128, 128, True, True, 16, 100_000, "bf16"),
        # a prompt batch without a cache (an encoder): interleaved pairs of a quarter of the head, an odd number of tokens
        _rope("rope_encoder", 8191, 24, 24, 128, 32, False, False, 0, 8192, "fp16"),
        # many long prompts at once, positions past the trained context
        _rope("rope_prompts", 65536, 32, 8, 128, 128, True, True, 64, 1_000_000, "bf16"),
        # one short prompt, causal
        _ruled("prompt_short", 1, 77, 77, 0, 24, 24, 128, True, 0, 0, 0.0, "", "bf16"),
        # an encoder's layer with a table of biases by distance: two prompts of 512 places packed, the padding a document of its own
        _ruled("encoder_distance_bias", 1, 1024, 1024, 4, 64, 64, 64, False, 0, 0, 0.0, "table", "bf16"),
        # capped scores, causal window of half the prompt, grouped heads
        _ruled("prompt_capped_window", 1, 8192, 8192, 0, 32, 8, 128, True, 4096, 0, 50.0, "", "bf16"),
        # ragged prompts packed into one sequence, each with a prefix that all its tokens see
        _ruled("prompts_packed_prefix", 1, 12007, 12007, 23, 32, 8, 64, True, 0, 96, 0.0, "", "fp16"),
        # a whole long prompt, causal, slopes by distance: the largest
        _ruled("prompt_long_slopes", 1, 16384, 16384, 0, 16, 16, 128, True, 0, 0, 0.0, "slopes", "bf16"),
        # one sequence decodes: latency
        _paged("decode_one", 1, 1000, 1000, 16, 32, 8, 128, 0, 0.0, "", "bf16"),
        # a batch of ragged lengths
        _paged("decode_ragged", 48, 17, 8192, 64, 32, 8, 128, 0, 0.0, "", "bf16"),
        # long contexts of a few sequences
        _paged("decode_long", 4, 100_000, 131_072, 64, 32, 8, 128, 0, 0.0, "", "bf16"),
        # heads without groups, capped scores in a window
        _paged("decode_capped_window", 32, 300, 4096, 32, 24, 24, 64, 1024, 30.0, "", "fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limit = {}
    for c in listed():
        w = work(c)
        for key in w:
            limit[c["kind"], key] = max(limit.get((c["kind"], key), 0), w[key])
    while True:
        case = _draw_one(rng)
        w = work(case)
        if all(w[key] <= limit[case["kind"], key] for key in w):
            return case


def _draw_one(rng):
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    dim = rng.choice((64, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 16, 24))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 4, 8)) if kv_heads <= 8 else kv_heads
    kind = rng.choice(("rope", "ruled", "ruled", "paged", "paged"))
    if kind == "rope":
        cache = rng.random() < 0.7
        case = _rope("", _log_int(rng, 1, 65536), heads, kv_heads, dim, rng.choice((dim, dim, dim // 2, dim // 4)), rng.random() < 0.6, cache,
                     rng.choice((16, 32, 64, 128)) if cache else 0, rng.choice((4096, 131_072, 1_000_000)), dtype)
    elif kind == "ruled":
        docs = rng.choice((0, 0, _log_int(rng, 1, 60)))
        sq = _log_int(rng, 1 if docs == 0 else max(2 * docs, 64), 16384)
        batch = 1 if docs else rng.choice((1, 1, 2, 3))
        sk = sq + (_log_int(rng, 1, 8192) if docs == 0 and rng.random() < 0.3 else 0)
        causal = rng.random() < 0.75
        case = _ruled("", batch, sq, sk, docs, heads, kv_heads, dim, causal, rng.choice((0, 0, _log_int(rng, 1, 6000))),
                      rng.choice((0, 0, _log_int(rng, 1, 600))) if causal else 0, rng.choice((0.0, 0.0, 30.0, 50.0)),
                      rng.choice(("", "", "slopes", "table")), dtype)
    else:
        most = _log_int(rng, 1, 131_072)
        case = _paged("", _log_int(rng, 1, 64), max(1, most // rng.choice((1, 2, 100))), most, rng.choice((16, 32, 64, 128)), heads, kv_heads, dim,
                      rng.choice((0, 0, 0, _log_int(rng, 1, 4096))), rng.choice((0.0, 0.0, 30.0)), rng.choice(("", "", "slopes", "table")), dtype)
    del case["name"]
    # what the plain form holds of a drawn case at once stays at what it holds of the largest listed one
    if kind == "ruled" and case["batch"] * heads * case["sq"] * case["sk"] > 16 * 16384 * 16384:
        return _draw_one(rng)
    if kind == "paged" and case["batch"] * most * heads * dim > 48 * 8192 * 32 * 128:
        return _draw_one(rng)
    return case


# ----------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """The lengths of a paged case's sequences, spread evenly over the logarithm of their range: plain numbers, the same for every seed."""
    n, lo, hi = case["batch"], case["least"], case["most"]
    if n == 1:
        return [hi]
    return [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _bounds(case):
    """Where the documents of a packed case begin and the last one ends: ragged, the same for every seed."""
    n, total = case["docs"], case["sq"]
    share = [1.0 + (7 * i * i + 3 * i) % 11 for i in range(n)]
    ends = [0]
    for i in range(n):
        ends.append(total if i == n - 1 else min(total, ends[-1] + int(total * share[i] / sum(share))))
    return ends


def _randn(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device=_DEVICE, dtype=torch.float32) * std).to(dtype)


def _bias(case, gen, state):
    if case["bias"] == "slopes":  # a geometric row of slopes, the steepest 1/2
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / case["heads"]) for i in range(case["heads"])], device=_DEVICE)
    elif case["bias"] == "table":  # one bias for each distance up to 128 either way, the last for all further ones
        state["distance"] = _randn(gen, (case["heads"], 257), torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE)
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    state = {"case": case}
    if case["kind"] == "rope":
        t = case["tokens"]
        # q, k and v are parts of one projection's output, as a model has them
        qkv = _randn(gen, (t, (h + 2 * hkv) * d), dtype)
        state["q"], state["k"], state["v"] = (x.view(t, -1, d) for x in qkv.split((h * d, hkv * d, hkv * d), dim=1))
        state["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device=_DEVICE)
        i = torch.arange(case["rot"] // 2, device=_DEVICE, dtype=torch.float64)
        # turns per position: base 10000, stretched four times for the longer context
        state["turns"] = torch.pow(10000.0, -2.0 * i / case["rot"]) / (4.0 * 2.0 * math.pi)
        state["magnitude"] = 0.1 * math.log(4.0) + 1.0
        if case["cache"]:
            pages = -(-2 * t // case["page"])
            state["key_cache"] = _randn(gen, (pages, case["page"], hkv, d), dtype)
            state["value_cache"] = _randn(gen, (pages, case["page"], hkv, d), dtype)
            state["slots"] = torch.randperm(pages * case["page"], generator=gen, device=_DEVICE)[:t].contiguous()
    elif case["kind"] == "ruled":
        b = case["batch"]
        state["q"] = _randn(gen, (b, case["sq"], h, d), dtype, 2.0)
        state["k"] = _randn(gen, (b, case["sk"], hkv, d), dtype)
        state["v"] = _randn(gen, (b, case["sk"], hkv, d), dtype)
        state["scale"] = d ** -0.5
        if case["docs"]:
            state["starts"] = torch.tensor(_bounds(case), dtype=torch.int32, device=_DEVICE)
        if case["prefix"]:
            state["prefix"] = torch.full((case["docs"] or b,), case["prefix"], dtype=torch.int32, device=_DEVICE)
        _bias(case, gen, state)
    else:
        lengths, page = _lengths(case), case["page"]
        most = -(-max(lengths) // page)
        used = [-(-n // page) for n in lengths]
        pages = sum(used)
        # pages in the order in which a server hands them out, which is no order
        order = torch.randperm(pages, generator=gen, device=_DEVICE).to(torch.int32)
        table = torch.zeros((case["batch"], most), dtype=torch.int32, device=_DEVICE)
        at = 0
        for i, n in enumerate(used):
            table[i, :n] = order[at:at + n]
            at += n
        state["table"] = table
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=_DEVICE)
        state["q"] = _randn(gen, (case["batch"], h, d), dtype, 2.0)
        state["key_cache"] = _randn(gen, (pages, page, hkv, d), dtype)
        state["value_cache"] = _randn(gen, (pages, page, hkv, d), dtype)
        state["scale"] = d ** -0.5
        _bias(case, gen, state)
    return state


# ------------------------------------------------------------------------------------------------ plain
def _rotate(x, cos, sin, neox):
    """float32 rotation of the first 2 * cos.shape[-1] features of x [T,H,D]."""
    half = cos.shape[-1]
    x = x.float()
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None], sin[:, None]
    if neox:
        a, b = turned[..., :half], turned[..., half:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    return torch.cat((out, rest), dim=-1)


def _plain_rope(s):
    case = s["case"]
    angle = s["positions"].double()[:, None] * s["turns"] * (2.0 * math.pi)
    cos, sin = ((f(angle) * s["magnitude"]).float() for f in (torch.cos, torch.sin))
    q = _rotate(s["q"], cos, sin, case["neox"]).to(s["q"].dtype)
    k = _rotate(s["k"], cos, sin, case["neox"]).to(s["k"].dtype)
    if not case["cache"]:
        return q, k
    page = s["slots"] // case["page"], s["slots"] % case["page"]
    s["key_cache"][page] = k
    s["value_cache"][page] = s["v"]
    return q, s["key_cache"], s["value_cache"]


def _seen(case, s, rows, keys):
    """Which keys each query sees, [Sq,Sk] or None for all of them, and the keys' distances from the queries' positions."""
    i, j = torch.arange(rows, device=_DEVICE)[:, None], torch.arange(keys, device=_DEVICE)[None]
    pos = i + (keys - rows)
    away = j - pos
    seen = away <= 0 if case["causal"] else torch.ones_like(away, dtype=torch.bool)
    if case["window"]:
        seen = seen & (away.abs() < case["window"])
    first = torch.zeros((), dtype=torch.int64, device=_DEVICE)
    if case["docs"]:
        doc = torch.searchsorted(s["starts"], torch.arange(keys, device=_DEVICE, dtype=torch.int32), right=True) - 1
        first = s["starts"].long()[doc]
    if case["prefix"]:
        seen = seen | (j - first < case["prefix"])
    if case["docs"]:
        seen = seen & (doc[:, None] == doc[None])
    return seen, away


def _biased(scores, case, s, away):
    """Capped and biased scores; `away` broadcasts against them from behind the head axis."""
    if case["cap"]:
        scores = scores.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["bias"] == "slopes":
        scores -= s["slopes"].to(scores.dtype)[:, None, None] * away.abs()
    elif case["bias"] == "table":
        scores += s["distance"].to(scores.dtype)[:, away.clamp(-128, 128) + 128]
    return scores


def _softmax(scores):
    scores = (scores - scores.amax(dim=-1, keepdim=True)).exp_()
    return scores.div_(scores.sum(dim=-1, keepdim=True))


def _plain_ruled(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    q = s["q"].float().transpose(1, 2).contiguous()
    k, v = (s[n].float().repeat_interleave(group, dim=2).transpose(1, 2).contiguous() for n in ("k", "v"))
    seen, away = _seen(case, s, case["sq"], case["sk"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    scores = _biased(scores, case, s, away).masked_fill_(~seen, -math.inf)
    return torch.matmul(_softmax(scores), v).transpose(1, 2).to(s["q"].dtype)


def _plain_paged(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    k, v = (s[n][s["table"].long()].flatten(1, 2).float().repeat_interleave(group, dim=2) for n in ("key_cache", "value_cache"))
    j = torch.arange(k.shape[1], device=_DEVICE)[None, None]
    away = j - (s["lengths"].long()[:, None, None] - 1)
    seen = (away <= 0) & (away > -(case["window"] or case["most"]))
    scores = (s["q"].float()[:, None] * k).sum(dim=-1).mul_(s["scale"]).transpose(1, 2)
    if case["bias"] == "table":
        scores = _capped(scores, case)
        scores = scores + s["distance"][:, away[:, 0].clamp(-128, 128) + 128].transpose(0, 1)
    else:
        scores = _biased(scores[:, :, None].contiguous(), case, s, away[:, None])[:, :, 0]
    weights = _softmax(scores.masked_fill(~seen, -math.inf))
    return (weights.transpose(1, 2)[..., None] * v).sum(dim=1).to(s["q"].dtype)


def _capped(scores, case):
    return (scores / case["cap"]).tanh() * case["cap"] if case["cap"] else scores


# -------------------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if own:
        return _own(state)
    return {"rope": _plain_rope, "ruled": _plain_ruled, "paged": _plain_paged}[case["kind"]](state)


def _own(s):
    from vllm_omni_amd import kernels

    case = s["case"]
    if case["kind"] == "rope":
        q, k = kernels.rope_append(s["q"], s["k"], s["v"] if case["cache"] else None, s["positions"], s["turns"], neox=case["neox"],
                                   magnitude=s["magnitude"], slots=s.get("slots"), key_cache=s.get("key_cache"),
                                   value_cache=s.get("value_cache"))
        return (q, s["key_cache"], s["value_cache"]) if case["cache"] else (q, k)
    if case["kind"] == "ruled":
        return kernels.attn_ruled(s["q"], s["k"], s["v"], s["scale"], causal=case["causal"], window=case["window"] or None,
                                  prefix=s.get("prefix"), q_starts=s.get("starts"), k_starts=s.get("starts"), cap=case["cap"],
                                  slopes=s.get("slopes"), distance=s.get("distance"))
    return kernels.attn_paged(s["q"], s["key_cache"], s["value_cache"], s["table"], s["lengths"], s["scale"], window=case["window"] or None,
                              cap=case["cap"], slopes=s.get("slopes"), distance=s.get("distance"))


# ------------------------------------------------------------------------------------------------- work
def _visible(rows, keys, causal, window, prefix):
    """Pairs of a query and a key it sees, of one document (or batch row) of so many rows and keys."""
    total = 0
    for i in range(rows):
        pos = i + keys - rows
        lo = max(0, pos - window + 1) if window else 0
        hi = min(keys, pos + 1) if causal else keys if not window else min(keys, pos + window)
        total += max(0, hi - lo) + max(0, min(prefix, keys, max(lo, 0))) + max(0, min(prefix, keys) - max(hi, 0))
    return total


def work(case):
    h, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rope":
        t, parts = case["tokens"], h + (2 if case["cache"] else 1) * hkv
        return {"bytes": 2 * 2 * t * parts * d + t * (16 if case["cache"] else 8) + 4 * case["rot"], "flops": 3 * t * (h + hkv) * case["rot"]}
    if case["kind"] == "ruled":
        rule = case["causal"], case["window"], case["prefix"]
        if case["docs"]:
            ends = _bounds(case)
            pairs = sum(_visible(b - a, b - a, *rule) for a, b in zip(ends, ends[1:]))
        else:
            pairs = case["batch"] * _visible(case["sq"], case["sk"], *rule)
        return {"bytes": 2 * case["batch"] * d * (2 * case["sq"] * h + 2 * case["sk"] * hkv), "flops": 4 * pairs * h * d}
    keys = sum(min(n, case["window"] or n) for n in _lengths(case))
    return {"bytes": 2 * d * (2 * keys * hkv + 2 * case["batch"] * h), "flops": 4 * keys * h * d}


# ------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "ruled": _exact_ruled, "paged": _exact_paged}[case["kind"]](case, s)


def _exact_rope(case, s):
    # pairs as complex numbers, turned by a complex number of the magnitude's size
    turn = torch.polar(torch.full_like(s["turns"][None] * s["positions"][:, None], s["magnitude"]),
                       (s["positions"][:, None].double() * s["turns"] % 1.0) * (2.0 * math.pi))[:, None]
    half = case["rot"] // 2

    def turned(x):
        y = x.double().clone()
        at = (slice(0, half), slice(half, 2 * half)) if case["neox"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        z = torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous()) * turn
        y[..., at[0]], y[..., at[1]] = z.real, z.imag
        return y

    q, k = turned(s["q"]), turned(s["k"])
    if not case["cache"]:
        return q, k
    caches = [s[n].double().flatten(0, 1) for n in ("key_cache", "value_cache")]
    caches[0][s["slots"]] = k
    caches[1][s["slots"]] = s["v"].double()
    return (q, *(c.view(s["key_cache"].shape) for c in caches))


def _exact_row(q, k, v, see, away, case, s, head):
    """One head's attention in 64 bits: q [n,D] against k, v [m,D]; `see` and `away` [n,m]."""
    scores = (q.double() @ k.double().t().contiguous()) * s["scale"]
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    if case["bias"] == "slopes":
        scores = scores - float(s["slopes"][head]) * away.abs()
    if case["bias"] == "table":
        scores = scores + s["distance"][head].double()[torch.clamp(away, -128, 128) + 128]
    scores = torch.where(see, scores, -math.inf)
    weights = torch.exp(scores - torch.logsumexp(scores, dim=-1, keepdim=True))
    return weights @ v.double()


def _exact_ruled(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEVICE)
    group = case["heads"] // case["kv_heads"]
    ends = _bounds(case) if case["docs"] else [0, case["sq"]]
    for a, b in zip(ends, ends[1:]):
        # queries a to b of keys a to b + (sk - sq), whose last ones the queries are
        n, m = b - a, b - a + case["sk"] - case["sq"]
        if n == 0:
            continue
        row, col = torch.meshgrid(torch.arange(m - n, m, device=_DEVICE), torch.arange(m, device=_DEVICE), indexing="ij")
        see = torch.full((n, m), True, device=_DEVICE)
        if case["causal"]:
            see &= col <= row
        if case["window"]:
            see &= (row - col < case["window"]) & (col - row < case["window"])
        if case["prefix"]:
            see |= col < case["prefix"]
        for x in range(case["batch"]):
            for head in range(case["heads"]):
                out[x, a:b, head] = _exact_row(s["q"][x, a:b, head], s["k"][x, a:a + m, head // group], s["v"][x, a:a + m, head // group],
                                               see, col - row, case, s, head)
    return out


def _exact_paged(case, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEVICE)
    group = case["heads"] // case["kv_heads"]
    for x, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        j = torch.arange(first, n, device=_DEVICE)
        page, at = s["table"][x].long()[j // case["page"]], j % case["page"]
        k, v = s["key_cache"][page, at], s["value_cache"][page, at]
        see = torch.ones((1, n - first), dtype=torch.bool, device=_DEVICE)
        for head in range(case["heads"]):
            out[x, head] = _exact_row(s["q"][x, head][None], k[:, head // group], v[:, head // group], see, (j - (n - 1))[None], case, s, head)[0]
    return out
