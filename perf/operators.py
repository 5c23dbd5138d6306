"""Workloads of the operators that answer from a model's prepared attention: writing keys and values into a
paged cache, attending to it token by token, reading it back, and the log probabilities of the answer.

The forms of a call (``op``):

* ``append``    ``norm_rope_to_cache``: per-head Q/K RMSNorm + RoPE of new tokens at positions of their own, K and V
  written into the cache's pages (bf16, or e4m3 with one power-of-two scale per row).  ``proj``: q, k and v are
  views of projections [B,S,H,D], as a model has them, else contiguous [B,H,S,D];
* ``decode``    ``attention_decode``: attention of the last ``s`` tokens of each sequence over its pages;
* ``dense``     ``cache_to_dense``: the pages of a batch as contiguous bf16 [B,Hkv,L,D];
* ``logprobs``  ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives.

Head geometries are those of the package's model table.  Activations are N(0,1), gamma = 1 + 0.1 N(0,1),
theta = 1e6, as in the package's benchmark.  ``ragged`` batches hold sequences of all lengths up to ``l``, an empty
one among them; their lengths belong to the case, everything else to the seed.
"""
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
HEADS = {"0.6B": (16, 8, 128), "8B": (32, 8, 128), "30B": (32, 4, 128), "32B": (64, 8, 128),
         "gemma-4B": (8, 4, 256), "gemma-12B": (16, 8, 256)}


def _append(name, model, b, s, *, kind="bf16", style="hf", rope=True, proj=True, page=PAGE):
    c = {"op": "append", "model": model, "b": b, "s": s, "kind": kind, "style": style, "rope": rope, "proj": proj,
         "page": page}
    return dict(c, name=name) if name else c


def _decode(name, model, b, l, *, s=1, kind="bf16", ragged=False, window=0, cap=0.0, page=PAGE):
    c = {"op": "decode", "model": model, "b": b, "l": l, "s": s, "kind": kind, "ragged": ragged, "window": window,
         "cap": cap, "page": page}
    return dict(c, name=name) if name else c


def _dense(name, model, b, l, *, kind="bf16", ragged=False, page=PAGE):
    c = {"op": "dense", "model": model, "b": b, "l": l, "kind": kind, "ragged": ragged, "page": page}
    return dict(c, name=name) if name else c


def _logprobs(name, n, v, *, kind="f32", top=0, masked=False, shifted=False):
    c = {"op": "logprobs", "n": n, "v": v, "kind": kind, "top": top, "masked": masked, "shifted": shifted}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One new token of one sequence, as every layer of a decode step writes it: latency.
        _append("append 8B b1 s1", "8B", 1, 1),
        # A ragged prefill batch of a D = 256 model into a quantised cache.
        _append("append gemma-12B b4 s1000 e4m3", "gemma-12B", 4, 1000, kind="e4m3", style="fp32"),
        # The largest write: a long prompt.
        _append("append 8B b1 s8192", "8B", 1, 8192, proj=False, style="fp32"),
        # One new token after a short prompt: latency.
        _decode("decode 8B b1 l333", "8B", 1, 333),
        # One long conversation alone on the card: the length has to be split.
        _decode("decode 8B b1 l32768", "8B", 1, 32768),
        # A serving batch of all lengths, the largest read.
        _decode("decode 8B b64 l8192 ragged", "8B", 64, 8192, ragged=True),
        # D = 256 with a sliding window over a quantised cache.
        _decode("decode gemma-12B b32 window e4m3", "gemma-12B", 32, 4096, kind="e4m3", window=1024, page=32),
        # Four drafted tokens checked at once, eight query heads to a KV head, scores capped.
        _decode("decode 32B b16 s4 cap e4m3", "32B", 16, 4096, s=4, kind="e4m3", cap=50.0),
        # A batch of sequences handed on as dense keys and values.
        _dense("dense gemma-12B b8 l4096 e4m3", "gemma-12B", 8, 4096, kind="e4m3", ragged=True),
        # One short sequence handed on: latency.
        _dense("dense 8B b1 l333", "8B", 1, 333),
        # A sampling step of a batch whose vocabulary is mostly ruled out by a grammar, odd vocabulary.
        _logprobs("logprobs n64 v131071 top20", 64, 131071, top=20, masked=True),
        # Scoring the tokens of eight prompts from their logits: no alternatives asked for.
        _logprobs("logprobs n4096 v32000 bf16", 4096, 32000, kind="bf16", shifted=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: 1 to 128 sequences, 1 to 8192 new or 1 to 32768 cached tokens, pages of 16 to 256,
    up to 4096 rows of logits over 1000 to 262144 tokens, at most the largest listed case's work."""
    while True:
        op = rng.choice(["append"] * 3 + ["decode"] * 5 + ["dense"] * 2 + ["logprobs"] * 4)
        model = rng.choice(sorted(HEADS))
        hq, hkv, d = HEADS[model]
        page = rng.choice([16, 32, 64, 64, 128, 256])
        kind = rng.choice(["bf16", "bf16", "e4m3"])
        if op == "append":
            b, s = (_log_int(rng, 1, 128), 1) if rng.random() < 0.4 else (_log_int(rng, 1, 16), _log_int(rng, 2, 8192))
            if b * s * (hq + 2 * hkv) * d > 8192 * 48 * 128:
                continue
            return _append(None, model, b, s, kind=kind, style=rng.choice(["hf", "fp32", "fp32", "legacy"]),
                           rope=rng.random() < 0.85, proj=rng.random() < 0.7, page=page)
        if op == "decode":
            b, l = _log_int(rng, 1, 128), _log_int(rng, 1, 32768)
            s = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
            if b * hkv * l * d > 64 * 8 * 8192 * 128 * 0.7 or l < s:
                continue
            return _decode(None, model, b, l, s=s, kind=kind, ragged=rng.random() < 0.6, page=page,
                           window=_log_int(rng, 16, 4096) if rng.random() < 0.3 else 0,
                           cap=rng.choice([30.0, 50.0]) if rng.random() < 0.25 else 0.0)
        if op == "dense":
            b, l = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
            if b * hkv * l * d > 8 * 8 * 4096 * 256:
                continue
            return _dense(None, model, b, l, kind=kind, ragged=rng.random() < 0.6, page=page)
        n, v = _log_int(rng, 1, 4096), _log_int(rng, 1000, 262144)
        if n * v > 4096 * 32000:
            continue
        top = rng.choice([0, 1, 1, 5, 20])
        if top and n * v > 2 ** 25:
            continue
        return _logprobs(None, n, v, kind=rng.choice(["f32", "bf16", "f16"]), top=top, masked=rng.random() < 0.25,
                         shifted=n >= 8 and rng.random() < 0.4)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """The lengths of a case's sequences: the case's own, so that its work is known without a seed."""
    b, l, s = case["b"], case["l"], case.get("s", 1)
    if not case["ragged"] or b == 1:
        return [l] * b
    r = random.Random(b * 1000003 + l)
    lens = [r.randint(min(s, l), l) for _ in range(b)]
    lens[0], lens[-1] = l, 0
    return lens


def _tables(n, d):
    pos = torch.arange(n, dtype=torch.float64, device="cuda")
    inv = 1.0 / (THETA ** (torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d))
    ang = torch.cat([pos[:, None] * inv[None, :]] * 2, dim=1)
    return ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)


def _quantised(x):
    """Rows of x as (e4m3 payload, power-of-two scale): the smallest scale that brings the row's largest magnitude
    to 448 or below; a row of zeros has scale 1."""
    x = x.float()
    mant, ex = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = (ex - 9 + (mant > 0.875)).clamp(-124, 127)
    e = torch.where(mant == 0, torch.zeros_like(e), e)
    payload = torch.ldexp(x, -e).to(torch.float8_e4m3fn)
    return payload, (e[..., 0] + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _empty_cache(n, hkv, page, d, kind):
    pair = [torch.zeros(n, hkv, page, d, device="cuda", dtype=DTYPES[kind]) for _ in range(2)]
    scales = [None, None] if kind == "bf16" else [
        torch.zeros(n, hkv, page, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    return pair + scales


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        return _logits(case, g)
    hq, hkv, d = HEADS[case["model"]]
    b, page, kind = case["b"], case["page"], case["kind"]
    if case["op"] == "append":
        s = case["s"]

        def rows(h):
            x = _normal(g, b, s, h, d).to(torch.bfloat16).transpose(1, 2)
            return x if case["proj"] else x.contiguous()

        x = {"q": rows(hq), "k": rows(hkv), "v": rows(hkv)}
        x["gq"], x["gk"] = ((1 + 0.1 * _normal(g, d)).to(torch.bfloat16) for _ in range(2))
        # every sequence has some tokens in the cache already and pages anywhere in it
        before = torch.randint(0, 3 * page, (b, 1), generator=g, device="cuda")
        x["positions"] = before + torch.arange(s, device="cuda")
        per = (s + 3 * page - 2) // page + 1
        x["cos"], x["sin"] = _tables(3 * page + s, d) if case["rope"] else (None, None)
        table = torch.randperm(b * per, generator=g, device="cuda").view(b, per)
        x["slots"] = torch.gather(table, 1, x["positions"] // page) * page + x["positions"] % page
        x["cache"] = _empty_cache(b * per, hkv, page, d, kind)
        return x
    lens = _lengths(case)
    per = -(-case["l"] // page)
    x = {"lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "pages": torch.randperm(b * per, generator=g, device="cuda").view(b, per).to(torch.int32)}
    if case["op"] == "decode":
        x["q"] = _normal(g, b, hq, case["s"], d).to(torch.bfloat16)
    kv = []
    for _ in range(2):
        rows = torch.empty(b * per, hkv, page, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
        kv.append((rows, None) if kind == "bf16" else _quantised(rows))
    x["cache"] = [kv[0][0], kv[1][0], kv[0][1], kv[1][1]]
    return x


def _logits(case, g):
    n, v = case["n"], case["v"]
    if case["shifted"]:  # prompts of a batch: the logits of all but the last position, the tokens that follow them
        b = 8 if n % 8 == 0 else 1
        shape = (b, n // b + 1)
    else:
        shape = (n,)
    rows = math.prod(shape)
    logits = 2.5 * _normal(g, rows, v)
    tokens = torch.randint(0, v, (rows,), generator=g, device="cuda")
    sure = torch.rand(rows, generator=g, device="cuda") < 0.5  # half of the tokens are likely ones
    nxt = torch.roll(tokens, -1) if case["shifted"] else tokens
    logits[torch.arange(rows, device="cuda"), nxt] += 12.0 * sure
    if case["masked"]:
        keep = torch.rand(rows, v, generator=g, device="cuda") < 100.0 / v
        keep[torch.arange(rows, device="cuda"), nxt] = True
        logits.masked_fill_(~keep, -math.inf)
    logits = logits.to(DTYPES[case["kind"]]).view(*shape, v)
    tokens = tokens.view(shape)
    return {"logits": logits[:, :-1], "ids": tokens[:, 1:]} if case["shifted"] else {"logits": logits, "ids": tokens}


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return {"append": _run_append, "decode": _run_decode, "dense": _run_dense, "logprobs": _run_logprobs}[
        state["case"]["op"]](state)


def _bf(x):
    return x.to(torch.bfloat16).float()


def _norm_rope(x, gamma, cos, sin, style):
    """RMSNorm * gamma and rotate-half RoPE of rows x [B,H,S,D] with tables [B,1,S,D]; hf and legacy are the
    chains of bf16 roundings that the styles stand for, fp32 rounds once."""
    x, gamma = x.float(), gamma.float()
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    if style == "hf":
        n = _bf(_bf(x * inv) * gamma)
    else:
        n = x * inv * gamma
        n = _bf(n) if style == "legacy" else n
    if cos is None:
        return n.to(torch.bfloat16)
    half = x.shape[-1] // 2
    turned = torch.cat([-n[..., half:], n[..., :half]], dim=-1)
    p, r = n * cos.float(), turned * sin.float()
    return (p + r if style == "fp32" else _bf(p) + _bf(r)).to(torch.bfloat16)


def _run_append(x):
    case = x["case"]
    kc, vc, ks, vs = x["cache"]
    if own:
        import kernelfuser_amd as kf
        qn = kf.norm_rope_to_cache(x["q"], x["k"], x["v"], x["gq"], x["gk"], x["cos"], x["sin"], x["positions"],
                                   x["slots"], kc, vc, ks, vs, norm_style=case["style"])
    else:
        cos, sin = (None, None) if x["cos"] is None else (t[x["positions"]][:, None] for t in (x["cos"], x["sin"]))
        qn = _norm_rope(x["q"], x["gq"], cos, sin, case["style"])
        kn = _norm_rope(x["k"], x["gk"], cos, sin, case["style"])
        page, at = x["slots"] // case["page"], x["slots"] % case["page"]
        for rows, cache, scales in ((kn, kc, ks), (x["v"], vc, vs)):
            rows = rows.transpose(1, 2)  # [B,S,Hkv,D], as cache[page, :, at] takes them
            if scales is None:
                cache[page, :, at] = rows
            else:
                payload, e = _quantised(rows)
                cache.view(torch.uint8)[page, :, at] = payload.view(torch.uint8)
                scales.view(torch.uint8)[page, :, at] = e.view(torch.uint8)
    return {"qn": qn, "k": kc, "v": vc, "ks": ks, "vs": vs}


def _pages_dense(cache, scales, pages, l):
    """The pages of a batch as 32-bit rows [B,Hkv,L,D]."""
    b, per = pages.shape
    _, h, page, d = cache.shape
    pages = pages.long()
    rows = (cache[pages] if scales is None else cache.view(torch.uint8)[pages].view(cache.dtype)).float()
    if scales is not None:
        rows = rows * scales.view(torch.uint8)[pages].view(scales.dtype).float()[..., None]
    return rows.transpose(1, 2).reshape(b, h, per * page, d)[:, :, :l]


def _run_decode(x):
    case = x["case"]
    kc, vc, ks, vs = x["cache"]
    q = x["q"]
    window, cap = case["window"] or None, case["cap"] or None
    if own:
        import kernelfuser_amd as kf
        return kf.attention_decode(q, kc, vc, x["pages"], x["lengths"], ks, vs, window=window, softcap=cap)
    b, hq, s, d = q.shape
    l, hkv = case["l"], kc.shape[1]
    k, v = (_pages_dense(c, e, x["pages"], l) for c, e in ((kc, ks), (vc, vs)))
    qt = q.float().reshape(b, hkv, hq // hkv * s, d).transpose(-1, -2).contiguous()
    scores = torch.matmul(k, qt) * d ** -0.5  # [B,Hkv,L,rows]
    if cap:
        scores = cap * torch.tanh(scores / cap)
    j = torch.arange(l, device=q.device)[None, :, None]
    at = (x["lengths"].long()[:, None] - s + torch.arange(s, device=q.device))[:, None]  # the queries' positions
    seen = j <= at
    if window:
        seen = seen & (j > at - window)
    seen = seen[:, None].repeat(1, 1, 1, hq // hkv)
    scores = torch.where(seen, scores, -math.inf)
    m = scores.amax(-2, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-2, keepdim=True)
    p = p / torch.where(z == 0, 1.0, z)
    out = torch.matmul(p.transpose(-1, -2).contiguous(), v)
    return out.reshape(b, hq, s, d).to(torch.bfloat16)


def _run_dense(x):
    case = x["case"]
    kc, vc, ks, vs = x["cache"]
    if own:
        import kernelfuser_amd as kf
        return kf.cache_to_dense(kc, vc, x["pages"], x["lengths"], case["l"], ks, vs)
    held = torch.arange(case["l"], device=kc.device)[None, None, :, None] < x["lengths"].view(-1, 1, 1, 1)
    return tuple(torch.where(held, _pages_dense(c, e, x["pages"], case["l"]), 0.0).to(torch.bfloat16)
                 for c, e in ((kc, ks), (vc, vs)))


def _run_logprobs(x):
    top = x["case"]["top"]
    if own:
        import kernelfuser_amd as kf
        got = kf.token_logprobs(x["logits"], x["ids"], top)
        return tuple(got)[: 4 if top else 2]
    logits = x["logits"].float()
    v = logits.shape[-1]
    m = logits.amax(-1, keepdim=True)
    shifted = logits - m
    e = torch.exp(shifted)
    z = e.sum(-1)
    lse = torch.log(z)
    logp = torch.gather(shifted, -1, x["ids"][..., None])[..., 0] - lse
    entropy = lse - torch.where(e > 0, e * shifted, 0.0).sum(-1) / z
    if not top:
        return logp, entropy
    # the order of (value, lowest index) as one whole number: floats in order as their bits, -0 as 0
    bits = (logits + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = bits * (1 << 20) + (v - 1 - torch.arange(v, device=logits.device))
    best = torch.topk(key, top, dim=-1).values
    at = v - 1 - (best & ((1 << 20) - 1))
    return logp, entropy, torch.gather(shifted, -1, at) - lse[..., None], at


# ---------------------------------------------------------------------------
# Work and exact values
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        size = torch.empty(0, dtype=DTYPES[case["kind"]]).element_size()
        n, v, top = case["n"], case["v"], case["top"]
        return {"bytes": n * v * size + n * (8 + 4 + 4 + 12 * top), "flops": 7 * n * v}
    hq, hkv, d = HEADS[case["model"]]
    row = 2 * d if case["kind"] == "bf16" else d + 1  # bytes of a cached row
    if case["op"] == "append":
        t = case["b"] * case["s"]
        tables = 4 * d * case["s"] + 8 * t if case["rope"] else 0
        return {"bytes": t * (4 * hq * d + 4 * hkv * d + 2 * hkv * row + 8) + tables + 4 * d,
                "flops": 10 * t * (hq + hkv) * d}
    lens, b, l = _lengths(case), case["b"], case["l"]
    if case["op"] == "dense":
        return {"bytes": 2 * hkv * (sum(lens) * row + b * l * 2 * d), "flops": 2 * hkv * d * sum(lens)}
    s, window = case["s"], case["window"]
    keys = sum(min(n, window + s - 1) if window else n for n in lens)
    seen = sum(min(n - i, window) if window else n - i for n in lens for i in range(min(s, n)))
    return {"bytes": 2 * hkv * keys * row + 4 * b * hq * s * d, "flops": 4 * d * hq * seen}


def _chain64(x, gamma, cos, sin, style=None):
    """The prepared rows in 64 bits; with a style, its roundings too."""
    def r(t):
        return t.to(torch.bfloat16).double() if style in ("hf", "legacy") else t

    x, gamma = x.double(), gamma.double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    y = r(r(y) * gamma) if style == "hf" else r(y * gamma)
    if cos is None:
        return y
    a, b = y.chunk(2, dim=-1)
    (ca, cb), (sa, sb) = (t.double().chunk(2, dim=-1) for t in (cos, sin))
    return torch.cat([r(a * ca) - r(b * sa), r(b * cb) + r(a * sb)], dim=-1)


def exact(case, seed):
    x = _inputs(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "dense": _exact_dense, "logprobs": _exact_logprobs}[
        case["op"]](case, x)


def _exact_append(case, x):
    """No roundings but the one that sets a row's scale; a quantised row in units of its scale."""
    cos, sin = (None, None) if x["cos"] is None else (t[x["positions"]][:, None] for t in (x["cos"], x["sin"]))
    out = {"qn": _chain64(x["q"], x["gq"], cos, sin)}
    k = _chain64(x["k"], x["gk"], cos, sin)
    k_held = _chain64(x["k"], x["gk"], cos, sin, case["style"]).to(torch.bfloat16)
    page, at = x["slots"] // case["page"], x["slots"] % case["page"]
    for name, rows, held in (("k", k, k_held), ("v", x["v"].double(), x["v"])):
        cache = torch.zeros(x["cache"][0].shape, device="cuda", dtype=torch.float64)
        out[name + "s"] = None
        if case["kind"] != "bf16":
            largest = held.double().abs().amax(-1)
            scale = torch.exp2(torch.ceil(torch.log2(largest / 448)))
            scale = torch.where(scale < largest / 448, 2 * scale, scale)  # a logarithm next to a whole number
            scale = torch.where(scale / 2 >= largest / 448, scale / 2, scale)
            rows = rows / scale[..., None]
            scales = torch.full(cache.shape[:3], 2.0 ** -127, device="cuda", dtype=torch.float64)
            scales[page, :, at] = scale.transpose(1, 2)
            out[name + "s"] = scales
        cache[page, :, at] = rows.transpose(1, 2)
        out[name] = cache
    return out


def _held64(cache, scales, pages, n):
    """The first n rows of one sequence, [Hkv,n,D]."""
    page = cache.shape[2]
    at = pages[: -(-n // page)].long()
    rows = cache.view(torch.uint8 if scales is not None else cache.dtype)[at].view(cache.dtype).double()
    if scales is not None:
        rows = rows * scales.view(torch.uint8)[at].view(scales.dtype).double()[..., None]
    return rows.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def _exact_decode(case, x):
    kc, vc, ks, vs = x["cache"]
    q = x["q"].double()
    b, hq, s, d = q.shape
    g = hq // kc.shape[1]
    out = torch.zeros_like(q)
    for i, n in enumerate(_lengths(case)):
        if not n:
            continue
        k, v = (_held64(c, e, x["pages"][i], n) for c, e in ((kc, ks), (vc, vs)))
        for t in range(s):
            last = n - s + t
            first = max(0, last - case["window"] + 1) if case["window"] else 0
            if last < 0:
                continue
            qi = q[i, :, t].view(-1, g, d)
            z = torch.matmul(qi, k[:, first:last + 1].transpose(1, 2).contiguous()) / math.sqrt(d)
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            out[i, :, t] = torch.matmul(torch.softmax(z, dim=-1), v[:, first:last + 1].contiguous()).view(hq, d)
    return out


def _exact_dense(case, x):
    kc, vc, ks, vs = x["cache"]
    outs = []
    for c, e in ((kc, ks), (vc, vs)):
        out = torch.zeros(case["b"], c.shape[1], case["l"], c.shape[3], device="cuda", dtype=torch.float64)
        for i, n in enumerate(_lengths(case)):
            if n:
                out[i, :, :n] = _held64(c, e, x["pages"][i], n)
        outs.append(out)
    return tuple(outs)


def _exact_logprobs(case, x):
    logits, ids = x["logits"], x["ids"]
    lead, v = ids.shape, logits.shape[-1]
    logits, ids = logits.reshape(-1, v), ids.reshape(-1)
    rows = max(1, (1 << 26) // v)
    got = []
    for r in range(0, logits.shape[0], rows):
        logp = torch.log_softmax(logits[r:r + rows].double(), dim=-1)
        p = torch.exp(logp)
        h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
        one = [torch.gather(logp, 1, ids[r:r + rows, None])[:, 0], h]
        if case["top"]:
            order = torch.sort(logits[r:r + rows].double(), dim=-1, descending=True, stable=True).indices
            one += [torch.gather(logp, 1, order[:, : case["top"]]), order[:, : case["top"]]]
        got.append(one)
    return tuple(torch.cat(t).view(*lead, *t[0].shape[1:]) for t in zip(*got))
