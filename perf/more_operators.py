"""What long chats give this library where memory is short, as cases that can be timed and compared: a key/value cache that is held in
4 bits, the attention that reads it, and the log probabilities that tell what a text is worth to the model (and what the smaller cache
costs it).

Each case is a pass through one operator.  ``run`` makes it in plain torch operations (``own`` false) or through ``llmops``
(``own`` true); ``exact`` evaluates the operator's definition in 64 bits.  Widths are those of the 7B-shape model that the
benchmark uses (32 heads of 128, 55296 tokens) or generic.

A row of the cache holds 128 values as 80 bytes, four groups of 32 values x one behind the other.  With u the smallest power of two from
2^-24 on for which max |x| <= 2032 u, lo = round(min x / u), hi = round(max x / u) and s = ceil((hi - lo) / 15), a group is the halves
d = s u and m = lo u and for each value the code round((x / u - lo) / s), 0 to 15 (rounding to even); it stands for d code + m, which is a
half.  16 bytes of codes for each group, then four pairs (d, m).  Eight codes lie in a word of 32 bits, code i at bit 4 (i / 2) + 16 (i % 2).

Kinds:
  attention  rotary + cache update + attention of ``tokens`` new tokens of each of ``batch`` sequences over caches of up to ``own`` rows,
             of which each sequence has got some so far.  ``ragged``: sequences bring different numbers of new tokens, the rest is
             padding.  q, k and v are columns of one projection's output.  The rows that the call has written are read back.
  cache      rows quantised as they are written, and the cache read back: new tokens' k (rotated) and v as columns of a projection's
             output, or (``rotate`` false) rows of a cache in full width that every sequence begins with
  logprobs   of given tokens against logits [batch, tokens, vocab], with the entropy and the ``top`` likeliest tokens.  ``shift``: a
             text's own tokens, each against the logits of the token before it
"""
import functools
import importlib
import math
import os
import sys

import torch

own = False

HEADS, HEAD, VOCAB = 32, 128, 55296
GROUP, ROW_BYTES = 32, 80
TYPES = {"fp32": torch.float32, "fp16": torch.float16}


@functools.lru_cache(None)
def _llmops():
    sys.path.insert(0, os.path.abspath("llama.cl_amd"))
    return importlib.import_module("llmops")


def listed():
    return [
        # two chats that have just begun: latency
        {"name": "q4_two_chats", "kind": "attention", "batch": 2, "tokens": 1, "heads": 32, "kv_heads": 32, "own": 200, "ragged": False},
        # a batch that generates in step, from chats that begin to chats of 4000 tokens
        {"name": "q4_step32", "kind": "attention", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 32, "own": 4096, "ragged": False},
        # heads that share keys and values, more and longer chats
        {"name": "q4_step64_grouped", "kind": "attention", "batch": 64, "tokens": 1, "heads": 32, "kv_heads": 8, "own": 8000, "ragged": False},
        # one chat about a long document
        {"name": "q4_long_one", "kind": "attention", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "own": 100001, "ragged": False},
        # a step of drafted tokens, not as many for every sequence
        {"name": "q4_drafts16", "kind": "attention", "batch": 16, "tokens": 5, "heads": 32, "kv_heads": 32, "own": 2200, "ragged": True},
        # the users' turns, a few hundred tokens each, read in one call
        {"name": "q4_turns", "kind": "attention", "batch": 4, "tokens": 300, "heads": 32, "kv_heads": 32, "own": 1777, "ragged": True},
        # one token's rows: latency
        {"name": "cache_one", "kind": "cache", "batch": 1, "tokens": 1, "kv_heads": 32, "own": 1, "type": "fp32", "rotate": True, "ragged": False},
        # turns of a few requests, not as long for every one, behind what is there
        {"name": "cache_turns", "kind": "cache", "batch": 5, "tokens": 77, "kv_heads": 8, "own": 301, "type": "fp32", "rotate": True, "ragged": True},
        # a system prompt that was read once, in halves, becomes the beginning of eight chats
        {"name": "cache_prefix", "kind": "cache", "batch": 8, "tokens": 2048, "kv_heads": 32, "own": 2048, "type": "fp16", "rotate": False, "ragged": False},
        # the token that one chat has drawn, with a few alternatives
        {"name": "logprobs_one", "kind": "logprobs", "batch": 1, "tokens": 1, "vocab": VOCAB, "top": 5, "shift": False},
        # a batch's drafted and drawn tokens, with as many alternatives as clients may ask for
        {"name": "logprobs_step32", "kind": "logprobs", "batch": 32, "tokens": 5, "vocab": VOCAB, "top": 20, "shift": False},
        # texts that are scored (perplexity), a vocabulary of odd size
        {"name": "logprobs_texts", "kind": "logprobs", "batch": 3, "tokens": 700, "vocab": 32003, "top": 0, "shift": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "cache", "logprobs"])
    while True:  # until it costs no more than the largest listed cases
        if kind == "attention":
            batch = _log(rng, 1, 64)
            tokens = rng.choice([1, _log(rng, 1, max(1, min(512, 1200 // batch)))])
            case = {"kind": kind, "batch": batch, "tokens": tokens, "heads": 32, "kv_heads": rng.choice([32, 32, 8, 4]),
                    "own": tokens + _log(rng, 1, 100000), "ragged": rng.random() < 0.5}
            if work(case)["bytes"] <= 3.3e8 and work(case)["flops"] <= 1.2e10 and case["own"] * batch * case["kv_heads"] <= 4.2e6:
                return case
        elif kind == "cache":
            batch, rotate = _log(rng, 1, 64), rng.random() < 0.6
            tokens = _log(rng, 1, 2048)
            case = {"kind": kind, "batch": batch, "tokens": tokens, "kv_heads": rng.choice([32, 8, 4]), "own": tokens + _log(rng, 1, 1000) - 1,
                    "type": "fp32" if rotate else rng.choice(["fp16", "fp32"]), "rotate": rotate, "ragged": rng.random() < 0.5}
            if work(case)["bytes"] <= 3.6e8:
                return case
        else:
            case = {"kind": kind, "batch": _log(rng, 1, 64), "tokens": _log(rng, 1, 700), "vocab": rng.choice([VOCAB, _log(rng, 500, 60000)]),
                    "top": rng.choice([0, 1, 5, 20, rng.randint(1, 32)]), "shift": rng.random() < 0.5}
            if work(case)["bytes"] <= 2.6e8:
                return case


class _State:
    pass


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std


def _spread(gen, lo, hi, count):
    """whole numbers spread evenly over lo..hi, in an order of the generator's: their sum does not depend on it"""
    values = torch.linspace(lo, hi, count + 2, device="cuda", dtype=torch.float64)[1:-1].round().to(torch.int32)
    return values[torch.randperm(count, generator=gen, device="cuda")].contiguous()


def _lens(gen, case):
    t = case["tokens"]
    return _spread(gen, max(1, t // 2), t, case["batch"]) if case["ragged"] else None


def prepare(case, seed):
    gen, s = torch.Generator(device="cuda").manual_seed(seed), _State()
    s.case, kind, b, t = case, case["kind"], case["batch"], case["tokens"]
    if kind == "logprobs":
        s.logits = _normal(gen, b, t + 1 if case["shift"] else t, case["vocab"], std=2.5)
        # a text's tokens are often the likeliest, and sometimes anything
        best = s.logits[:, :t].argmax(-1)
        ids = torch.where(torch.rand(b, t, generator=gen, device="cuda") < 0.6, best, torch.randint(0, case["vocab"], (b, t), generator=gen, device="cuda"))
        s.ids = torch.cat((torch.zeros_like(ids[:, :1]), ids), dim=1) if case["shift"] else ids
        return s
    hk = case["kv_heads"]
    width = _normal(gen, 2, hk, HEAD, std=0.5).exp()  # (a model's channels differ in their spread)
    s.lengths, s.q_lens = _spread(gen, 0, case["own"] - t, b), _lens(gen, case)
    s.inv_freq = 1.0 / (10000.0 ** (torch.arange(0, HEAD, 2, device="cuda").float() / HEAD))
    s.cache = torch.zeros(2, b, hk, case["own"], ROW_BYTES, device="cuda", dtype=torch.int8)
    if kind == "attention":
        h = case["heads"]
        s.qkv = _normal(gen, b, t, (h + 2 * hk) * HEAD)
        s.qkv[..., h * HEAD:] *= width.reshape(-1)
        for plane in range(2):
            for row in range(b):
                s.cache[plane, row] = _packed(*_quantised(_normal(gen, hk, case["own"], HEAD) * width[plane][:, None]))
    elif case["rotate"]:
        s.kv = _normal(gen, b, t, 2 * hk * HEAD) * width.reshape(-1)
    else:
        s.full = (_normal(gen, 2, 1, hk, t, HEAD) * width[:, None, :, None]).to(TYPES[case["type"]])
    return s


def _new_rows(s):
    """k and v, as the operators take them"""
    c = s.case
    hk = c["kv_heads"] * HEAD
    if c["kind"] == "attention":
        h = c["heads"] * HEAD
        return s.qkv[..., h:h + hk], s.qkv[..., h + hk:]
    if c["rotate"]:
        return s.kv[..., :hk], s.kv[..., hk:]
    return tuple(s.full[i].transpose(1, 2).expand(c["batch"], -1, -1, -1) for i in (0, 1))  # [batch, tokens, heads, 128]


def run(s):
    c, kind = s.case, s.case["kind"]
    if kind == "logprobs":
        logits, ids = (s.logits[:, :-1], s.ids[:, 1:]) if c["shift"] else (s.logits, s.ids)
        return _llmops().token_logprobs(logits, ids, c["top"]) if own else _plain_logprobs(logits, ids, c["top"])
    k, v = _new_rows(s)
    if kind == "cache":
        if not own:
            _plain_write(s, k, v, c["rotate"])
            return _unpacked(s.cache).to(torch.float16)
        _llmops().cache_write_q4(k, v, s.cache, s.lengths, 0, inv_freq=s.inv_freq if c["rotate"] else None, q_lens=s.q_lens)
        return _llmops().cache_read_q4(s.cache, c["own"])
    q = s.qkv[..., :c["heads"] * HEAD]
    if not own:
        return _plain_attention(s, q, k, v)
    out = _llmops().attention_rope_q4(q, k, v, s.inv_freq, s.cache, s.lengths, 0, q_lens=s.q_lens)
    return [out, _llmops().cache_read_q4(s.cache, c["tokens"], starts=s.lengths)]


# ---- plain forms ----
def _quantised(x):
    """x [..., 128] (64 bits where codes have to be right at the borders): codes, d and m of its groups"""
    x = x.unflatten(-1, (HEAD // GROUP, GROUP))
    fraction, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    exponent = torch.where(fraction > 2032 / 2048, exponent + 1, exponent).clamp(min=11 - 24)
    t = x * _power(11 - exponent).to(x.dtype)  # x / u
    lo, hi = t.amin(-1, keepdim=True).round(), t.amax(-1, keepdim=True).round()
    step = ((hi - lo) / 15).ceil()
    codes = ((t - lo) / step.clamp(min=1)).round().clamp(0, 15)
    u = _power(exponent - 11).to(x.dtype)
    return codes.to(torch.int32), (step * u).to(torch.float16), (lo * u).to(torch.float16)


def _power(e):
    """2^e, exactly"""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _shifts():
    i = torch.arange(8, device="cuda", dtype=torch.int32)
    return (i // 2) * 4 + (i % 2) * 16


def _packed(codes, d, m):
    words = (codes.unflatten(-1, (4, 8)) << _shifts()).sum(-1, dtype=torch.int32)  # [..., 4 groups, 4 words]
    pairs = torch.stack((d[..., 0], m[..., 0]), dim=-1)
    return torch.cat((words.flatten(-2).view(torch.int8), pairs.flatten(-2).view(torch.int8)), dim=-1)


def _unpacked(rows):
    """the values that rows [..., 80] stand for, fp32 [..., 128]"""
    words, pairs = rows.view(torch.int32)[..., :16], rows.view(torch.float16)[..., 32:].unflatten(-1, (4, 2)).float()
    codes = (words[..., None] >> _shifts()) & 15
    return (codes.unflatten(-2, (4, 4)).flatten(-2) * pairs[..., :1] + pairs[..., 1:]).flatten(-2)


def _angles(s):
    row = s.lengths[:, None] + torch.arange(s.case["tokens"], device="cuda")  # [batch, tokens], inside the cache
    angle = row.double()[..., None] * s.inv_freq.double()
    return row, angle.cos()[:, :, None], angle.sin()[:, :, None]


def _rotated(x, cos, sin):
    lo, hi = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)


def _live(s):
    c = s.case
    if s.q_lens is None:
        return torch.ones(c["batch"], c["tokens"], dtype=torch.bool, device="cuda")
    return torch.arange(c["tokens"], device="cuda") < s.q_lens[:, None]


def _plain_write(s, k, v, rotate):
    b, t, hk = s.case["batch"], s.case["tokens"], s.case["kv_heads"]
    row, cos, sin = _angles(s)
    at = (torch.arange(b, device="cuda")[:, None, None], torch.arange(hk, device="cuda")[None, None, :], row[:, :, None].long())
    k, v = k.reshape(b, t, hk, HEAD).double(), v.reshape(b, t, hk, HEAD).double()
    live = _live(s)[:, :, None, None]
    for plane, new in ((0, _rotated(k, cos, sin) if rotate else k), (1, v)):
        s.cache[plane][at] = torch.where(live, _packed(*_quantised(new)), s.cache[plane][at])


def _plain_attention(s, q, k, v):
    c = s.case
    b, t, h, hk, rows = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["own"]
    _plain_write(s, k, v, True)
    row, cos, sin = _angles(s)
    q = _rotated(q.reshape(b, t, h, HEAD), cos.float(), sin.float())
    g = h // hk
    q = q.reshape(b, t, hk, g, HEAD).permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, HEAD)
    keys, values = _unpacked(s.cache[0]), _unpacked(s.cache[1])  # [b, hk, rows, d]
    scores = torch.matmul(q, keys.transpose(2, 3)) * HEAD ** -0.5
    seen = (torch.arange(rows, device="cuda") <= row[..., None])[:, :, None].expand(b, t, g, rows).reshape(b, 1, t * g, rows)
    scores = scores.masked_fill(~seen, -math.inf)
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    out = torch.matmul(e, values) / e.sum(-1, keepdim=True)
    out = out.reshape(b, hk, t, g, HEAD).permute(0, 2, 1, 3, 4).reshape(b, t, h * HEAD)
    at = (torch.arange(2, device="cuda")[:, None, None, None], torch.arange(b, device="cuda")[None, :, None, None],
          torch.arange(hk, device="cuda")[None, None, :, None], row[None, :, None, :].long())
    return [torch.where(_live(s)[..., None], out, 0.0), _unpacked(s.cache[at]).to(torch.float16)]


def _plain_logprobs(logits, ids, top):
    z = logits - logits.amax(-1, keepdim=True)
    z = z - z.exp().sum(-1, keepdim=True).log()  # log probabilities
    entropy = -(z.exp() * z).sum(-1)
    order = logits.sort(dim=-1, descending=True, stable=True).indices[..., :top] if top else ids.new_empty(ids.shape + (0,))
    return z.gather(-1, ids[..., None])[..., 0], entropy, order, z.gather(-1, order)


def work(case):
    kind, b, t = case["kind"], case["batch"], case["tokens"]
    if kind == "logprobs":
        rows = b * t
        return {"bytes": rows * (4 * case["vocab"] + 8 + 8 + 12 * case["top"]), "flops": 4 * rows * case["vocab"]}
    hk = case["kv_heads"]
    new = b * t * (0.75 if case["ragged"] and t > 1 else 1.0)
    if kind == "cache":
        source = 2 * hk * HEAD * (4 * new if case["rotate"] else (2 if case["type"] == "fp16" else 4) * t)
        kept = b * case["own"] - new  # rows that the call did not write are read
        return {"bytes": source + 2 * hk * ROW_BYTES * (new + kept) + 4 * hk * HEAD * b * case["own"], "flops": 12 * hk * HEAD * new}
    h, mean = case["heads"], (case["own"] - t) / 2  # rows that a sequence has so far
    # (the rows that were written are returned as halves, padding's included)
    return {"bytes": 4 * HEAD * (b * t * h + new * (h + 2 * hk)) + 2 * hk * ROW_BYTES * (b * mean + new) + 4 * hk * HEAD * b * t,
            "flops": 4 * HEAD * h * new * (mean + (new / b + 1) / 2)}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(s)
    cache = _exact_values(s.cache)
    k, v = (x.to(torch.float64).reshape(case["batch"], case["tokens"], case["kv_heads"], HEAD) for x in _new_rows(s))
    q = s.qkv[..., :case["heads"] * HEAD].to(torch.float64).unflatten(-1, (-1, HEAD)) if case["kind"] == "attention" else None
    out = torch.zeros_like(q) if q is not None else None
    for b in range(case["batch"]):
        n, past = int(s.q_lens[b]) if s.q_lens is not None else case["tokens"], int(s.lengths[b])
        # a pair of dimensions as a complex number, turned by the angle of its position
        turn = torch.polar(torch.ones(n, HEAD // 2, dtype=torch.float64, device="cuda"),
                           torch.outer(torch.arange(past, past + n, dtype=torch.float64, device="cuda"), s.inv_freq.to(torch.float64)))[:, None]
        keys = _turned(k[b, :n], turn) if case.get("rotate", True) else k[b, :n]
        for plane, new in ((0, keys), (1, v[b, :n])):
            cache[plane, b, :, past:past + n] = _nearest(new).transpose(0, 1)
        if q is None:
            continue
        hk, g = case["kv_heads"], case["heads"] // case["kv_heads"]
        turned = _turned(q[b, :n], turn)
        hidden = torch.arange(past + n, device="cuda")[None, :] > past + torch.arange(n, device="cuda")[:, None]
        for head in range(hk):
            mine = slice(head * g, (head + 1) * g)
            scores = torch.einsum("lgd,rd->lgr", turned[:, mine], cache[0, b, head, :past + n]) / math.sqrt(HEAD)
            weights = torch.softmax(scores.masked_fill(hidden[:, None], -math.inf), dim=-1)
            out[b, :n, mine] = torch.einsum("lgr,rd->lgd", weights, cache[1, b, head, :past + n])
    if q is None:
        return cache
    t = case["tokens"]
    written = torch.stack([cache[:, b, :, int(s.lengths[b]):int(s.lengths[b]) + t] for b in range(case["batch"])], dim=1)
    return [out.flatten(-2), written]


def _turned(x, turn):
    z = torch.complex(x[..., :HEAD // 2], x[..., HEAD // 2:]) * turn
    return torch.cat((z.real, z.imag), dim=-1)


def _nearest(x):
    """the values that the codes of x stand for: the level of each group that is nearest, the even one of two"""
    x = x.unflatten(-1, (4, GROUP))
    u = torch.full_like(x[..., :1], 2.0 ** -24)
    while bool((x.abs().amax(-1, keepdim=True) > 2032 * u).any()):
        u = torch.where(x.abs().amax(-1, keepdim=True) > 2032 * u, 2 * u, u)
    t = x / u
    lo, hi = torch.round(t.min(-1, keepdim=True).values), torch.round(t.max(-1, keepdim=True).values)
    step = torch.floor((hi - lo + 14) / 15)
    code = torch.zeros_like(t)
    for j in range(15):  # past the middle between levels j and j + 1, or on it with j odd
        middle = (j + 0.5) * step
        code += ((t - lo > middle) | ((t - lo == middle) & (j % 2 == 1))) & (step > 0)
    return ((lo + step * code) * u).flatten(-2)


def _exact_values(rows):
    halves = rows[..., 64:].contiguous().view(torch.float16).to(torch.float64)
    out = torch.empty(rows.shape[:-1] + (HEAD,), dtype=torch.float64, device="cuda")
    for at in range(HEAD):
        group, word, i = at // 32, at // 8, at % 8
        byte = rows[..., 4 * word + (i // 2) // 2 + 2 * (i % 2)].to(torch.int16) & 255
        code = (byte // 16 if (i // 2) % 2 else byte % 16).to(torch.float64)
        out[..., at] = halves[..., 2 * group] * code + halves[..., 2 * group + 1]
    return out


def _exact_logprobs(s):
    logits, ids = (s.logits[:, :-1], s.ids[:, 1:]) if s.case["shift"] else (s.logits, s.ids)
    parts = []
    for z32, line in zip(logits.flatten(0, 1).split(64), ids.flatten().split(64)):
        z = z32.to(torch.float64)
        log_p = z - torch.logsumexp(z, dim=1, keepdim=True)
        p = torch.softmax(z, dim=1)
        left, places, place = z32.clone(), [], torch.arange(z.shape[1], device="cuda")
        for _ in range(s.case["top"]):
            first = torch.where(left == left.max(dim=1, keepdim=True).values, place, z.shape[1]).min(dim=1, keepdim=True).values
            places.append(first)
            left.scatter_(1, first, -math.inf)
        places = torch.cat(places, dim=1) if places else line.new_empty(len(line), 0)
        parts.append((log_p[torch.arange(len(line), device="cuda"), line], -torch.special.xlogy(p, p).sum(1), places, log_p.gather(1, places)))
    return tuple(torch.cat(x).unflatten(0, tuple(ids.shape)) for x in zip(*parts))
