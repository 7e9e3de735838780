"""What a step of several requests gives this library, as cases that can be timed and compared: attention over a prefix that
the requests share, low-rank adapters beside a projection, and drafted tokens checked against the model's logits.

Each case is one call of one operator.  ``run`` makes it in plain torch operations (``own`` false) or through ``llmops``
(``own`` true); ``exact`` evaluates the operator's definition in 64 bits.  Widths are those of the 7B-shape model that the
benchmark uses (hidden 4096, FFN 11008, 32 heads of 128, 55296 tokens) or generic.

Kinds:
  prefix   rotary + cache update + attention of ``tokens`` new tokens of each of ``batch`` sequences.  All sequences see the same
           ``prefix`` rows; behind them each has rows of its own, up to ``own`` with the new ones, as many as it has got so far.
           ``ragged``: sequences bring different numbers of new tokens, the rest is padding.  q, k and v are columns of one
           projection's output, as the projections leave them.
  lora     y + scale * (x A^T) B^T, the adapter (or none) chosen by sequence, beside a projection k -> n
  verify   ``drafts`` drafted tokens of each sequence against logits [batch, drafts + 1, vocab]; with the probabilities that
           the drafts were drawn from, or for drafts without any (a lookup in the text so far)
"""
import functools
import importlib
import math
import os
import sys

import torch

own = False

HIDDEN, FFN, HEADS, HEAD, VOCAB = 4096, 11008, 32, 128, 55296
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@functools.lru_cache(None)
def _llmops():
    sys.path.insert(0, os.path.abspath("llama.cl_amd"))
    return importlib.import_module("llmops")


def listed():
    return [
        # two chats that have just begun behind a short system prompt: latency
        {"name": "prefix_two_chats", "kind": "prefix", "batch": 2, "tokens": 1, "heads": 32, "kv_heads": 32, "prefix": 130, "own": 64,
         "half": False, "ragged": False},
        # a batch that generates in step behind a long system prompt, cache of halves
        {"name": "prefix_step32", "kind": "prefix", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 32, "prefix": 2048, "own": 512,
         "half": True, "ragged": False},
        # heads that share keys and values, a document that many requests ask about
        {"name": "prefix_step64_grouped", "kind": "prefix", "batch": 64, "tokens": 1, "heads": 32, "kv_heads": 8, "prefix": 4001, "own": 1000,
         "half": True, "ragged": False},
        # a step of drafted tokens, not as many for every sequence
        {"name": "prefix_drafts16", "kind": "prefix", "batch": 16, "tokens": 5, "heads": 32, "kv_heads": 32, "prefix": 1500, "own": 700,
         "half": False, "ragged": True},
        # the users' turns, a few hundred tokens each, read in one call
        {"name": "prefix_turns", "kind": "prefix", "batch": 4, "tokens": 300, "heads": 32, "kv_heads": 32, "prefix": 1000, "own": 777,
         "half": False, "ragged": True},
        # one request with an adapter of low rank
        {"name": "lora_one", "kind": "lora", "batch": 1, "tokens": 1, "n": HIDDEN, "k": HIDDEN, "rank": 8, "adapters": 1, "type": "fp16"},
        # a batch that generates in step, most requests with an adapter of their own
        {"name": "lora_step32", "kind": "lora", "batch": 32, "tokens": 1, "n": FFN, "k": HIDDEN, "rank": 16, "adapters": 20, "type": "bf16"},
        # drafted tokens, sizes that fill nothing
        {"name": "lora_drafts_ragged", "kind": "lora", "batch": 7, "tokens": 5, "n": 4090, "k": 4100, "rank": 10, "adapters": 4, "type": "fp32"},
        # prompts of a few requests
        {"name": "lora_prompts", "kind": "lora", "batch": 4, "tokens": 300, "n": HIDDEN, "k": FFN, "rank": 64, "adapters": 3, "type": "fp16"},
        # one request, four drafted tokens
        {"name": "verify_one", "kind": "verify", "batch": 1, "drafts": 4, "vocab": VOCAB, "probs": True},
        # a batch with drafts of a small model
        {"name": "verify_batch32", "kind": "verify", "batch": 32, "drafts": 4, "vocab": VOCAB, "probs": True},
        # drafts looked up in the text so far, a vocabulary of odd size
        {"name": "verify_lookup48", "kind": "verify", "batch": 48, "drafts": 7, "vocab": 32003, "probs": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "lora", "verify"])
    if kind == "prefix":
        while True:  # until no more rows are kept, and no more scores formed, than in the largest listed cases
            batch = _log(rng, 1, 64)
            tokens = _log(rng, 1, max(1, min(512, 1200 // batch)))
            case = {"kind": kind, "batch": batch, "tokens": tokens, "heads": 32, "kv_heads": rng.choice([32, 32, 8, 4]),
                    "prefix": rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 4096)]), "own": tokens + _log(rng, 1, 2048),
                    "half": rng.random() < 0.5, "ragged": rng.random() < 0.5}
            w = work(case)
            if w["bytes"] <= 2.3e8 and w["flops"] <= 1.9e10:
                return case
    if kind == "lora":
        batch = _log(rng, 1, 64)
        tokens = rng.choice([1, _log(rng, 1, max(1, 1200 // batch))])
        return {"kind": kind, "batch": batch, "tokens": tokens, "n": rng.choice([HIDDEN, FFN, _log(rng, 100, 11008)]),
                "k": rng.choice([HIDDEN, _log(rng, 100, 6000)]), "rank": rng.choice([4, 8, 16, 32, 64, _log(rng, 1, 64)]),
                "adapters": _log(rng, 1, 24), "type": rng.choice(["fp16", "bf16", "fp32"])}
    drafts = rng.choice([0, 1, 3, 5, 8])
    return {"kind": kind, "batch": _log(rng, 1, max(1, 300 // (drafts + 1))), "drafts": drafts, "vocab": rng.choice([VOCAB, _log(rng, 500, 60000)]),
            "probs": drafts > 0 and rng.random() < 0.5}


class _State:
    pass


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std


def _spread(gen, lo, hi, count):
    """whole numbers spread evenly over lo..hi, in an order of the generator's: their sum does not depend on it"""
    values = torch.linspace(lo, hi, count + 2, device="cuda", dtype=torch.float64)[1:-1].round().to(torch.int32)
    return values[torch.randperm(count, generator=gen, device="cuda")].contiguous()


def prepare(case, seed):
    gen, s = torch.Generator(device="cuda").manual_seed(seed), _State()
    s.case, kind, b = case, case["kind"], case["batch"]
    if kind == "prefix":
        t, h, hk, half = case["tokens"], case["heads"], case["kv_heads"], torch.float16 if case["half"] else torch.float32
        s.qkv = _normal(gen, b, t, (h + 2 * hk) * HEAD)
        s.inv_freq = 1.0 / (10000.0 ** (torch.arange(0, HEAD, 2, device="cuda").float() / HEAD))
        s.prefix_cache = _normal(gen, 2, 1, hk, max(1, case["prefix"]), HEAD).to(half)
        s.kv_cache = torch.zeros(2, b, hk, case["own"], HEAD, device="cuda", dtype=half)
        s.lengths = _spread(gen, 0, case["own"] - t, b)
        s.kv_cache.copy_(_normal(gen, *s.kv_cache.shape))
        s.q_lens = _spread(gen, max(1, t // 2), t, b) if case["ragged"] else None
    elif kind == "lora":
        dtype, n, k, r = TYPES[case["type"]], case["n"], case["k"], case["rank"]
        s.x, s.y = _normal(gen, b, case["tokens"], k), _normal(gen, b, case["tokens"], n)
        s.A = _normal(gen, case["adapters"], r, k, std=k ** -0.5).to(dtype)
        s.B = _normal(gen, case["adapters"], n, r, std=r ** -0.5).to(dtype)
        s.scales = torch.rand(case["adapters"], generator=gen, device="cuda") + 0.5
        s.adapters = torch.randint(0, case["adapters"], (b,), generator=gen, device="cuda", dtype=torch.int32)
        s.adapters[5::8] = -1  # (a request now and then runs the model as it is)
    else:
        k, v = case["drafts"], case["vocab"]
        s.logits = _normal(gen, b, k + 1, v, std=2.5)
        # a small model's distribution is the large one's, blurred: about two of three drafts are accepted
        s.probs = torch.softmax(s.logits[:, :k] + _normal(gen, b, k, v, std=0.7), dim=-1) if case["probs"] else None
        if case["probs"]:
            s.drafts = torch.multinomial(s.probs.reshape(b * k, v), 1, generator=gen).reshape(b, k)
        else:  # a lookup is often right: the likeliest token, which is then made likelier, or any
            best = s.logits[:, :k].argmax(-1)
            s.logits[:, :k].scatter_add_(2, best[..., None], torch.full((b, k, 1), 8.0, device="cuda"))
            s.drafts = torch.where(torch.rand(b, k, generator=gen, device="cuda") < 0.8, best, torch.randint(0, v, (b, k), generator=gen, device="cuda"))
        s.uniforms = torch.rand(b, k + 1, generator=gen, device="cuda")
        s.temperature = torch.tensor([1.0, 0.7, 0.0, 1.3], device="cuda").repeat(b // 4 + 1)[:b].contiguous()  # 0: the likeliest
        s.draft_lens = _spread(gen, k // 2, k, b) if k else None
    return s


def _qkv(s):
    h, hk = s.case["heads"] * HEAD, s.case["kv_heads"] * HEAD
    return s.qkv[..., :h], s.qkv[..., h:h + hk], s.qkv[..., h + hk:]


def run(s):
    kind = s.case["kind"]
    if own:
        if kind == "prefix":
            out = _llmops().attention_rope_prefix(*_qkv(s), s.inv_freq, s.prefix_cache, s.case["prefix"], s.kv_cache, s.lengths, 0, q_lens=s.q_lens)
            return [out, s.kv_cache]
        if kind == "lora":
            return _llmops().lora_add(s.y, s.x, s.A, s.B, s.adapters, s.scales)
        return _llmops().verify_drafts(s.logits, s.drafts, s.uniforms, draft_probs=s.probs, temperature=s.temperature, draft_lens=s.draft_lens)
    return {"prefix": _plain_prefix, "lora": _plain_lora, "verify": _plain_verify}[kind](s)


def _rotated(x, cos, sin):
    lo, hi = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)


def _plain_prefix(s):
    c = s.case
    b, t, h, hk, p, rows = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["prefix"], c["own"]
    q, k, v = (x.reshape(b, t, -1, HEAD) for x in _qkv(s))
    token = torch.arange(t, device="cuda")
    row = s.lengths[:, None] + token  # [b, t], inside the cache
    angle = (row + p).double()[..., None] * s.inv_freq.double()  # (far positions: 32 bits lose the angle)
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    live = token < s.q_lens[:, None] if s.q_lens is not None else torch.ones(b, t, dtype=torch.bool, device="cuda")
    at = (torch.arange(b, device="cuda")[:, None, None], torch.arange(hk, device="cuda")[None, None, :], row[:, :, None].long())
    for plane, new in ((0, k), (1, v)):
        cache = s.kv_cache[plane]
        cache[at] = torch.where(live[:, :, None, None], new.to(cache.dtype), cache[at])
    g = h // hk
    q = q.reshape(b, t, hk, g, HEAD).permute(2, 0, 1, 3, 4)  # [hk, b, t, g, d]
    flat = q.reshape(hk, b * t * g, HEAD)
    pk, pv = (s.prefix_cache[i, 0, :, :p].float() for i in (0, 1))
    ok, ov = (s.kv_cache[i].float().transpose(0, 1) for i in (0, 1))  # [hk, b, rows, d]
    common = torch.matmul(flat, pk.transpose(1, 2)).reshape(hk, b, t * g, p)
    apart = torch.matmul(q.reshape(hk, b, t * g, HEAD), ok.transpose(2, 3))
    seen = (torch.arange(rows, device="cuda") <= row[..., None])[:, :, None].expand(b, t, g, rows).reshape(b, t * g, rows)
    scores = torch.cat((common, apart.masked_fill(~seen, -math.inf)), dim=-1) * HEAD ** -0.5
    e = (scores - scores.amax(-1, keepdim=True)).exp()
    e_p, e_o, total = e[..., :p], e[..., p:], e.sum(-1, keepdim=True)
    # (rows past a sequence's own hold whatever they hold, and count for nothing)
    out = torch.matmul(e_p.reshape(hk, b * t * g, p), pv).reshape(hk, b, t * g, HEAD) + torch.matmul(e_o, ov)
    out = (out / total).reshape(hk, b, t, g, HEAD).permute(1, 2, 0, 3, 4).reshape(b, t, h * HEAD)
    return [torch.where(live[..., None], out, 0.0), s.kv_cache]


def _plain_lora(s):
    pick = s.adapters.clamp(min=0).long()
    scale = torch.where(s.adapters >= 0, s.scales[pick], 0.0)[:, None, None]
    inner = torch.matmul(s.x, s.A[pick].float().transpose(1, 2))
    return s.y + scale * torch.matmul(inner, s.B[pick].float().transpose(1, 2))


def _plain_verify(s):
    # 64 bits: an answer is a whole number, and 32 bits misplace the borders between tokens
    b, k, v = s.case["batch"], s.case["drafts"], s.case["vocab"]
    z, u = s.logits.double(), s.uniforms.double()
    n = s.draft_lens.long() if s.draft_lens is not None else torch.full((b,), k, device="cuda")
    greedy, t = s.temperature == 0, torch.where(s.temperature == 0, 1.0, s.temperature).double()
    w = ((z - z.amax(-1, keepdim=True)) / t[:, None, None]).exp()
    p = w / w.sum(-1, keepdim=True)
    best = z.argmax(-1)
    place = torch.arange(k, device="cuda")
    drawn = s.drafts[..., None]
    q_of = s.probs.double().gather(2, drawn)[..., 0] if s.probs is not None else torch.ones(b, k, device="cuda", dtype=torch.float64)
    fine = u[:, :k] * q_of < p[:, :k].gather(2, drawn)[..., 0]
    fine = torch.where(greedy[:, None], s.drafts == best[:, :k], fine) & (place < n[:, None])
    accepted = fine.long().cumprod(1).sum(1)
    row = p.gather(1, accepted[:, None, None].expand(b, 1, v))[:, 0]
    all_of = accepted == n
    if k:
        i = accepted.clamp(max=k - 1)
        if s.probs is not None:
            q = s.probs.gather(1, i[:, None, None].expand(b, 1, v))[:, 0].double()
        else:
            q = torch.zeros(b, v, device="cuda", dtype=torch.float64).scatter_(1, s.drafts.gather(1, i[:, None]), 1.0)
        row = torch.where(all_of[:, None], row, (row - q).clamp(min=0))
    sums = row.cumsum(-1)
    sample = (sums <= (u[:, k] * sums[:, -1])[:, None]).sum(-1).clamp(max=v - 1)
    sample = torch.where(greedy, best.gather(1, accepted[:, None])[:, 0], sample)
    place = torch.arange(k + 1, device="cuda")
    tokens = torch.cat((s.drafts, torch.full((b, 1), -1, device="cuda")), dim=1)
    tokens = torch.where(place < accepted[:, None], tokens, -1)
    return torch.where(place == accepted[:, None], sample[:, None], tokens), accepted.to(torch.int32)


def work(case):
    kind, b = case["kind"], case["batch"]
    if kind == "prefix":
        t, h, hk, p, e = case["tokens"], case["heads"], case["kv_heads"], case["prefix"], 2 if case["half"] else 4
        mean = (case["own"] - t) / 2  # rows that a sequence has so far
        new = t * (0.75 if case["ragged"] and t > 1 else 1.0)
        return {"bytes": 4 * HEAD * b * (t * h + new * (h + 2 * hk)) + 2 * hk * HEAD * e * (p + b * (mean + new)),
                "flops": 4 * HEAD * h * b * new * (p + mean + (new + 1) / 2)}
    if kind == "lora":
        rows, e = b * case["tokens"], 4 if case["type"] == "fp32" else 2
        used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** b)  # adapters that come up, on average
        return {"bytes": 4 * rows * (case["k"] + 2 * case["n"]) + used * case["rank"] * e * (case["k"] + case["n"]),
                "flops": 2 * rows * case["rank"] * (case["k"] + case["n"])}
    k, v = case["drafts"], case["vocab"]
    return {"bytes": 4 * b * v * (k + 1 + (1 if case["probs"] else 0)), "flops": 4 * b * v * (k + 2)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"prefix": _exact_prefix, "lora": _exact_lora, "verify": _exact_verify}[case["kind"]](s)


def _exact_prefix(s):
    c, f64 = s.case, torch.float64
    h, hk, p = c["heads"], c["kv_heads"], c["prefix"]
    out = torch.zeros(c["batch"], c["tokens"], h, HEAD, dtype=f64, device="cuda")
    cache = s.kv_cache.to(f64)
    for b in range(c["batch"]):
        n, past = int(s.q_lens[b]) if s.q_lens is not None else c["tokens"], int(s.lengths[b])
        # a pair of dimensions as a complex number, turned by the angle of its position
        turn = torch.polar(torch.ones(n, HEAD // 2, dtype=f64, device="cuda"),
                           torch.outer(torch.arange(p + past, p + past + n, dtype=f64, device="cuda"), s.inv_freq.to(f64)))[:, None]
        q, k, v = (x[b, :n].to(f64).reshape(n, -1, 2, HEAD // 2) for x in _qkv(s))
        q, k = (torch.complex(x[:, :, 0], x[:, :, 1]) * turn for x in (q, k))
        q, k = (torch.cat((x.real, x.imag), dim=-1) for x in (q, k))
        for plane, new in ((0, k), (1, v.reshape(n, hk, HEAD))):
            cache[plane, b, :, past:past + n] = new.transpose(0, 1).to(s.kv_cache.dtype).to(f64) if c["half"] else new.transpose(0, 1)
        for head in range(hk):
            keys, values = (torch.cat((s.prefix_cache[i, 0, head, :p].to(f64), cache[i, b, head, :past + n])) for i in (0, 1))
            mine = slice(head * (h // hk), (head + 1) * (h // hk))
            scores = torch.einsum("lgd,rd->lgr", q[:, mine], keys) / math.sqrt(HEAD)
            hidden = torch.arange(p + past + n, device="cuda")[None, :] > p + past + torch.arange(n, device="cuda")[:, None]
            out[b, :n, mine] = torch.einsum("lgr,rd->lgd", torch.softmax(scores.masked_fill(hidden[:, None], -math.inf), dim=-1), values)
    return [out.reshape(c["batch"], c["tokens"], h * HEAD), cache]


def _exact_lora(s):
    y = s.y.double()
    for b, a in enumerate(s.adapters.tolist()):
        if a >= 0:
            y[b] += s.scales[a].double() * (s.x[b].double() @ s.A[a].double().T @ s.B[a].double().T)
    return y


def _exact_verify(s):
    k, tokens, accepted = s.case["drafts"], [], []
    for b in range(s.case["batch"]):
        n, t = int(s.draft_lens[b]) if s.draft_lens is not None else k, float(s.temperature[b])
        line, i = [], 0
        while True:
            z = s.logits[b, i].double()
            p = torch.softmax(z / t, dim=0) if t else torch.nn.functional.one_hot(z.argmax(), z.numel()).double()
            if i == n:
                break
            x = int(s.drafts[b, i])
            q = s.probs[b, i].double() if s.probs is not None else torch.nn.functional.one_hot(s.drafts[b, i], z.numel()).double()
            if not (p[x] > 0.5 if not t else float(s.uniforms[b, i]) * q[x] < p[x]):
                p = torch.relu(p - q) if t else p
                break
            line.append(x)
            i += 1
        sums = torch.cumsum(p, 0)
        line.append(int(torch.searchsorted(sums, sums[-1] * float(s.uniforms[b, k]), right=True).clamp(max=z.numel() - 1)))
        accepted.append(i)
        tokens.append(line + [-1] * (k + 1 - len(line)))
    return torch.tensor(tokens, device="cuda"), torch.tensor(accepted, dtype=torch.int32, device="cuda")
