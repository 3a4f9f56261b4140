"""The operators of caches that hold less, as cases that can be timed and checked: keys and values in 4 bits, and caches that tokens leave.

A cache holds less when its numbers take fewer bits, and when the tokens that nobody attends to leave it:

* ``write``: the rows of new tokens are rounded to 4 bits into the paged cache (``ops.kv4_write``) and pages are read back
  (``ops.kv4_unpack``);
* ``attention``: decoded tokens and prompt portions attend over the cache in 4 bits (``ops.kv4_attention``);
* ``weights``: what every cached key got of the softmax of given queries is added to a running sum beside the key (``ops.key_weights``),
  for a cache in 4 bits behind the attention of the same step, or for a plain cache and the last tokens of a prompt;
* ``evict``: of every key/value head, the keys with the largest sums stay, the first and the last ones among them, and move to the front of
  the request's pages (``ops.cache_evict``).

The format: the head's numbers lie in groups of 32.  A group has a scale, a number with 5 bits of exponent and 3 of mantissa (the upper byte
behind the sign of a 16-bit float), the nearest one to the group's largest magnitude / 7, at most 61,440; a number is the nearest whole multiple of the
scale between -7 and 7, stored plus 8; halves go to the even one.  A group with a number that is not finite has the scale 255 and reads as NaN.
A page of a head is ``page_size`` rows of ``d / 2`` bytes, then ``page_size`` rows of ``d / 32`` scales.  Keys lie in words of 8 numbers: word ``t * (d / 32) +
j`` of a row is numbers ``32 j + 8 t ..``, the first in the lowest bits; values in half words of 4: half word ``g * (d / 32) + j`` is numbers ``32 j + 4 g ..``.
"""
from __future__ import annotations

import json
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

#: query heads, key/value heads, head size, layers: the Llama models that the benchmarks run, and heads without groups
HEADS = {"llama-3.2-1b": (32, 8, 64, 16), "llama-3.2-3b": (24, 8, 128, 28), "llama-3.1-8b": (32, 8, 128, 32),
         "ungrouped": (16, 16, 64, 16)}


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # one decoded token of a small model: the latency of a call
        {"name": "write_token", "kind": "write", "shape": "llama-3.2-1b", "tokens": 1, "page": 16, "dtype": "bf16"},
        # a long prompt portion, an odd number of tokens
        {"name": "write_prompt", "kind": "write", "shape": "llama-3.1-8b", "tokens": 8191, "page": 16, "dtype": "bf16"},
        # one user's next token behind a short conversation: the latency of a call
        {"name": "attention_one", "kind": "attention", "shape": "llama-3.2-1b", "requests": 1, "tokens": 1, "context": 640,
         "ragged": False, "page": 16, "dtype": "bf16"},
        # two very long documents: few rows, very many keys
        {"name": "attention_long", "kind": "attention", "shape": "llama-3.1-8b", "requests": 2, "tokens": 1, "context": 100003,
         "ragged": False, "page": 16, "dtype": "bf16"},
        # a full batch: the largest pass over cached keys
        {"name": "attention_batch_64", "kind": "attention", "shape": "llama-3.2-3b", "requests": 64, "tokens": 1, "context": 6000,
         "ragged": True, "page": 32, "dtype": "bf16"},
        # layers with a window, a score beside the keys and bounded scores; a few tokens a request
        {"name": "attention_window", "kind": "attention", "shape": "llama-3.2-1b", "requests": 8, "tokens": 3, "context": 2500,
         "ragged": True, "page": 16, "window": 1024, "sink": True, "softcap": 30.0, "dtype": "bf16"},
        # a prompt portion behind what is cached already
        {"name": "attention_prompt", "kind": "attention", "shape": "llama-3.1-8b", "requests": 1, "tokens": 2048, "context": 6144,
         "ragged": False, "page": 16, "dtype": "bf16"},
        # the true 32-bit run
        {"name": "attention_f32", "kind": "attention", "shape": "llama-3.2-1b", "requests": 4, "tokens": 1, "context": 2001,
         "ragged": True, "page": 16, "dtype": "f32"},
        # a decode step that keeps account of its keys: attention and weights
        {"name": "weights_step", "kind": "weights", "cache": "kv4", "shape": "llama-3.1-8b", "requests": 16, "tokens": 1,
         "context": 4001, "ragged": True, "page": 16, "dtype": "bf16"},
        # the last tokens of a prompt say which of its keys matter: a plain cache
        {"name": "weights_prompt", "kind": "weights", "cache": "plain", "shape": "llama-3.1-8b", "requests": 2, "tokens": 32,
         "context": 8009, "ragged": False, "page": 16, "dtype": "bf16"},
        # one request of a small model falls back to its budget, a cache in 4 bits
        {"name": "evict_one", "kind": "evict", "cache": "kv4", "shape": "llama-3.2-1b", "requests": 1, "context": 1152, "ragged": False,
         "keep": 1024, "first": 4, "last": 64, "page": 16, "dtype": "bf16"},
        # a batch of long prompts of a larger model, a plain cache
        {"name": "evict_batch", "kind": "evict", "cache": "plain", "shape": "llama-3.2-3b", "requests": 8, "context": 6001, "ragged": True,
         "keep": 2048, "first": 4, "last": 256, "page": 16, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _no_dearer(case, than):
    a, b = work(case), work(than)
    return a["flops"] <= b["flops"] and a["bytes"] <= b["bytes"]


def draw(rng):
    kind = rng.choice(("write", "attention", "attention", "attention", "weights", "evict"))
    most = {x["name"]: x for x in listed()}
    while True:
        shape, page = rng.choice(sorted(HEADS)), rng.choice((8, 16, 16, 32, 64))
        dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
        if kind == "write":
            case = {"kind": kind, "shape": shape, "tokens": _spread(rng, 1, 8191), "page": page, "dtype": dtype}
            if _no_dearer(case, most["write_prompt"]):
                return case
        elif kind == "attention":
            prompt = rng.random() < 0.25
            tokens = _spread(rng, 33, 2048) if prompt else rng.choice((1, 1, 1, _spread(rng, 1, 8)))
            case = {"kind": kind, "shape": shape, "requests": _spread(rng, 1, 4 if prompt else 64 if dtype == "bf16" else 8), "tokens": tokens,
                    "context": tokens + _spread(rng, 1, 8192 if prompt or dtype == "f32" else 131072), "ragged": rng.random() < 0.7,
                    "page": page, "dtype": dtype}
            if rng.random() < 0.25:
                case["window"] = _spread(rng, 64, 4096)
            if rng.random() < 0.2:
                case["sink"] = True
            if rng.random() < 0.2:
                case["softcap"] = 30.0
            if prompt and dtype == "f32" and tokens > 256:
                continue
            if _no_dearer(case, most["attention_prompt" if prompt else "attention_batch_64"] | ({"requests": 4} if prompt else {})):
                return case
        elif kind == "weights":
            plain = rng.random() < 0.5
            tokens = _spread(rng, 1, 64) if plain else 1
            case = {"kind": kind, "cache": "plain" if plain else "kv4", "shape": shape, "requests": _spread(rng, 1, 4 if tokens > 1 else 32),
                    "tokens": tokens, "context": tokens + _spread(rng, 1, 16384 if dtype == "bf16" else 4096), "ragged": rng.random() < 0.7,
                    "page": page, "dtype": dtype}
            if _no_dearer(case, most["attention_batch_64"]) or (tokens > 1 and case["context"] * tokens * case["requests"] <= 1 << 20):
                return case
        else:
            context = _spread(rng, 64, 8192)
            keep = rng.randint(context // 4 + 1, context)
            last = rng.randint(0, min(keep, 256))
            case = {"kind": kind, "cache": rng.choice(("plain", "kv4")), "shape": shape, "requests": _spread(rng, 1, 16), "context": context,
                    "ragged": rng.random() < 0.7, "keep": keep, "first": rng.randint(0, min(4, keep - last)), "last": last, "page": page,
                    "dtype": dtype}
            if _no_dearer(case, most["evict_batch"]) and _pool_bytes(case) <= 12 << 30:
                return case


def _sizes(case):
    """(tokens of each request in the step, its cached tokens with them): from the case alone."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    n, tokens, context = case["requests"], case.get("tokens", 0), case["context"]
    if not case.get("ragged") or n == 1:
        return [tokens] * n, [context] * n
    count = [rng.randint(max(1, tokens // 2), tokens) if tokens else 0 for _ in range(n)]
    held = [rng.randint(max(tokens, context // 8, 1), context) for _ in range(n)]
    count[-1], held[-1] = tokens, context                       # the largest is as large as the case says
    return count, held


def _row_bytes(case):
    """Bytes of one key or value of one head."""
    d = HEADS[case["shape"]][2]
    return d // 2 + d // 32 if case.get("cache", "kv4") == "kv4" else d * (2 if case["dtype"] == "bf16" else 4)


def _pool_bytes(case):
    _, kv, _, layers = HEADS[case["shape"]]
    return layers * kv * (2 * _row_bytes(case) + 4) * sum(-(-h // case["page"]) * case["page"] for h in _sizes(case)[1])


def work(case):
    heads, kv, d, layers = HEADS[case["shape"]]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "write":
        # rows in and their 4 bits out; the pages back, and their numbers
        n, pages = case["tokens"], -(-case["tokens"] // case["page"])
        rows = 2 * kv
        return {"bytes": n * rows * d * size + n * rows * (d // 2 + d // 32) + pages * case["page"] * rows * (d // 2 + d // 32 + d * size) + 4 * n + 4 * pages,
                "flops": 4 * n * rows * d}
    count, held = _sizes(case)
    if case["kind"] == "evict":
        # every sum is read; of the rows that stay, all but the first ones move
        moved = sum(case["keep"] - case["first"] for h in held if h > case["keep"])
        return {"bytes": layers * kv * (sum(4 * h for h in held if h > case["keep"]) + moved * (4 * _row_bytes(case) + 4)), "flops": layers * kv * sum(held)}
    window = case.get("window") or (1 << 30)
    seen = [min(h, window + n - 1) for n, h in zip(count, held)]
    row = _row_bytes(case)
    # a query row's keys: all cached ones, less half of the portion's own triangle, and not more than the window
    pairs = sum(n * min(h - (n - 1) / 2, window) for n, h in zip(count, held))
    q = sum(count) * heads * d * size
    if case["kind"] == "attention":
        return {"bytes": 2 * kv * row * sum(seen) + 2 * q, "flops": int(4 * heads * d * pairs)}
    if case["cache"] == "kv4":
        return {"bytes": kv * (2 * row + 8) * sum(seen) + 2 * q, "flops": int(4 * heads * d * pairs)}
    return {"bytes": kv * (row + 8) * sum(seen) + q, "flops": int(2 * heads * d * pairs)}


# ----------------------------------------------------------------------------- the format

def _order(d, values):
    """Which number of the head lies at each place of a stored row."""
    groups, run = d // 32, 4 if values else 8
    place = torch.arange(d)
    piece = place // run
    return 32 * (piece % groups) + run * (piece // groups) + place % run


def _scales(largest):
    """The scales' bytes of groups with these largest magnitudes (64 bits), and what they stand for."""
    fine = torch.isfinite(largest)
    x = torch.where(fine, largest, 0.0) / 7
    step = torch.exp2((torch.frexp(x).exponent.double() - 1).clamp(min=-14) - 3)
    x = (torch.round(x / step) * step).clamp(max=61440.0)
    byte = torch.where(fine, x.half().view(torch.int16).int() >> 7, 255)
    return byte.to(torch.uint8), torch.where(fine, x, math.nan)


def _to_bits(x, values):
    """Rows [..., d] as codes [..., d / 2] and scales [..., d / 32] in bytes.  In 64 bits: what lies beside a border falls on its side."""
    d = x.shape[-1]
    x = x.double().unflatten(-1, (-1, 32))
    byte, scale = _scales(x.abs().amax(-1))
    live = (scale > 0)[..., None]
    code = torch.where(live, torch.round(x / torch.where(live, scale[..., None], 1.0)).clamp(-7, 7), 0.0) + 8
    code = code.flatten(-2).to(torch.uint8)[..., _order(d, values).to(x.device)]
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def _numbers(codes, scales, values, dtype=torch.float32):
    """The numbers that codes [..., d / 2] and scales [..., d / 32] stand for."""
    d = codes.shape[-1] * 2
    stored = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    back = torch.argsort(_order(d, values)).to(codes.device)
    scale = (scales.to(torch.int16) << 7).view(torch.float16).to(dtype)
    return (stored[..., back].to(dtype) - 8) * scale.repeat_interleave(32, dim=-1)


def _parts(cache, page, d):
    """Views of a pool [..., bytes of a page]: codes [..., page, d / 2] and scales [..., page, d / 32]."""
    n = page * d // 2
    return cache[..., :n].unflatten(-1, (page, d // 2)), cache[..., n:].unflatten(-1, (page, d // 32))


# ----------------------------------------------------------------------------- what a program has in hand

def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + salt)


def _int(values):
    return torch.as_tensor(np.asarray(values, dtype=np.int32)).cuda()


def _normal(shape, seed, salt, dtype, std=1.0):
    return torch.randn(shape, generator=_generator(seed, salt), device="cuda", dtype=dtype).mul_(std)


def _pool(case, pages, seed, salt, values):
    """One plane of one layer, filled with rows of normal numbers."""
    _, kv, d, _ = HEADS[case["shape"]]
    page, dtype = case["page"], DTYPES[case["dtype"]]
    if case.get("cache", "kv4") != "kv4":
        return _normal((pages, kv, page, d), seed, salt, dtype)
    out = torch.empty((pages, kv, page * (d // 2 + d // 32)), dtype=torch.uint8, device="cuda")
    at_once = max(1, (1 << 25) // (kv * page * d))
    for lo in range(0, pages, at_once):
        n = min(at_once, pages - lo)
        x = _normal((n, kv, page, d), seed, salt * 100003 + lo, dtype)
        for part, bits in zip(_parts(out[lo:lo + n], page, d), _to_bits(x, values)):
            part.copy_(bits)
    return out


def _table(case, held, seed):
    """A block table over a pool of pages in no order, the size of the pool, and a page that nobody has."""
    rng = np.random.default_rng([seed, 91])
    counts = [-(-h // case["page"]) for h in held]
    pool = sum(counts) + 3
    free = rng.permutation(pool)
    table = np.full((len(held), -(-max(counts) // 8) * 8), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = free[at:at + c]
        at += c
    return _int(table), pool, int(free[-1])


def prepare(case, seed):
    heads, kv, d, layers = HEADS[case["shape"]]
    page, dtype = case["page"], DTYPES[case["dtype"]]
    s = {"case": case, "err": torch.zeros(4, dtype=torch.int32, device="cuda")}
    if case["kind"] == "write":
        T = case["tokens"]
        pages = -(-T // page)
        order = np.random.default_rng([seed, 92]).permutation(pages + 1)
        # keys and values as sections of one row of the projection, some channels of the keys larger than the others
        s["rows"] = _normal((T, (heads + 2 * kv) * d), seed, 1, dtype)
        s["rows"] *= torch.exp2(_normal((s["rows"].shape[1],), seed, 2, torch.float32).clamp_(-2, 2)).to(dtype)
        s["slots"] = _int((order[:pages, None] * page + np.arange(page)[None, :]).reshape(-1)[:T])
        s["pages"] = _int(order[:pages])
        s["k"], s["v"] = (_pool(case, pages + 1, seed, salt, values) for salt, values in ((3, False), (4, True)))
        return s
    count, held = _sizes(case)
    s["block_table"], pool, s["spare"] = _table(case, held, seed)
    s["context_lens"] = _int(held)
    if case["kind"] == "evict":
        s["kv"] = torch.stack([torch.stack([_pool(case, pool, seed, 10 + 2 * layer + values, bool(values)) for values in (0, 1)])
                               for layer in range(layers)])
        # sums as softmax weights leave them: a few keys have most
        s["weights"] = torch.exp(_normal((layers, pool, kv, page), seed, 5, torch.float32, 2.0))
        return s
    s["cu_tokens"] = _int(np.concatenate([[0], np.cumsum(count)]))
    s["held"] = _int([h - n for n, h in zip(count, held)])
    s["k"] = _pool(case, pool, seed, 3, False)
    if case["kind"] == "attention" or case["cache"] == "kv4":
        s["v"] = _pool(case, pool, seed, 4, True)
    # scores with a deviation of 2: a few keys take most of a row's weight, as they do in a trained model
    s["q"] = _normal((sum(count), heads * d), seed, 1, dtype, 2.0)
    s["sink"] = torch.randn(heads, generator=_generator(seed, 6), device="cuda") if case.get("sink") else None
    if case["kind"] == "weights":
        s["weights"] = torch.rand((pool, kv, page), generator=_generator(seed, 5), device="cuda")
    return s


# ----------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"write": _own_write, "attention": _own_attention, "weights": _own_weights, "evict": _own_evict}[kind](state)
    return {"write": _plain_write, "attention": _plain_attention, "weights": _plain_weights, "evict": _plain_evict}[kind](state)


def _sections(s):
    heads, kv, d, _ = HEADS[s["case"]["shape"]]
    return s["rows"][:, heads * d:(heads + kv) * d], s["rows"][:, (heads + kv) * d:]


def _own_write(s):
    from photon_infer_b200.kernels import ops
    c = s["case"]
    _, kv, d, _ = HEADS[c["shape"]]
    k, v = _sections(s)
    ops.kv4_write(k, v, s["slots"], s["k"], s["v"], n_kv=kv, head_dim=d, err=s["err"])
    numbers = [torch.empty((s["pages"].numel(), kv, c["page"], d), dtype=k.dtype, device="cuda") for _ in range(2)]
    ops.kv4_unpack(s["k"], s["v"], s["pages"], numbers[0], numbers[1], err=s["err"])
    return numbers


def _attention_args(s):
    c = s["case"]
    heads, kv, d, _ = HEADS[c["shape"]]
    return dict(num_seqs=c["requests"], max_tokens_per_seq=c["tokens"], max_keys=c["context"], n_q=heads, n_kv=kv, head_dim=d,
                window=c.get("window"), scale=d ** -0.5, err=s["err"], sink=s["sink"], softcap=c.get("softcap"))


def _own_attention(s):
    from photon_infer_b200.kernels import ops
    out = torch.empty_like(s["q"])
    ops.kv4_attention(s["q"], out, s["k"], s["v"], s["block_table"], s["cu_tokens"], s["context_lens"], **_attention_args(s))
    return out


def _own_weights(s):
    from photon_infer_b200.kernels import ops
    args = _attention_args(s)
    if s["case"]["cache"] != "kv4":
        ops.key_weights(s["q"], s["weights"], s["k"], s["block_table"], s["cu_tokens"], s["context_lens"], held=s["held"], **args)
        return s["weights"]
    out, lse = torch.empty_like(s["q"]), torch.empty((s["q"].shape[0], args["n_q"]), dtype=torch.float32, device="cuda")
    ops.kv4_attention(s["q"], out, s["k"], s["v"], s["block_table"], s["cu_tokens"], s["context_lens"], lse=lse, **args)
    ops.key_weights(s["q"], s["weights"], s["k"], s["block_table"], s["cu_tokens"], s["context_lens"], held=s["held"], lse=lse, **args)
    return out, lse, s["weights"]


def _own_evict(s):
    from photon_infer_b200.kernels import ops
    c = s["case"]
    lens = torch.empty_like(s["context_lens"])
    ops.cache_evict(s["kv"], s["weights"], s["block_table"], s["context_lens"], lens, num_seqs=c["requests"], max_keys=c["context"], keep=c["keep"],
                    keep_first=c["first"], keep_last=c["last"], err=s["err"])
    return s["kv"], s["weights"], lens


def _plain_write(s):
    c = s["case"]
    _, kv, d, _ = HEADS[c["shape"]]
    slots, pages = s["slots"].long(), s["pages"].long()
    numbers = []
    for cache, x, values in zip((s["k"], s["v"]), _sections(s), (False, True)):
        codes, scales = _parts(cache, c["page"], d)
        new = _to_bits(x.unflatten(1, (kv, d)), values)
        codes[slots // c["page"], :, slots % c["page"]] = new[0]
        scales[slots // c["page"], :, slots % c["page"]] = new[1]
        numbers.append(_numbers(codes[pages], scales[pages], values).to(x.dtype))
    return numbers


def _keys(s, cache, values):
    """The requests' rows side by side in 32 bits, [S, kv, keys, d], as far as the longest."""
    c = s["case"]
    _, kv, d, _ = HEADS[c["shape"]]
    pages = s["block_table"].long().clamp(min=0)
    if cache.dtype == torch.uint8:
        x = _numbers(*(part[pages] for part in _parts(cache, c["page"], d)), values)
    else:
        x = cache[pages].float()
    return x.permute(0, 2, 1, 3, 4).reshape(c["requests"], kv, -1, d)[:, :, :c["context"]]


def _plain_scores(s):
    """(weights [S, kv, N * G, keys] without their sum in the denominator, that sum, the maximum they are relative to)."""
    c = s["case"]
    heads, kv, d, _ = HEADS[c["shape"]]
    S, N, G = c["requests"], c["tokens"], heads // kv
    cu, lens = s["cu_tokens"].long(), s["context_lens"].long()
    n = cu[1:] - cu[:-1]
    place = torch.arange(N, device="cuda")
    token = (cu[:-1, None] + place).clamp(max=s["q"].shape[0] - 1)               # places behind a request's last token repeat some token
    q = s["q"][token].float().view(S, N, kv, G, d).permute(0, 2, 1, 3, 4).reshape(S, kv, N * G, d)
    x = torch.matmul(q, _keys(s, s["k"], False).transpose(2, 3)) * d ** -0.5
    if c.get("softcap"):
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    key, at = torch.arange(x.shape[3], device="cuda"), (lens - n)[:, None] + place
    seen = (key <= at[:, :, None]) & (place < n[:, None])[:, :, None]
    if c.get("window"):
        seen = seen & (key > at[:, :, None] - c["window"])
    x = torch.where(seen[:, None, :, None, :].expand(S, 1, N, G, -1).flatten(2, 3), x, -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].float().view(1, kv, 1, G).expand(S, kv, N, G).reshape(S, kv, N * G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    return x, torch.where(total == 0, 1.0, total), top


def _per_token(s, x):
    """[S, kv, N * G, w] as rows of the step's tokens, [T, heads * w]."""
    c = s["case"]
    heads, kv, _, _ = HEADS[c["shape"]]
    cu = s["cu_tokens"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    return x.view(c["requests"], kv, c["tokens"], heads // kv, -1).permute(0, 2, 1, 3, 4).flatten(2)[seq, t - cu[seq]]


def _plain_attention(s):
    x, total, _ = _plain_scores(s)
    return _per_token(s, torch.matmul(x, _keys(s, s["v"], True)) / total).to(s["q"].dtype)


def _plain_weights(s):
    x, total, top = _plain_scores(s)
    sums = (x / total).sum(2).transpose(1, 2)                                     # [S, keys, kv]
    key = torch.arange(sums.shape[1], device="cuda")[None, :]
    held, lens = s["held"].long()[:, None], s["context_lens"].long()[:, None]
    table = s["block_table"].long()
    page, at = torch.where(key < lens, table[:, :-(-sums.shape[1] // s["case"]["page"])].repeat_interleave(s["case"]["page"], 1)[:, :sums.shape[1]], s["spare"]), key % s["case"]["page"]
    old = s["weights"][page, :, at]
    new = torch.where((key < held)[..., None], old, 0.0) + sums
    s["weights"][page, :, at] = torch.where((key < lens)[..., None], new, old)
    if s["case"]["cache"] != "kv4":
        return s["weights"]
    out = _per_token(s, torch.matmul(x, _keys(s, s["v"], True)) / total).to(s["q"].dtype)
    return out, _per_token(s, top + torch.log(total)), s["weights"]


def _plain_evict(s):
    c = s["case"]
    _, kv, d, layers = HEADS[c["shape"]]
    page, keep = c["page"], min(c["keep"], c["context"])
    lens = s["context_lens"].long()
    key = torch.arange(c["context"], device="cuda")
    table = torch.where(s["block_table"] < 0, s["spare"], s["block_table"]).long()
    pages = table[:, key // page]                                                 # [S, keys]
    sums = s["weights"][:, pages, :, key % page].permute(2, 0, 3, 1)              # [layers, S, kv, keys] from [S, keys, layers, kv]
    # first those that stay anyway, then by their sums, then what is not there; of equals the first
    always = (key < c["first"]) | ((key >= lens[:, None] - c["last"]) & (key < lens[:, None]))
    sums = torch.where(always[None, :, None], math.inf, torch.where((key < lens[:, None])[None, :, None], sums, -math.inf))
    kept = torch.sort(sums, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    target = key[:keep].expand_as(kept)
    source = torch.where((lens > c["keep"])[None, :, None, None], kept, target)
    layer, head = torch.arange(layers, device="cuda")[:, None, None, None], torch.arange(kv, device="cuda")[None, None, :, None]
    request = torch.arange(c["requests"], device="cuda")[None, :, None, None]
    of, to = table[request, source // page], table[request, target // page]
    pools = [s["weights"].unsqueeze(1)] + (list(_parts(s["kv"], page, d)) if c["cache"] == "kv4" else [s["kv"]])
    for pool in pools:
        pool[layer, :, to, head, target % page] = pool[layer, :, of, head, source % page]
    return s["kv"], s["weights"], torch.minimum(lens, torch.full_like(lens, c["keep"])).int()


# ----------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["kind"] == "evict":
        return None                                             # rows moved as they are: nothing is computed
    s = prepare(case, seed)
    return _exact_write(case, s) if case["kind"] == "write" else _exact_attention(case, s)


def _exact_rounded(x):
    """Groups [n, 32] to the multiples of their scales that are kept, by looking among all scales and all codes."""
    # every scale there is, in ascending order, and the borders between neighbours
    scales = torch.cat([torch.arange(8, dtype=torch.float64) * 2.0 ** -17] +
                       [(8 + torch.arange(8, dtype=torch.float64)) * 2.0 ** (e - 18) for e in range(1, 31)]).cuda()
    want = x.abs().amax(1) / 7
    above = torch.searchsorted(scales, want).clamp(max=len(scales) - 1)           # the first one that is not below
    below = (above - 1).clamp(min=0)
    up, down = scales[above] - want, want - scales[below]
    pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    scale = scales[torch.where(want >= scales[-1], torch.full_like(pick, len(scales) - 1), pick)][:, None]
    best, code = torch.full_like(x, math.inf), torch.zeros_like(x)
    for c in (0, 2, -2, 4, -4, 6, -6, 1, -1, 3, -3, 5, -5, 7, -7):               # the even ones first: they have the ties
        away = (x - c * scale).abs()
        code = torch.where(away < best, float(c), code)
        best = torch.minimum(best, away)
    return code * scale


def _exact_write(case, s):
    heads, kv, d, _ = HEADS[case["shape"]]
    T, page, answers = case["tokens"], case["page"], []
    first = s["slots"].long() // page
    where = torch.empty(int(first.max()) + 1, dtype=torch.long, device="cuda")
    where[s["pages"].long()] = torch.arange(s["pages"].numel(), device="cuda")
    for cache, at, values in ((s["k"], heads * d, False), (s["v"], (heads + kv) * d, True)):
        codes, scales = _parts(cache[s["pages"].long()], page, d)
        whole = _numbers(codes, scales, values, torch.float64)   # what is in the pages' other places stays
        x = s["rows"][:, at:at + kv * d].double().reshape(T, kv, d // 32, 32)
        for lo in range(0, T, 1024):
            part = _exact_rounded(x[lo:lo + 1024].reshape(-1, 32)).view(-1, kv, d)
            slots = s["slots"].long()[lo:lo + 1024]
            whole[where[slots // page], :, slots % page] = part
        answers.append(whole)
    return answers


def _exact_attention(case, s):
    heads, kv, d, _ = HEADS[case["shape"]]
    count, held = _sizes(case)
    if sum(n * h for n, h in zip(count, held)) * heads * d > 2e13:
        return None
    weighs, at = case["kind"] == "weights", 0
    outs, lses = [], []
    sums = s["weights"].double() if weighs else None
    for r, (n, h) in enumerate(zip(count, held)):
        pages = s["block_table"][r, :-(-h // case["page"])].long()

        def rows(cache, values):
            x = _numbers(*_parts(cache[pages], case["page"], d), values, torch.float64) if cache.dtype == torch.uint8 else cache[pages].double()
            return x.transpose(0, 1).reshape(kv, -1, d)[:, :h]
        keys, values = rows(s["k"], False), rows(s["v"], True) if "v" in s else None
        q = s["q"][at:at + n].double().view(n, heads, d)
        where = torch.arange(h, device="cuda")
        hidden = where[None, :] > torch.arange(h - n, h, device="cuda")[:, None]
        if case.get("window"):
            hidden |= where[None, :] <= torch.arange(h - n, h, device="cuda")[:, None] - case["window"]
        out, lse = torch.empty((n, heads, d), dtype=torch.float64, device="cuda"), torch.empty((n, heads), dtype=torch.float64, device="cuda")
        got = torch.zeros((kv, h), dtype=torch.float64, device="cuda")
        for head in range(heads):
            group = head * kv // heads
            x = q[:, head] @ keys[group].T / math.sqrt(d)
            if case.get("softcap"):
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            x = x.masked_fill(hidden, -math.inf)
            if case.get("sink"):
                x = torch.cat([x, s["sink"][head].double().expand(n, 1)], dim=1)
            lse[:, head] = torch.logsumexp(x, dim=1)
            p = torch.softmax(x, dim=-1)[:, :h]
            got[group] += p.sum(0)
            if values is not None:
                out[:, head] = p @ values[group]
        if weighs:
            had = sums[pages].transpose(0, 1).reshape(kv, -1)
            had[:, :h] = torch.where(where < h - n, had[:, :h], 0.0) + got
            sums[pages] = had.view(kv, -1, case["page"]).transpose(0, 1)
        outs.append(out.view(n, heads * d))
        lses.append(lse)
        at += n
    if not weighs:
        return torch.cat(outs)
    return sums if case["cache"] != "kv4" else (torch.cat(outs), torch.cat(lses), sums)
