"""The operators of speculative decoding with trees of drafted tokens, as cases that can be timed and checked.

A step of tree decoding has the model score several drafted continuations of a request at once.  The drafted tokens are the
nodes of a tree whose root (node 0) is the request's last token; a node sees the request's cached tokens, its ancestors and
itself.  Three things happen that an ordinary decode step does not have:

* ``attention``: the nodes' queries over the paged cache and over the nodes they descend from (``ops.tree_attention``);
* ``accept``: from the nodes' logits, the path from the root along which the drafts are what the model itself would have
  generated, greedily or by sampling with given uniform numbers (``ops.tree_accept``);
* ``keep``: the accepted nodes' keys and values move, in every layer, to the places behind the request's cached tokens
  (``ops.cache_keep``);

and ``copy`` is what a request that forks needs of the same cache: whole pages copied in every layer
(``ops.cache_copy_pages``).  ``exact`` restates each in 64 bits, request by request.
"""
from __future__ import annotations

import json
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 128256

#: query heads, key/value heads, head size, layers: the Llama models that the benchmarks run, and heads without groups
HEADS = {"llama-3.2-1b": (32, 8, 64, 16), "llama-3.2-3b": (24, 8, 128, 28), "llama-3.1-8b": (32, 8, 128, 32),
         "ungrouped": (16, 16, 64, 16)}


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # one user, a short chain of drafts from a lookup in the prompt: the latency of one call
        {"name": "attention_chain", "kind": "attention", "shape": "llama-3.2-1b", "requests": 1, "nodes": 5, "depth": 4,
         "context": 640, "ragged": False, "page": 16, "dtype": "bf16"},
        # eight users of a small model, trees of an odd number of nodes behind contexts of very different lengths
        {"name": "attention_tree_8", "kind": "attention", "shape": "llama-3.2-1b", "requests": 8, "nodes": 27, "depth": 5,
         "context": 2500, "ragged": True, "page": 16, "dtype": "bf16"},
        # two long conversations with wide trees: few rows, very many keys
        {"name": "attention_long", "kind": "attention", "shape": "llama-3.1-8b", "requests": 2, "nodes": 64, "depth": 8,
         "context": 32768, "ragged": False, "page": 16, "dtype": "bf16"},
        # a full batch: the largest pass over cached keys
        {"name": "attention_batch_64", "kind": "attention", "shape": "llama-3.2-3b", "requests": 64, "nodes": 32, "depth": 6,
         "context": 6000, "ragged": True, "page": 32, "dtype": "bf16"},
        # layers with a window, a score beside the keys and bounded scores
        {"name": "attention_window", "kind": "attention", "shape": "llama-3.1-8b", "requests": 16, "nodes": 16, "depth": 5,
         "context": 8000, "ragged": True, "page": 64, "window": 1024, "sink": True, "softcap": 30.0, "dtype": "bf16"},
        # the true 32-bit run
        {"name": "attention_f32", "kind": "attention", "shape": "llama-3.2-1b", "requests": 4, "nodes": 13, "depth": 4,
         "context": 700, "ragged": True, "page": 16, "dtype": "f32"},
        # greedy acceptance for one user
        {"name": "accept_one", "kind": "accept", "requests": 1, "nodes": 8, "depth": 3, "vocab": VOCAB, "sampled": False},
        # a full batch, half of it sampling: the largest logits
        {"name": "accept_batch", "kind": "accept", "requests": 32, "nodes": 64, "depth": 6, "vocab": VOCAB, "sampled": True},
        # the accepted nodes of eight small trees, in all layers of a small model
        {"name": "keep_8", "kind": "keep", "shape": "llama-3.2-1b", "requests": 8, "nodes": 27, "depth": 5, "context": 200,
         "page": 16, "dtype": "bf16"},
        # the same for a full batch of a larger model
        {"name": "keep_48", "kind": "keep", "shape": "llama-3.2-3b", "requests": 48, "nodes": 64, "depth": 8, "context": 100,
         "page": 16, "dtype": "bf16"},
        # the last, partly filled pages of eight requests that fork
        {"name": "copy_8", "kind": "copy", "shape": "llama-3.2-1b", "pages": 8, "page": 16, "dtype": "bf16"},
        # a pool packed together: hundreds of pages of a larger model
        {"name": "copy_512", "kind": "copy", "shape": "llama-3.2-3b", "pages": 512, "page": 16, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _tree_size(rng, most):
    nodes = _spread(rng, 1, most)
    return nodes, (rng.randint(1, min(8, nodes - 1)) if nodes > 1 else 0)


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "accept", "keep", "copy"))
    while True:
        if kind == "attention":
            dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
            nodes, depth = _tree_size(rng, 128 if dtype == "bf16" else 32)
            case = {"kind": kind, "shape": rng.choice(sorted(HEADS)), "requests": _spread(rng, 1, 64 if dtype == "bf16" else 8),
                    "nodes": nodes, "depth": depth, "context": _spread(rng, 8, 65536 if dtype == "bf16" else 2048),
                    "ragged": rng.random() < 0.7, "page": rng.choice((8, 16, 16, 32, 64)), "dtype": dtype}
            if rng.random() < 0.25:
                case["window"] = _spread(rng, 64, 4096)
            if rng.random() < 0.2:
                case["sink"] = True
            if rng.random() < 0.2:
                case["softcap"] = 30.0
            if work(case)["flops"] <= work(listed()[3])["flops"] and work(case)["bytes"] <= work(listed()[3])["bytes"]:
                return case
        elif kind == "accept":
            nodes, depth = _tree_size(rng, 64)
            return {"kind": kind, "requests": _spread(rng, 1, 32), "nodes": nodes, "depth": depth,
                    "vocab": rng.choice((VOCAB, VOCAB, _spread(rng, 1000, VOCAB))), "sampled": rng.random() < 0.5}
        elif kind == "keep":
            depth = rng.randint(1, 8)
            return {"kind": kind, "shape": rng.choice(("llama-3.2-1b", "llama-3.2-3b", "ungrouped")),
                    "requests": _spread(rng, 1, 48), "nodes": _spread(rng, 2 * depth + 1, 64), "depth": depth,
                    "context": _spread(rng, 1, 100), "page": rng.choice((8, 16, 16, 32)), "dtype": rng.choice(("bf16", "bf16", "f32"))}
        else:
            case = {"kind": kind, "shape": rng.choice(("llama-3.2-1b", "llama-3.2-3b", "ungrouped")), "pages": _spread(rng, 1, 512),
                    "page": rng.choice((8, 16, 16, 32)), "dtype": rng.choice(("bf16", "bf16", "f32"))}
            if work(case)["bytes"] <= work(listed()[11])["bytes"]:
                return case


def _sizes(case):
    """(nodes of each request, cached tokens of each request, accepted nodes of each request, the root among them): from the case alone."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    n, context = case["requests"], case.get("context", 0)
    ragged = case.get("ragged", False) and n > 1
    least = case["depth"] + 1
    nodes = [rng.randint(max(least, case["nodes"] // 2), case["nodes"]) if ragged else case["nodes"] for _ in range(n)]
    held = [rng.randint(max(1, context // 8), context) if ragged else context for _ in range(n)]
    if ragged:
        nodes[-1], held[-1] = case["nodes"], context            # the largest is as large as the case says
    return nodes, held, [rng.randint(1, case["depth"] + 1) for _ in range(n)]


def work(case):
    if case["kind"] == "copy":
        _, kv, d, layers = HEADS[case["shape"]]
        page = layers * 2 * kv * d * case["page"] * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": 2 * case["pages"] * page + 8 * case["pages"], "flops": 0}
    nodes, held, accepted = _sizes(case)
    if case["kind"] == "accept":
        # the logits of the nodes on the path: the others' answers nobody asks for
        rows = sum(accepted)
        return {"bytes": 4 * rows * case["vocab"] + 8 * sum(nodes) + 8 * rows, "flops": rows * case["vocab"] * (4 if case["sampled"] else 1)}
    if case["kind"] == "keep":
        # every accepted node but the root moves
        _, kv, d, layers = HEADS[case["shape"]]
        row = layers * 2 * kv * d * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": sum(2 * (a - 1) * row + 4 * a for a in accepted) + 4 * case["requests"], "flops": 0}
    heads, kv, d, _ = HEADS[case["shape"]]
    size = 2 if case["dtype"] == "bf16" else 4
    window = case.get("window") or (1 << 30)
    seen = [min(h, window - 1) for h in held]                   # of the cached tokens, by the root
    rows = sum(nodes)
    return {"bytes": size * (2 * kv * d * sum(s + n for s, n in zip(seen, nodes)) + 2 * rows * heads * d) + rows * 4 * (-(-case["nodes"] // 32)),
            "flops": sum(4 * heads * d * n * (s + 1) for s, n in zip(seen, nodes))}


# ----------------------------------------------------------------------------- trees

def _tree(rng, nodes, depth, accepted, apart):
    """Parents of a tree's nodes, by levels, and a path of `accepted` nodes from the root that can be gone `depth` levels down.
    ``apart``: the first level is wide and the path leaves it behind its first `accepted` nodes, so that no accepted node but the
    root lies where another one belongs."""
    if nodes == 1:
        return np.array([-1], dtype=np.int32), [0]
    if apart:
        level = np.concatenate([np.ones(depth, dtype=np.int64), np.arange(1, depth + 1), rng.integers(1, depth + 1, nodes - 1 - 2 * depth)])
    else:
        level = np.concatenate([np.arange(1, depth + 1), rng.integers(1, depth + 1, nodes - 1 - depth)])
    level = np.concatenate([[0], np.sort(level)])
    first = np.searchsorted(level, np.arange(depth + 2))        # first node of each level
    spine = [0]
    for d in range(1, depth + 1):
        low = first[d] + (depth if apart and d == 1 else 0)
        spine.append(int(rng.integers(low, first[d + 1])))
    parents = np.full(nodes, -1, dtype=np.int32)
    for i in range(1, nodes):
        d = int(level[i])
        parents[i] = spine[d - 1] if i == spine[d] else rng.integers(first[d - 1], first[d])
    return parents, spine[:accepted]


def _ancestors(parents):
    """(bit masks of the nodes that each node sees, their depths)."""
    n = len(parents)
    seen = np.zeros((n, n), dtype=bool)
    depth = np.zeros(n, dtype=np.int64)
    for i in range(n):
        if parents[i] >= 0:
            seen[i] = seen[parents[i]]
            depth[i] = depth[parents[i]] + 1
        seen[i, i] = True
    return seen, depth


def _words(seen, words):
    bits = np.zeros((seen.shape[0], words * 32), dtype=np.uint64)
    bits[:, :seen.shape[1]] = seen
    w = (bits.reshape(seen.shape[0], words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32).view(np.int32)


def _trees(case, seed):
    """The trees of a case: one dict of host arrays per request."""
    rng = np.random.default_rng([seed, 77])
    nodes, held, accepted = _sizes(case)
    out = []
    for n, h, a in zip(nodes, held, accepted):
        parents, path = _tree(rng, n, case["depth"] if n > 1 else 0, a, case["kind"] == "keep")
        seen, depth = _ancestors(parents)
        out.append({"parents": parents, "path": path, "seen": seen, "depth": depth, "held": h})
    return out


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + salt)


def _int(values):
    return torch.as_tensor(np.asarray(values, dtype=np.int32)).cuda()


def _indices(case, trees):
    """What every step of tree decoding has on the device: where each request's nodes begin, their masks and parents."""
    cu = np.concatenate([[0], np.cumsum([len(t["parents"]) for t in trees])])
    words = -(-case["nodes"] // 32)
    return {"cu_tokens": _int(cu), "context_lens": _int([t["held"] + len(t["parents"]) for t in trees]),
            "positions": _int(np.concatenate([t["held"] + t["depth"] for t in trees])),
            "parents": _int(np.concatenate([t["parents"] for t in trees])),
            "tree_mask": _int(np.concatenate([_words(t["seen"], words) for t in trees]))}


def _table(case, trees, seed):
    """A block table over a pool of pages in no order, and the size of the pool."""
    rng = np.random.default_rng([seed, 78])
    counts = [-(-(t["held"] + len(t["parents"])) // case["page"]) for t in trees]
    pool = sum(counts) + 3
    free = rng.permutation(pool)
    table = np.full((len(trees), -(-max(counts) // 8) * 8), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = free[at:at + c]
        at += c
    return _int(table), pool


# ----------------------------------------------------------------------------- what a program has in hand

def prepare(case, seed):
    state = {"case": case, "err": torch.zeros(4, dtype=torch.int32, device="cuda")}
    if case["kind"] == "copy":
        _, kv, d, layers = HEADS[case["shape"]]
        n = case["pages"]
        order = np.random.default_rng([seed, 79]).permutation(2 * n + 1)
        state["kv"] = torch.randn((layers, 2, 2 * n + 1, kv, case["page"], d), generator=_generator(seed, 1), device="cuda", dtype=DTYPES[case["dtype"]])
        state["pairs"] = _int(np.stack([order[:n], order[n:2 * n]], axis=1))
        return state
    trees = _trees(case, seed)
    state.update(_indices(case, trees))
    if case["kind"] == "accept":
        state.update(_logits(case, trees, seed))
        return state
    heads, kv, d, layers = HEADS[case["shape"]]
    dtype = DTYPES[case["dtype"]]
    state["block_table"], pool = _table(case, trees, seed)
    if case["kind"] == "keep":
        state["kv"] = torch.randn((layers, 2, pool, kv, case["page"], d), generator=_generator(seed, 1), device="cuda", dtype=dtype)
        path = np.full((len(trees), case["depth"] + 1), -1, dtype=np.int32)
        for s, t in enumerate(trees):
            path[s, :len(t["path"])] = t["path"]
        state["path"], state["counts"] = _int(path), _int([len(t["path"]) for t in trees])
        return state
    T = sum(len(t["parents"]) for t in trees)
    normal = lambda shape, salt, std: torch.randn(shape, generator=_generator(seed, salt), device="cuda", dtype=dtype).mul_(std)
    # scores with a deviation of 2: a few keys take most of a row's weight, as they do in a trained model
    state["q"] = normal((T, heads * d), 1, 2.0)
    state["k"], state["v"] = normal((pool, kv, case["page"], d), 2, 1.0), normal((pool, kv, case["page"], d), 3, 1.0)
    state["sink"] = torch.randn(heads, generator=_generator(seed, 4), device="cuda") if case.get("sink") else None
    return state


def _logits(case, trees, seed):
    """Logits of all nodes, the drafted tokens, and the numbers that decide what is sampled.  Along each tree's accepted path the
    drafted child is the token that its parent's logits give: greedily the largest, with a temperature one that holds a fair part of the
    probability, with a uniform number from the middle of its part (so that sums in another order give the same token)."""
    g, rng = _generator(seed, 5), np.random.default_rng([seed, 80])
    V, T = case["vocab"], sum(len(t["parents"]) for t in trees)
    logits = torch.randn((T, V), generator=g, device="cuda").mul_(2.5)
    temperature = np.array([rng.uniform(0.6, 1.0) if case["sampled"] and s % 2 == 0 else 0.0 for s in range(len(trees))], dtype=np.float32)
    uniforms = (rng.integers(0, 1 << 24, T) / float(1 << 24)).astype(np.float32)
    token = rng.integers(0, V, T).astype(np.int32)
    rows, temps, wanted = [], [], []
    at = 0
    for t, temp in zip(trees, temperature):
        for i, node in enumerate(t["path"]):
            rows.append(at + node)
            temps.append(temp if temp > 0 else 1.0)
            wanted.append(int(rng.integers(0, V)))
            if i + 1 < len(t["path"]):
                token[at + t["path"][i + 1]] = wanted[-1]
        at += len(t["parents"])
    row, want = torch.as_tensor(rows).cuda(), torch.as_tensor(wanted).cuda()
    logits[row, want] = 14.0 + torch.rand(len(rows), generator=g, device="cuda")
    chosen = torch.empty(len(rows), dtype=torch.float64, device="cuda")
    for lo in range(0, len(rows), 64):
        part = slice(lo, lo + 64)
        p = torch.softmax(logits[row[part]].double() / torch.as_tensor(np.asarray(temps[part])).cuda().double()[:, None], dim=-1)
        at_want = p.gather(1, want[part, None])[:, 0]
        chosen[part] = p.cumsum(-1).gather(1, want[part, None])[:, 0] - at_want / 2
    device_uniforms = torch.as_tensor(uniforms).cuda()
    device_uniforms[row] = chosen.float()
    return {"logits": logits, "tokens": torch.as_tensor(token).cuda(), "temperature": torch.as_tensor(temperature).cuda(), "uniforms": device_uniforms}


# ----------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": _own_attention, "accept": _own_accept, "keep": _own_keep, "copy": _own_copy}[kind](state)
    return {"attention": _plain_attention, "accept": _plain_accept, "keep": _plain_keep, "copy": _plain_copy}[kind](state)


def _own_attention(s):
    from photon_infer_b200.kernels import ops
    c = s["case"]
    heads, kv, d, _ = HEADS[c["shape"]]
    out = torch.empty_like(s["q"])
    ops.tree_attention(s["q"], out, s["k"], s["v"], s["block_table"], s["cu_tokens"], s["context_lens"], s["positions"], s["tree_mask"],
                       num_seqs=c["requests"], max_tokens_per_seq=c["nodes"], max_keys=c["context"] + c["nodes"], n_q=heads, n_kv=kv,
                       head_dim=d, window=c.get("window"), scale=d ** -0.5, err=s["err"], sink=s["sink"], softcap=c.get("softcap"))
    return out


def _own_accept(s):
    from photon_infer_b200.kernels import ops
    c = s["case"]
    path = torch.empty((c["requests"], c["depth"] + 1), dtype=torch.int32, device="cuda")
    sampled, counts = torch.empty_like(path), torch.empty(c["requests"], dtype=torch.int32, device="cuda")
    ops.tree_accept(s["logits"], s["tokens"], s["parents"], s["cu_tokens"], num_seqs=c["requests"], max_tokens_per_seq=c["nodes"],
                    path=path, counts=counts, sampled=sampled, temperature=s["temperature"] if c["sampled"] else None,
                    uniforms=s["uniforms"] if c["sampled"] else None, err=s["err"])
    return path, counts, sampled


def _own_keep(s):
    from photon_infer_b200.kernels import ops
    ops.cache_keep(s["kv"], s["block_table"], s["cu_tokens"], s["context_lens"], s["path"], s["counts"], num_seqs=s["case"]["requests"], err=s["err"])
    return s["kv"]


def _own_copy(s):
    from photon_infer_b200.kernels import ops
    ops.cache_copy_pages(s["kv"], s["pairs"], err=s["err"])
    return s["kv"]


def _places(s):
    """(request of each node, its place in the request): from the nodes' ranges."""
    cu = s["cu_tokens"].long()
    t = torch.arange(s["parents"].numel(), device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    return cu, seq, t - cu[seq]


def _seen(s, width):
    """Which nodes of its request each node sees, as truth values [T, width]."""
    bit = torch.arange(32, device="cuda", dtype=torch.int32)
    return ((s["tree_mask"][:, :, None] >> bit) & 1).bool().flatten(1)[:, :width]


def _plain_attention(s):
    c = s["case"]
    heads, kv, d, _ = HEADS[c["shape"]]
    S, N, G = c["requests"], c["nodes"], heads // kv
    cu, seq, place = _places(s)
    # [S, N, ...]: the nodes of each request side by side; places behind a request's last node repeat some node
    node = (cu[:-1, None] + torch.arange(N, device="cuda")).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][node].float().view(S, N, kv, G, d).permute(0, 2, 1, 3, 4).reshape(S, kv, N * G, d)
    pages = s["block_table"].long().clamp(min=0)
    k = s["k"][pages].float().permute(0, 2, 1, 3, 4).reshape(S, kv, -1, d)[:, :, :c["context"] + N]
    v = s["v"][pages].float().permute(0, 2, 1, 3, 4).reshape(S, kv, -1, d)[:, :, :c["context"] + N]
    L = k.shape[2]
    scores = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    if c.get("softcap"):
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    key = torch.arange(L, device="cuda")
    base = s["context_lens"].long() - (cu[1:] - cu[:-1])
    of_tree = key[None, :] - base[:, None]                                       # [S, L]: a key's place among the nodes
    seen = torch.gather(_seen(s, N)[node], 2, of_tree.clamp(0, N - 1)[:, None, :].expand(S, N, L))
    position = s["positions"].long()[node]                                       # [S, N]
    visible = torch.where((of_tree < 0)[:, None, :], torch.ones_like(seen), seen & (of_tree < (cu[1:] - cu[:-1])[:, None])[:, None, :])
    if c.get("window"):
        where = torch.gather(position, 1, of_tree.clamp(0, N - 1))               # positions of the keys that are nodes
        where = torch.where(of_tree < 0, key[None, :], where)
        visible = visible & (where[:, None, :] > position[:, :, None] - c["window"])
    visible = visible[:, None, :, None, :].expand(S, 1, N, G, L).reshape(S, 1, N * G, L)
    scores = torch.where(visible, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].float().view(1, kv, 1, G).expand(1, kv, N, G).reshape(1, kv, N * G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weight = torch.exp(scores - top)
    total = weight.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(weight, v) / torch.where(total == 0, torch.ones_like(total), total)
    return o.view(S, kv, N, G, d).permute(0, 2, 1, 3, 4).reshape(S, N, heads * d)[seq, place].to(s["q"].dtype)


def _plain_accept(s):
    c = s["case"]
    S, N, D = c["requests"], c["nodes"], c["depth"] + 1
    cu, seq, _ = _places(s)
    sampled = s["logits"].argmax(-1)
    if c["sampled"]:
        temperature = s["temperature"][seq]
        warm = torch.where(temperature > 0, temperature, torch.ones_like(temperature))[:, None]
        p = torch.exp((s["logits"] - s["logits"].amax(-1, keepdim=True)) / warm)
        total = p.cumsum(-1)
        drawn = (total < (s["uniforms"] * total[:, -1])[:, None]).sum(-1).clamp(max=c["vocab"] - 1)
        sampled = torch.where(temperature > 0, drawn, sampled)
    # a node is right when its token is its parent's, and it is the first such child
    own_place = cu[:-1, None] + torch.arange(N, device="cuda")
    valid = own_place < cu[1:, None]
    node = own_place.clamp(max=s["parents"].numel() - 1)
    parent, token = s["parents"].long()[node], s["tokens"].long()[node]
    of_parent = sampled[(cu[:-1, None] + parent.clamp(min=0)).clamp(max=sampled.numel() - 1)]
    right = valid & (parent >= 0) & (token == of_parent)
    earlier = torch.ones((N, N), dtype=torch.bool, device="cuda").tril(-1)
    right = right & ~((parent[:, :, None] == parent[:, None, :]) & right[:, None, :] & earlier).any(-1)
    right[:, 0] = True                                                           # the root
    # it is accepted when everything it descends from is right as well
    accepted = valid & ~(_seen(s, N)[node] & ~right[:, None, :]).any(-1)
    counts = accepted.sum(-1)
    order = torch.where(accepted, torch.arange(N, device="cuda"), N).sort(-1).values
    order = torch.cat([order, torch.full((S, D), N, device="cuda")], dim=1)[:, :D]
    there = order < N
    path = torch.where(there, order, -1)
    tokens = torch.where(there, sampled[(cu[:-1, None] + order).clamp(max=sampled.numel() - 1)], -1)
    return path.int(), counts.int(), tokens.int()


def _plain_keep(s):
    c = s["case"]
    cu = s["cu_tokens"].long()
    base = (s["context_lens"].long() - (cu[1:] - cu[:-1]))[:, None]
    path = s["path"].long()
    moved = torch.arange(path.shape[1], device="cuda")[None, :].expand_as(path)
    there = moved < s["counts"][:, None]
    source, target = base + torch.where(there, path, 0), base + torch.where(there, moved, 0)
    table = s["block_table"].long()
    page, place = (lambda at: table.gather(1, at // c["page"])), (lambda at: at % c["page"])
    s["kv"][:, :, page(target), :, place(target)] = s["kv"][:, :, page(source), :, place(source)]
    return s["kv"]


def _plain_copy(s):
    source, target = s["pairs"].long().unbind(1)
    s["kv"][:, :, target] = s["kv"][:, :, source]
    return s["kv"]


# ----------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    if case["kind"] in ("keep", "copy"):
        return None                                             # rows moved as they are: nothing is computed
    s, trees = prepare(case, seed), _trees(case, seed)
    return _exact_accept(case, s, trees) if case["kind"] == "accept" else _exact_attention(case, s, trees)


def _exact_attention(case, s, trees):
    heads, kv, d, _ = HEADS[case["shape"]]
    outs, at = [], 0
    for r, t in enumerate(trees):
        n, h = len(t["parents"]), t["held"]
        pages = s["block_table"][r, :-(-(h + n) // case["page"])].long()
        keys, values = (s[x][pages].transpose(0, 1).reshape(kv, -1, d)[:, :h + n].double() for x in ("k", "v"))
        where = torch.as_tensor(np.concatenate([np.arange(h), h + t["depth"]])).cuda()
        visible = torch.ones((n, h + n), dtype=torch.bool, device="cuda")
        visible[:, h:] = torch.as_tensor(t["seen"]).cuda()
        if case.get("window"):
            visible &= where[None, :] > where[h:, None] - case["window"]
        q = s["q"][at:at + n].double().view(n, heads, d)
        out = torch.empty((n, heads, d), dtype=torch.float64, device="cuda")
        for head in range(heads):
            x = q[:, head] @ keys[head * kv // heads].T / math.sqrt(d)
            if case.get("softcap"):
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            x = x.masked_fill(~visible, -math.inf)
            if case.get("sink"):
                x = torch.cat([x, s["sink"][head].double().expand(n, 1)], dim=1)
            out[:, head] = torch.softmax(x, dim=-1)[:, :h + n] @ values[head * kv // heads]
        outs.append(out.view(n, heads * d))
        at += n
    return torch.cat(outs)


def _exact_accept(case, s, trees):
    D = case["depth"] + 1
    path, counts, sampled = [], [], []
    token, uniforms, temperature = s["tokens"].tolist(), s["uniforms"].double().tolist(), s["temperature"].double().tolist()
    at = 0
    for r, t in enumerate(trees):
        node, nodes, got = 0, [], []
        while node is not None:
            x = s["logits"][at + node].double()
            if case["sampled"] and temperature[r] > 0:
                p = torch.softmax(x / temperature[r], dim=0).cumsum(0)
                answer = int(torch.searchsorted(p, uniforms[at + node] * p[-1:]).clamp(max=case["vocab"] - 1))
            else:
                answer = int((x == x.max()).nonzero()[0])
            nodes.append(node)
            got.append(answer)
            children = [i for i in range(len(t["parents"])) if t["parents"][i] == node and token[at + i] == answer]
            node = children[0] if children and len(nodes) < D else None
        path.append(nodes + [-1] * (D - len(nodes)))
        counts.append(len(nodes))
        sampled.append(got + [-1] * (D - len(got)))
        at += len(t["parents"])
    return _int(path), _int(counts), _int(sampled)
