"""The operators of steps with drafted tokens and of forked requests, as cases that can be prepared, run once and compared.

    attention   the nodes of a tree of drafted tokens per request look at the request's cached tokens and at their own
                ancestors (`ops.attention_tree`)
    accept      which drafted tokens the model agrees with; the rows of the accepted ones move together in the caches of all
                layers (`ops.accept_tree`)
    fork        pages of all layers, and state slots, copied for requests that part ways (`ops.copy_blocks`)

Head counts and sizes are those of the benchmark's models (Qwen2.5 0.5B, 3B and 7B). Requests hold pages of 16 tokens in any order.
"""
import math
import random

import torch

own = False

PAGE = 16
MOST_NODES = 64
VOCAB = 151936

# (query heads, key/value heads, head size, layers)
MODELS = {"0.5b": (14, 2, 64, 24), "3b": (16, 2, 128, 36), "7b": (28, 4, 128, 28)}


def listed():
    return [
        # one user at a prompt, a few drafted tokens: the smallest call, all latency
        {"name": "attention 1 short", "op": "attention", "model": "0.5b", "requests": 1, "nodes": 8, "longest": 300, "shortest": 300},
        # a handful of users with long answers, small trees
        {"name": "attention 8 long", "model": "0.5b", "op": "attention", "requests": 8, "nodes": 16, "longest": 4000, "shortest": 3700},
        # a full server, contexts of all lengths, nodes of all counts
        {"name": "attention 64 ragged", "op": "attention", "model": "3b", "requests": 64, "nodes": 17, "longest": 4003, "shortest": 205},
        # a full server with the widest trees: as much arithmetic as there can be
        {"name": "attention 64 wide", "op": "attention", "model": "7b", "requests": 64, "nodes": 64, "longest": 4001, "shortest": 2003},
        # one user in a very long document: the keys of one request over the whole device
        {"name": "attention 1 long", "op": "attention", "model": "7b", "requests": 1, "nodes": 33, "longest": 32500, "shortest": 32500},
        # a windowed layer: most of the context is out of sight
        {"name": "attention window", "op": "attention", "model": "3b", "requests": 16, "nodes": 24, "longest": 4003, "shortest": 900,
         "window": 1024},
        # the true 32-bit path
        {"name": "attention 32-bit", "op": "attention", "model": "0.5b", "requests": 4, "nodes": 13, "longest": 2001, "shortest": 411,
         "dtype": "float32"},
        # one user's step: nothing but latency
        {"name": "accept 1", "op": "accept", "model": "0.5b", "requests": 1, "nodes": 8, "depth": 5, "longest": 300},
        # a full server's step, wide trees
        {"name": "accept 64", "op": "accept", "model": "7b", "requests": 64, "nodes": 64, "depth": 12, "longest": 101},
        # the same choice on 32-bit caches, a few users
        {"name": "accept 32-bit", "op": "accept", "model": "0.5b", "requests": 7, "nodes": 23, "depth": 9, "longest": 150, "dtype": "float32"},
        # one answer is continued in two ways: its last page
        {"name": "fork 1", "op": "fork", "model": "0.5b", "pages": 1, "pool": 65},
        # many at once, the last pages of 64 requests and the windows' pages with them, at the larger model's sizes
        {"name": "fork 256", "op": "fork", "model": "7b", "pages": 256, "pool": 700},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "accept", "fork"])
    case = {"op": op, "model": rng.choice(sorted(MODELS))}
    if op == "attention":
        case["requests"] = _log(rng, 1, 64)
        case["nodes"] = _log(rng, 1, MOST_NODES)
        case["longest"] = _log(rng, 20, min(32000, 190000 // case["requests"]))
        case["shortest"] = rng.randint(1, case["longest"])
        if rng.random() < 0.25:
            case["window"] = _log(rng, 5, 4096)
        if rng.random() < 0.25:
            case["dtype"] = "float32"
            case["requests"] = min(case["requests"], 16)
            case["longest"] = min(case["longest"], 4000)
            case["shortest"] = min(case["shortest"], case["longest"])
    elif op == "accept":
        case["requests"] = _log(rng, 1, 64)
        case["nodes"] = _log(rng, 2, MOST_NODES)
        case["depth"] = rng.randint(1, min(16, case["nodes"] - 1))
        case["longest"] = _log(rng, 20, 101)
        if rng.random() < 0.3:
            case["dtype"] = "float32"
            case["requests"] = min(case["requests"], 16)
    else:
        case["pages"] = _log(rng, 1, 256)
        case["pool"] = 2 * case["pages"] + rng.randint(1, 180)
        if rng.random() < 0.3:
            case["dtype"] = "float32"
            case["pages"] = min(case["pages"], 100)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------


def _dtype(case):
    return torch.float32 if case.get("dtype") == "float32" else torch.bfloat16


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _counts(case):
    """Nodes of each request: most have all of them, every third fewer."""
    n = case["nodes"]
    return [max(1, n - (n * (r % 7)) // 9) if r % 3 == 2 else n for r in range(case["requests"])]


def _tables(rng, lengths):
    """Pages for requests of these lengths, handed out in any order: (table [requests, width], pages in the pool)."""
    need = [-(-n // PAGE) for n in lengths]
    order = list(range(sum(need)))
    rng.shuffle(order)
    width = -(-max(need) // 8) * 8
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32), sum(need)


def _masks(parents):
    """Each node's ancestors and itself as the bits of a number."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else 0) | (1 << i))
    return out


def _signed(m):
    return m - (1 << 64) if m >= 1 << 63 else m


def _grown_tree(rng, n):
    """Parents of n nodes: mostly the node before, else any node before."""
    return [-1] + [i - 1 if rng.random() < 0.6 else rng.randrange(i) for i in range(1, n)]


def _chain_tree(rng, n, depth):
    """Parents of n nodes: a chain of `depth` behind node 0, then branches off it that go no deeper."""
    parents, deep = [-1], [0]
    for i in range(1, n):
        if i <= depth:
            p = i - 1
        elif deep[i - 1] < depth and rng.random() < 0.6 and i - 1 > depth:
            p = i - 1
        else:
            p = rng.choice([k for k in range(i) if deep[k] < depth])
        parents.append(p)
        deep.append(deep[p] + 1)
    return parents


def _accepted(r, n, depth):
    """How many drafted tokens of request r the model agrees with."""
    return (3 * r + 2) % (min(depth, n - 1) + 1)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _dtype(case)
    H, KV, dh, layers = MODELS[case["model"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)

    if case["op"] == "fork":
        pages = list(range(case["pool"]))
        rng.shuffle(pages)
        n = case["pages"]
        sources = [pages[rng.randrange(max(1, n // 2))] if i % 2 else pages[i] for i in range(n)]
        state = {"op": "fork", "pairs": list(zip(sources, pages[n:2 * n])),
                 "kv": torch.empty(layers, 2, case["pool"] + 1, KV, PAGE, dh, device="cuda", dtype=dtype)}
        for layer in state["kv"]:
            layer.normal_(generator=gen)
        return state

    counts = _counts(case)
    committed = _spread(case.get("shortest", max(1, case["longest"] // 3)), case["longest"], case["requests"])
    held = [c + n for c, n in zip(committed, counts)]
    table, pool = _tables(rng, held)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    T = starts[-1]
    state = {"op": case["op"], "most": max(counts), "table": table.cuda(),
             "cu_q": torch.tensor(starts, dtype=torch.int32).cuda(), "ctx_len": torch.tensor(held, dtype=torch.int32).cuda()}
    if case["op"] == "attention":
        masks = [m for n in counts for m in _masks(_grown_tree(rng, n))]
        # queries and keys as a trained layer has them: scores of a few units, some rows sharp
        state.update(q=normal(T, H * dh, std=1.5), k=normal(pool + 1, KV, PAGE, dh), v=normal(pool + 1, KV, PAGE, dh),
                     heads=H, window=case.get("window", 0), scale=1.0 / math.sqrt(dh))
    else:
        masks, tokens, sampled = [], [], []
        for r, n in enumerate(counts):
            parents = _chain_tree(rng, n, case["depth"])
            own_masks = _masks(parents)
            good = _accepted(r, n, case["depth"])
            ends = [i for i in range(n) if bin(own_masks[i]).count("1") == good + 1]
            path = own_masks[rng.choice(ends)]                    # the way that the model goes
            tok = rng.sample(range(VOCAB), n)                     # every drafted token another
            smp = [rng.randrange(VOCAB) for _ in range(n)]        # (a chance hit is one in 150,000)
            for i in range(1, n):
                if path >> i & 1:
                    smp[parents[i]] = tok[i]
            masks += own_masks
            tokens += tok
            sampled += smp
        kv = torch.empty(layers, 2, pool + 1, KV, PAGE, dh, device="cuda", dtype=dtype)
        for layer in kv:
            layer.normal_(generator=gen)
        state.update(kv=kv, tokens=torch.tensor(tokens, dtype=torch.int32).cuda(), sampled=torch.tensor(sampled, dtype=torch.int32).cuda())
    state["mask"] = torch.tensor([_signed(m) for m in masks], dtype=torch.int64).cuda()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------


def run(state):
    if state["op"] == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if state["op"] == "accept":
        return _accept_own(state) if own else _accept_plain(state)
    return _fork_own(state) if own else _fork_plain(state)


def _attention_own(s):
    from boring_llm_b200.kernels import ops
    out = torch.empty_like(s["q"])
    ops.attention_tree(s["q"], s["k"], s["v"], s["cu_q"], s["ctx_len"], s["mask"], s["table"], out, s["heads"], s["window"], s["scale"])
    return out


def _accept_own(s):
    from boring_llm_b200.kernels import ops
    counts, path, tokens = ops.accept_tree(s["sampled"], s["tokens"], s["mask"], s["cu_q"], s["ctx_len"], s["kv"][:, 0], s["kv"][:, 1],
                                           s["table"])
    return {"counts": counts, "path": path, "tokens": tokens, "kv": s["kv"]}


def _fork_own(s):
    from boring_llm_b200.kernels import ops
    ops.copy_blocks([s["kv"][:, 0], s["kv"][:, 1]], s["pairs"])
    return s["kv"]


def _padded(s):
    """Node i of request r is row at[r, i] of the flat arrays where real[r, i] is true."""
    i = torch.arange(s["most"], device="cuda")
    begin, end = s["cu_q"][:-1, None].long(), s["cu_q"][1:, None].long()
    real = begin + i < end
    return torch.where(real, begin + i, begin), real


def _bits(mask):
    """[.., 64] truth values."""
    return (mask[..., None] >> torch.arange(64, device="cuda")) & 1 == 1


def _attention_plain(s):
    q, H, window = s["q"], s["heads"], s["window"]
    at, real = _padded(s)
    R, N = at.shape
    _, KV, _, dh = s["k"].shape
    G = H // KV
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    c = s["ctx_len"].long() - n
    pages = s["table"].long().clamp(min=0)
    L = pages.shape[1] * PAGE
    keys = s["k"][pages].float().permute(0, 2, 1, 3, 4).reshape(R, KV, L, dh)
    j = torch.arange(L, device="cuda")
    values = s["v"][pages].float().permute(0, 2, 1, 3, 4).reshape(R, KV, L, dh)
    bits = _bits(s["mask"][at])                                   # [R, N, 64]
    depth = (bits.sum(-1) - 1).clamp(min=0)                       # [R, N]
    node = (j - c[:, None]).clamp(0, 63)                          # [R, L]: the node that a row holds
    drafted = (j >= c[:, None]) & (j < (c + n)[:, None])
    seen = torch.where(drafted[:, None, :], bits.gather(2, node[:, None, :].expand(R, N, L)), (j < c[:, None])[:, None, :])
    if window > 0:
        place = torch.where(drafted, c[:, None] + depth.gather(1, node.clamp(max=N - 1)), j)
        seen = seen & (place[:, None, :] + window > (c[:, None] + depth)[:, :, None])
    rows = q[at].float().view(R, N, KV, G, dh).permute(0, 2, 3, 1, 4).reshape(R, KV, G * N, dh)
    scores = (rows @ keys.transpose(-1, -2)).view(R, KV, G, N, L) * s["scale"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(R, KV, G * N, L) @ values).view(R, KV, G, N, dh) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(R * N, H * dh)
    # back to the flat order: the padded places write what their request's first node has
    flat = torch.empty_like(q)
    first = torch.arange(R, device="cuda")[:, None] * N + torch.where(real, torch.arange(N, device="cuda"), 0)
    flat[at.reshape(-1)] = out[first.reshape(-1)].to(q.dtype)
    return flat


def _accept_plain(s):
    at, real = _padded(s)
    R, N = at.shape
    i = torch.arange(N, device="cuda")
    mask = s["mask"][at]
    bits = _bits(mask)[:, :, :N]                                  # [R, node, ancestor]
    parent = torch.where(bits & (i < i[:, None]), i, -1).amax(-1)
    sampled, tokens = s["sampled"][at], s["tokens"][at]
    agrees = (parent >= 0) & (sampled.gather(1, parent.clamp(min=0)) == tokens)
    agrees = agrees & (mask == mask.gather(1, parent.clamp(min=0)) | (1 << i))
    agrees[:, 0] = mask[:, 0] == 1
    taken = real & ~(bits & ~agrees[:, None, :]).any(-1)
    depth = bits.sum(-1)
    best = (torch.where(taken, depth, 0) * N + (N - 1 - i)).argmax(1)
    some = taken.any(1)
    on_path = bits[torch.arange(R, device="cuda"), best] & some[:, None]
    counts = on_path.sum(1)
    order = torch.where(on_path, i, N).sort(1).values
    path = torch.full((R, MOST_NODES), -1, dtype=torch.int32, device="cuda")
    path[:, :N] = torch.where(order < N, order, -1).to(torch.int32)
    out = torch.full((R, MOST_NODES), -1, dtype=torch.int32, device="cuda")
    out[:, :N] = torch.where(order < N, sampled.gather(1, order.clamp(max=N - 1)), -1)
    # rows of the path move to the first places behind the committed ones; the others stay (here: row 0 onto itself)
    c = s["ctx_len"].long() - (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    moved = order < N
    source = c[:, None] + torch.where(moved, order, 0)
    target = c[:, None] + torch.where(moved, i, 0)
    table = s["table"].long()
    rows = s["kv"][:, :, table.gather(1, source // PAGE), :, source % PAGE]
    s["kv"][:, :, table.gather(1, target // PAGE), :, target % PAGE] = rows
    return {"counts": counts.to(torch.int32), "path": path, "tokens": out, "kv": s["kv"]}


def _fork_plain(s):
    source, target = torch.tensor(s["pairs"], device="cuda").unbind(1)
    s["kv"][:, :, target] = s["kv"][:, :, source]
    return s["kv"]


# ---- what a pass cannot do without, and what it should give ---------------------------------------------------------


def work(case):
    H, KV, dh, layers = MODELS[case["model"]]
    size = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "fork":
        return {"bytes": 2 * case["pages"] * layers * 2 * KV * PAGE * dh * size, "flops": 0}
    counts = _counts(case)
    if case["op"] == "accept":
        rows = sum(_accepted(r, n, case["depth"]) for r, n in enumerate(counts))
        # accepted rows are read and written, but for those that lie in place already (about half); ids, masks and answers
        return {"bytes": rows * layers * 2 * KV * dh * size + sum(counts) * 16 + len(counts) * (2 * MOST_NODES + 1) * 4, "flops": 0}
    committed = _spread(case["shortest"], case["longest"], case["requests"])
    window = case.get("window", 0)
    seen = [min(c, window) if window else c for c in committed]
    rows = sum(c + n for c, n in zip(seen, counts))
    return {"bytes": rows * 2 * KV * dh * size + sum(counts) * (2 * H * dh * size + 8),
            "flops": 4 * H * dh * sum(n * (c + (n + 1) // 2) for c, n in zip(seen, counts))}


def exact(case, seed):
    """The attention of each request by itself in 64 bits; the other operators move numbers and compute none."""
    if case["op"] != "attention":
        return None
    s = prepare(case, seed)
    H, KV, dh, _ = MODELS[case["model"]]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begins, held, masks = s["cu_q"].tolist(), s["ctx_len"].tolist(), s["mask"].tolist()
    for r, length in enumerate(held):
        a, b = begins[r], begins[r + 1]
        c = length - (b - a)
        pages = s["table"][r, :-(-length // PAGE)].long()
        place = list(range(c)) + [c + bin(masks[t] & (1 << 64) - 1).count("1") - 1 for t in range(a, b)]
        place = torch.tensor(place, device="cuda")
        sees = torch.ones(b - a, length, dtype=torch.bool)
        sees[:, c:] = torch.tensor([[masks[t] >> k & 1 for k in range(b - a)] for t in range(a, b)]) == 1
        sees = sees.cuda()
        if s["window"]:
            sees &= place[c:, None] - place[None, :] < s["window"]
        for g in range(KV):
            k = s["k"][pages, g].reshape(-1, dh)[:length].double()
            v = s["v"][pages, g].reshape(-1, dh)[:length].double()
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                x = s["q"][a:b, h * dh:(h + 1) * dh].double() @ k.t() * s["scale"]
                out[a:b, h * dh:(h + 1) * dh] = torch.softmax(x.masked_fill(~sees, -math.inf), -1) @ v
    return out
