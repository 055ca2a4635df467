"""The operators of a batch whose requests answer with drafted trees, case by case: each tree's positions and ancestors
from its parents, the attention of its nodes over the paged cache, the rules on the logits of every node (penalties for
repeated tokens, biases, grammar masks) with the token chosen, and the walk down the tree that keeps the accepted nodes.

Where `own` is false `run` computes them in elementary torch operations in 32 bits; where it is true it calls
edgeexpert_b200.drafts and edgeexpert_b200.sampling, as a serving loop does."""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases ----
def _plan(name, requests, nodes, history, spare):
    return {"name": name, "op": "plan", "requests": requests, "nodes_min": nodes[0], "nodes_max": nodes[1],
            "history_min": history[0], "history_max": history[1], "spare": spare}


def _attention(name, requests, nodes, history, prefix, heads, kv_heads, dim, dtype, page, window):
    return {"name": name, "op": "attention", "requests": requests, "nodes_min": nodes[0], "nodes_max": nodes[1],
            "history_min": history[0], "history_max": history[1], "prefix": prefix, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "window": window}


def _logits(name, requests, nodes, vocab, dtype, history, biases, grammar):
    return {"name": name, "op": "logits", "requests": requests, "nodes_min": nodes[0], "nodes_max": nodes[1],
            "vocab": vocab, "dtype": dtype, "history_min": history[0], "history_max": history[1], "biases": biases,
            "grammar": grammar}


def _accept(name, requests, nodes, history, layers, kv_heads, dim, dtype, page, given):
    return {"name": name, "op": "accept", "requests": requests, "nodes_min": nodes[0], "nodes_max": nodes[1],
            "history_min": history[0], "history_max": history[1], "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "page": page, "given": given}


def listed():
    return [
        # one user's step with a tree of 12: latency
        _plan("plan-1", 1, (12, 12), (700, 700), 0),
        # a busy server: hundreds of trees of all sizes, a few rows of padding
        _plan("plan-301", 301, (1, 64), (0, 4000), 37),
        # the decoder's own layer at batch 1: 16 query and 8 KV heads of 256, a tree of 12
        _attention("attention-1", 1, (12, 12), (700, 700), 0, 16, 8, 256, "fp16", 16, 0),
        # a step of 256 rows: 16 users with trees of 16, no shared prompt
        _attention("attention-16", 16, (16, 16), (1, 4096), 0, 16, 8, 256, "fp16", 16, 0),
        # 24 users behind a shared prompt of 4096, trees of 20 to 40
        _attention("attention-prompt-24", 24, (20, 40), (1, 1000), 4096, 16, 4, 128, "bf16", 32, 0),
        # small ragged trees, eight query heads to a KV head, a sliding window over prompt and history
        _attention("attention-window-61", 61, (1, 5), (3, 3000), 501, 16, 2, 64, "bf16", 16, 1024),
        # long contexts: four users of up to 65536 positions with trees of 64
        _attention("attention-long-4", 4, (60, 64), (32768, 65536), 0, 16, 8, 256, "fp16", 64, 0),
        # one row of the decoder's vocabulary after a step without a tree
        _logits("logits-1", 1, (1, 1), 262144, "fp32", (500, 500), 5, False),
        # 16 users with trees of 16, every node under its own grammar state
        _logits("logits-256", 16, (16, 16), 262144, "fp32", (1, 4096), 300, True),
        # ragged batch of another vocabulary in 16 bits, most requests without a tree
        _logits("logits-bf16-61", 61, (1, 5), 100003, "bf16", (0, 30000), 40, True),
        # one user's tree of 12 in the decoder's 30 layers
        _accept("accept-1", 1, (12, 12), (700, 700), 30, 8, 256, "fp16", 16, False),
        # 32 users, trees of 8 to 24, some of the rows the end of a prompt
        _accept("accept-32", 32, (8, 24), (1, 200), 30, 8, 256, "fp16", 16, True),
    ]


HEADS = [(16, 8, 256), (16, 4, 128), (16, 2, 64), (8, 1, 128), (12, 4, 256), (4, 4, 80)]


def draw(rng):
    def spread(lo, hi):  # evenly over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["plan", "attention", "attention", "attention", "logits", "logits", "accept"])
    if op == "plan":
        most = spread(1, 256)
        requests = min(spread(1, 301), 10000 // most)
        c = _plan("", requests, (rng.randint(1, most), most), (0, spread(1, 4000)), rng.randint(0, 40))
    elif op == "attention":
        heads, kv_heads, dim = rng.choice(HEADS)
        most = spread(1, 100)
        requests = min(spread(1, 64), max(1, 1000 // most))
        history = (rng.randint(0, 3), min(spread(4, 65536), 200000 // requests))
        prefix = rng.choice([0, 0, spread(16, 4096) - rng.choice([0, 1, 7])])
        c = _attention("", requests, (rng.randint(1, most), most), history, prefix, heads, kv_heads, dim,
                       rng.choice(["fp16", "bf16"]), rng.choice([8, 16, 24, 32, 64, 128]),
                       rng.choice([0, 0, 512, 1024]))
    elif op == "logits":
        most = rng.choice([1, 1, spread(2, 64)])
        vocab = spread(1000, 262144)
        requests = min(spread(1, 128), max(1, 256 // most))
        c = _logits("", requests, (rng.randint(1, most), most), vocab, rng.choice(["fp32", "fp16", "bf16"]),
                    (0, spread(1, 30000)), rng.choice([0, spread(1, 300)]), rng.random() < 0.6)
    else:
        kv_heads, dim = rng.choice(HEADS)[1:]
        most = spread(1, 64)
        requests = min(spread(1, 32), max(1, 512 // most))
        c = _accept("", requests, (rng.randint(1, most), most), (0, spread(1, 200)), rng.randint(1, 30), kv_heads, dim,
                    rng.choice(["fp16", "bf16"]), rng.choice([1, 8, 16, 24, 64]), rng.random() < 0.5)
    del c["name"]
    return c


def _spaced(lo, hi, n):
    """n whole numbers from lo to hi, evenly: the same ones for every seed, which only deals them out."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _ceil(a, b):
    return -(-a // b)


def work(c):
    B = c["requests"]
    nodes, hist = _spaced(c["nodes_min"], c["nodes_max"], B), _spaced(c["history_min"], c["history_max"], B)
    T = sum(nodes)
    if c["op"] == "plan":
        words = _ceil(c["nodes_max"], 32)
        return {"bytes": 4 * T + 8 * B + (T + c["spare"]) * 4 * (1 + words), "flops": 0}
    if c["op"] == "attention":
        W, P, row = c["window"] or 1 << 40, c["prefix"], c["heads"] * c["dim"]
        mean = T / B
        depth = math.log(mean) + 1  # of a random tree's node, about
        keys = sum(min(h, W) + mean for h in hist) + max(0, min(P, W - 1 - min(hist)))
        seen = sum(mean * (min(h + P, W - 1) + depth) for h in hist)
        nbytes = keys * c["kv_heads"] * c["dim"] * 4 + T * (row * 4 + c["heads"] * 4 + 4 * _ceil(c["nodes_max"], 32))
        return {"bytes": nbytes + keys / c["page"] * 4 + 8 * B, "flops": 4 * row * seen}
    if c["op"] == "logits":
        size = 4 if c["dtype"] == "fp32" else 2
        nbytes = T * c["vocab"] * (2 * size) + 4 * sum(hist) + 8 * B * c["biases"] + 12 * T + 24 * B
        nbytes += T // 2 * (c["vocab"] / 8) if c["grammar"] else 0
        return {"bytes": nbytes, "flops": 0}
    # a path of ln(n) nodes behind the root is moved, about, in every layer
    moved = sum(math.log(n) for n in nodes) * c["layers"] * c["kv_heads"] * c["dim"] * 4
    return {"bytes": 2 * moved + 12 * T + 16 * B + 8 * B * c["nodes_max"], "flops": 0}


# --------------------------------------------------------------- inputs ----
def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    host = torch.Generator().manual_seed(seed * 104729 + 5)
    B = c["requests"]
    nodes = torch.tensor(_spaced(c["nodes_min"], c["nodes_max"], B))[torch.randperm(B, generator=host)]
    hist = torch.tensor(_spaced(c["history_min"], c["history_max"], B))[torch.randperm(B, generator=host)]
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), nodes.cumsum(0)])
    T, most = int(starts[-1]), c["nodes_max"]
    # every node under one of the nodes before it, any of them: trees that are a few levels deep
    index = torch.cat([torch.arange(n) for n in nodes.tolist()])
    parents = (torch.rand(T, generator=host, dtype=torch.float64) * index).long()
    parents[index == 0] = -1
    s = dict(op=c["op"], most=most, words=_ceil(most, 32), nodes=nodes, hist=hist, parents_host=parents,
             index=index, starts_host=starts, parents=_i32(parents), lens=_i32(hist + nodes), starts=_i32(starts))
    return {"plan": _prepare_plan, "attention": _prepare_attention, "logits": _prepare_logits,
            "accept": _prepare_accept}[c["op"]](c, s, gen, host)


def _i32(t):
    return t.to(device="cuda", dtype=torch.int32)


def _ancestors(s):
    """int32 [T][words]: bit i of a row is node i of its request, on the way from the root to the row's node."""
    parents, starts = s["parents_host"].tolist(), s["starts_host"].tolist()
    rows = []
    for a, z in zip(starts, starts[1:]):
        for t in range(a, z):
            rows.append((1 << (t - a)) | (rows[a + parents[t]] if parents[t] >= 0 else 0))
    words = [[(r >> (32 * w)) & 0xFFFFFFFF for w in range(s["words"])] for r in rows]
    t = torch.tensor(words, dtype=torch.int64)
    return _i32(torch.where(t >= 1 << 31, t - (1 << 32), t)), [bin(r).count("1") - 1 for r in rows]


def _paged(c, lens, host, spare=8):
    """Page table of requests of these lengths, the number of pages, and the prefix's pages."""
    ps, B = c["page"], len(lens)
    held, shared = (lens + ps - 1) // ps, _ceil(c.get("prefix", 0), ps)
    used, total = shared + int(held.sum()), shared + spare  # a pool of one size, however the lengths are dealt
    total += sum(_ceil(n, ps) for n in _spaced(c["history_min"], c["history_max"], B))
    total += sum(n // ps + 1 for n in _spaced(c["nodes_min"], c["nodes_max"], B))
    ids = torch.randperm(total, generator=host).to(torch.int32)  # pages lie anywhere
    width = _ceil(c["history_max"] + c["nodes_max"], ps)
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[torch.arange(width)[None, :] < held[:, None]] = ids[shared:used]
    return table.cuda(), total, ids[:shared].cuda()


def _prepare_plan(c, s, gen, host):
    T = int(s["starts_host"][-1]) + c["spare"]
    s["parents"] = torch.cat([s["parents"], torch.full((c["spare"],), -1, dtype=torch.int32, device="cuda")])
    s.update(base=c["history_max"] // 3, positions=_i32(torch.zeros(T)), ancestors=_i32(torch.zeros(T, s["words"])))
    if own:
        from edgeexpert_b200.drafts import DraftTree
        s["handle"] = DraftTree()
    return s


def _prepare_attention(c, s, gen, host):
    nq, nkv, hd, dt = c["heads"], c["kv_heads"], c["dim"], DTYPES[c["dtype"]]
    T = int(s["starts_host"][-1])
    s["table"], pages, s["prefix_pages"] = _paged(c, s["hist"] + s["nodes"], host)

    def normal(std, *shape):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(0, std, generator=gen)

    s["ancestors"], depth = _ancestors(s)
    s["positions"] = _i32(c["prefix"] + s["hist"].repeat_interleave(s["nodes"]) + torch.tensor(depth))
    s.update(prefix=c["prefix"], window=c["window"], scale=hd ** -0.5, longest=c["history_max"] + c["nodes_max"],
             q=normal(1.5, T, nq, hd), k=normal(1.0, pages, c["page"], nkv, hd),
             v=normal(1.0, pages, c["page"], nkv, hd), out=torch.zeros(T, nq, hd, dtype=dt, device="cuda"),
             lse=torch.zeros(T, nq, device="cuda"))
    if own:
        from edgeexpert_b200.drafts import TreeAttention
        from edgeexpert_b200.paged import PagedKV
        s["handle"], s["kv"] = TreeAttention(), PagedKV(s["k"], s["v"])
        s["workspace"] = torch.empty(s["handle"].workspace_bytes(s["kv"], nq, T, c["requests"], c["prefix"], s["most"]),
                                     dtype=torch.uint8, device="cuda")
    return s


def _tokens(n, vocab, host):
    """Token ids as text has them: a few very often, most hardly ever."""
    return (torch.rand(n, generator=host, dtype=torch.float64) ** 4 * vocab).long()


def _prepare_logits(c, s, gen, host):
    B, V, T, longest = c["requests"], c["vocab"], int(s["starts_host"][-1]), max(1, c["history_max"])
    logits = torch.empty(T, V, dtype=DTYPES[c["dtype"]], device="cuda").normal_(0, 4, generator=gen)
    uniform = torch.rand(3, B, generator=host)
    count = torch.randint(c["biases"] // 2, c["biases"] + 1, (B,), generator=host)
    biased = [torch.randperm(V, generator=host)[:n] for n in count.tolist()] if c["biases"] else []
    s.update(logits=logits, out=torch.zeros_like(logits), tokens=_i32(torch.zeros(T)),
             history=_i32(_tokens(B * longest, V, host).view(B, longest)), history_lens=_i32(s["hist"]),
             prompt_lens=_i32(s["hist"] * uniform[2]), repetition=(1 + 0.3 * uniform[0]).cuda(),
             presence=(uniform[1] - 0.2).cuda(), frequency=(0.5 * uniform[2] - 0.1).cuda(),
             bias_starts=None, bias_tokens=None, bias_values=None, allowed=None, allowed_rows=None,
             drafted=None, ancestors=None)
    if c["biases"]:
        s["bias_starts"] = _i32(torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)]))
        s["bias_tokens"] = _i32(torch.cat(biased))
        values = torch.randn(int(count.sum()), generator=host) * 5
        values[torch.rand(len(values), generator=host) < 0.2] = -math.inf  # tokens that are never wanted
        s["bias_values"] = values.cuda()
    if c["grammar"]:  # every second row is under a grammar; some states allow most tokens, some a few
        words = _ceil(V, 32)
        share = torch.rand(T // 2, 1, generator=gen, device="cuda") ** 3
        bits = [(torch.rand(T // 2, words, generator=gen, device="cuda") < share).int() << i for i in range(32)]
        s["allowed"] = torch.stack(bits).sum(0, dtype=torch.int32) if T > 1 else _i32(torch.zeros(1, words))
        rows = torch.full((T,), -1)
        rows[torch.randperm(T, generator=host)[:T // 2]] = torch.randperm(T // 2, generator=host)
        s["allowed_rows"] = _i32(rows)
    if c["nodes_max"] > 1:
        s["ancestors"], _ = _ancestors(s)
        s["drafted"] = _i32(_tokens(T, V, host))
    if own:
        from edgeexpert_b200.sampling import LogitRules
        s["handle"] = LogitRules()
        biases = 0 if s["bias_tokens"] is None else s["bias_tokens"].numel()
        s["workspace"] = torch.empty(s["handle"].workspace_bytes(T, V, B, longest, biases), dtype=torch.uint8, device="cuda")
    return s


def _prepare_accept(c, s, gen, host):
    B, T, most, ps = c["requests"], int(s["starts_host"][-1]), s["most"], c["page"]
    parents, starts, nodes = s["parents_host"].tolist(), s["starts_host"].tolist(), s["nodes"].tolist()
    drafted = torch.randint(0, 262144, (T,), generator=host)
    choices = torch.randint(262144, 300000, (T,), generator=host)  # nothing that was drafted
    given = torch.ones(B, dtype=torch.int64)
    if c["given"]:  # every fourth request brings the end of a prompt, then its tree
        given[::4] = (s["nodes"][::4] + 1) // 2
    for b, a in enumerate(starts[:-1]):
        first = int(given[b])
        for i in range(1, first):
            parents[a + i] = i - 1
        paths = {first - 1: list(range(first))}
        for i in range(first, nodes[b]):
            parents[a + i] = max(parents[a + i], first - 1)
            paths[i] = paths[parents[a + i]] + [i]
        # the longest way that moves no node onto another of its nodes: a pass leaves what the next needs
        best = max((p for p in paths.values() if len(p) == first or p[first] >= len(p)), key=lambda p: (len(p), p))
        for i, j in zip(best[first - 1:], best[first:]):
            choices[a + i] = drafted[a + j]
    s["table"], pages, _ = _paged(c, s["hist"] + s["nodes"], host)

    def normal():
        shape = (c["layers"], pages, ps, c["kv_heads"], c["dim"])
        return torch.empty(*shape, dtype=DTYPES[c["dtype"]], device="cuda").normal_(0, 1, generator=gen)

    s.update(page=ps, parents=_i32(torch.tensor(parents)), drafted=_i32(drafted), choices=_i32(choices),
             given=_i32(given) if c["given"] else None, k=normal(), v=normal(), counts=_i32(torch.zeros(B)),
             paths=_i32(torch.zeros(B, most)), tokens=_i32(torch.zeros(B, most)), targets=_i32(torch.zeros(B)))
    if own:
        from edgeexpert_b200.drafts import DraftAccept
        from edgeexpert_b200.paged import PagedKVLayers
        s["handle"], s["layers"] = DraftAccept(), PagedKVLayers(s["k"], s["v"])
    return s


# ------------------------------------------------------------------ run ----
def run(s):
    if own:
        return {"plan": _own_plan, "attention": _own_attention, "logits": _own_logits, "accept": _own_accept}[s["op"]](s)
    return {"plan": _plain_plan, "attention": _plain_attention, "logits": _plain_logits,
            "accept": _plain_accept}[s["op"]](s)


def _own_plan(s):
    s["handle"].encode_plan(s["parents"], s["lens"], s["starts"], s["positions"], s["ancestors"], s["most"],
                            position_base=s["base"])
    return s["positions"], s["ancestors"]


def _own_attention(s):
    s["handle"].encode(s["q"], s["kv"], s["table"], s["lens"], s["starts"], s["ancestors"], s["out"], s["workspace"],
                       prefix_pages=s["prefix_pages"], prefix_len=s["prefix"], max_query=s["most"], scale=s["scale"],
                       window=s["window"], positions=s["positions"], lse=s["lse"])
    return s["out"], s["lse"]


def _own_logits(s):
    s["handle"].encode(s["logits"], s["out"], s["starts"], s["workspace"], max_query=s["most"], history=s["history"],
                       history_lens=s["history_lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
                       presence=s["presence"], frequency=s["frequency"], bias_starts=s["bias_starts"],
                       bias_tokens=s["bias_tokens"], bias_values=s["bias_values"], allowed=s["allowed"],
                       allowed_rows=s["allowed_rows"], token_ids=s["drafted"], ancestors=s["ancestors"],
                       tokens=s["tokens"])
    return s["out"], s["tokens"]


def _own_accept(s):
    s["handle"].encode(s["drafted"], s["parents"], s["choices"], s["lens"], s["starts"], s["counts"], s["paths"],
                       s["tokens"], s["targets"], max_query=s["most"], given=s["given"], layers=s["layers"],
                       page_table=s["table"])
    return s["counts"], s["paths"], s["tokens"], s["targets"], s["k"], s["v"]


def _rows(s, T):
    """Request of each of T rows, its place in the request, and whether it has one."""
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    live = b < s["lens"].numel()
    b = b.clamp(max=s["lens"].numel() - 1)
    return b, t - s["starts"].long()[b], live


def _padded(s, x, fill):
    """x [T...] as [requests][most...], `fill` beyond a request's nodes."""
    start, end = s["starts"][:-1].long(), s["starts"][1:].long()
    j = torch.arange(s["most"], device="cuda")
    at = start[:, None] + j
    inside = at < end[:, None]
    return torch.where(inside, x[at.clamp(max=x.shape[0] - 1)].long(), fill), inside


def _twice(reach):
    return ((reach @ reach) > 0).float()


def _reach(parents):
    """[requests][most][most]: node j is on the way to node i, from the parents [requests][most]."""
    j = torch.arange(parents.shape[1], device="cuda")
    one = ((parents[:, :, None] == j) | (j[:, None] == j)).float()
    return _twice(_twice(_twice(_twice(_twice(_twice(_twice(_twice(one)))))))) > 0  # ways of up to 256 nodes


def _plain_plan(s):
    parents, _ = _padded(s, s["parents"], -1)
    b, j, live = _rows(s, s["parents"].numel())
    reach = _reach(parents)
    depth = reach.sum(-1) - 1
    history = s["lens"].long() - (s["starts"][1:] - s["starts"][:-1]).long()
    at = j.clamp(max=s["most"] - 1)
    s["positions"].copy_(torch.where(live, s["base"] + history[b] + depth[b, at], -1))
    bits = torch.nn.functional.pad(reach[b, at] & live[:, None], (0, s["words"] * 32 - s["most"]))
    weight = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
    s["ancestors"].copy_((bits.view(-1, s["words"], 32) * weight).sum(-1))  # (the low 32 bits are kept)
    return s["positions"], s["ancestors"]


def _plain_attention(s):
    q, P, (T, nq, hd) = s["q"].float(), s["prefix"], s["q"].shape
    nkv, B, n = s["k"].shape[2], s["lens"].numel(), s["most"]
    start, count = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    j = torch.arange(n, device=q.device)
    at = (start[:, None] + j).clamp(max=T - 1)
    rows = q[at].view(B, n, nkv, nq // nkv, hd)
    table = s["table"].clamp(min=0).long()
    history = P + s["lens"].long() - count

    def shared(x):
        return x[s["prefix_pages"].long()].flatten(0, 1)[:P].float()

    def mine(x):
        return x[table].flatten(1, 2)[:, :s["longest"]].float()

    scores = torch.cat([torch.einsum("bnkgd,pkd->bkgnp", rows, shared(s["k"])),
                        torch.einsum("bnkgd,bpkd->bkgnp", rows, mine(s["k"]))], -1) * s["scale"]
    key = torch.arange(P + s["longest"], device=q.device)
    node = key - history[:, None]  # [B][keys]: the node that a key is, if it is one
    word = s["ancestors"][at].long()  # [B][n][words]
    where = node.clamp(0, s["words"] * 32 - 1)
    bit = (torch.gather(word, 2, (where // 32)[:, None, :].expand(B, n, -1)) >> (where % 32)[:, None, :]) & 1
    seen = (node < 0)[:, None, :].expand(B, n, -1)
    if s["window"]:
        seen = seen & (key > s["positions"][at].long()[:, :, None] - s["window"])
    seen = seen | ((node >= 0) & (node < count[:, None]))[:, None, :] & (bit > 0)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    # what the masks leave out has weight 0, and lies in pages that other requests have written
    out = torch.einsum("bkgnp,pkd->bnkgd", scores[..., :P], shared(s["v"]))
    out += torch.einsum("bkgnp,bpkd->bnkgd", scores[..., P:], mine(s["v"]))
    out = (out / total.permute(0, 3, 1, 2, 4)).reshape(B, n, nq, hd)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(B, n, nq)
    b, i, _ = _rows(s, T)
    s["out"].copy_(out[b, i])
    s["lse"].copy_(lse[b, i])
    return s["out"], s["lse"]


def _plain_logits(s):
    (T, V), B = s["logits"].shape, s["lens"].numel()
    b, _, _ = _rows(s, T)
    where = torch.arange(s["history"].shape[1], device="cuda")
    inside, prompt = where < s["history_lens"][:, None], where < s["prompt_lens"][:, None]
    tokens = s["history"].long()
    said = torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, (inside & ~prompt).float())
    asked = torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, (inside & prompt).float())
    count, seen = said[b], asked[b] > 0
    if s["ancestors"] is not None:  # the drafted tokens down to a row's node are said too
        node = torch.arange(s["most"], device="cuda")
        path = (s["ancestors"].long()[:, node // 32] >> (node % 32)) & 1
        drafted, _ = _padded(s, s["drafted"], 0)
        count.scatter_add_(1, drafted[b], path.float())
    z = s["logits"].float()
    rep = s["repetition"][b, None]
    z = torch.where(seen | (count > 0), torch.where(z > 0, z / rep, z * rep), z)
    z = z - s["frequency"][b, None] * count
    z = torch.where(count > 0, z - s["presence"][b, None], z)
    if s["bias_starts"] is not None:
        entry = torch.arange(s["bias_tokens"].numel(), device="cuda")
        whose = torch.searchsorted(s["bias_starts"][1:].long(), entry, right=True)
        bias = torch.zeros(B, V, device="cuda")
        bias[whose, s["bias_tokens"].long()] = s["bias_values"]
        z = z + bias[b]
    if s["allowed"] is not None:
        v = torch.arange(V, device="cuda")
        rows = s["allowed_rows"].long()
        ok = (s["allowed"][rows.clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        z = torch.where((ok > 0) | (rows < 0)[:, None], z, -math.inf)
    best, token = z.max(-1)
    first = torch.where(z == best[:, None], torch.arange(V, device="cuda"), V).amin(-1)  # ties to the lowest
    s["out"].copy_(z)
    s["tokens"].copy_(torch.where(best > -math.inf, first, -1))
    return s["out"], s["tokens"]


def _plain_accept(s):
    most, B = s["most"], s["lens"].numel()
    parents, inside = _padded(s, s["parents"], -1)
    drafted, _ = _padded(s, s["drafted"], -1)
    choices, _ = _padded(s, s["choices"], -2)
    j = torch.arange(most, device="cuda")
    given = torch.ones_like(s["lens"]).long() if s["given"] is None else s["given"].long()
    fits = inside & (parents >= 0) & (choices.gather(1, parents.clamp(min=0)) == drafted)
    twins = fits[:, None, :] & (parents[:, :, None] == parents[:, None, :]) & (j < j[:, None])
    # the walk begins at the last node that was given
    ok = (fits & ~twins.any(-1) & (parents >= given[:, None] - 1)) | (j < given[:, None])
    kept = inside & ~(_reach(parents) & ~ok[:, None, :]).any(-1)
    count = kept.sum(-1)
    path = torch.where(kept, j, most).sort(-1).values
    live = j < count[:, None]
    path = torch.where(live, path, -1)
    answer = choices.gather(1, path.clamp(min=0))
    new = j < (count - given + 1)[:, None]
    answer = torch.where(new, answer.gather(1, (j + given[:, None] - 1).clamp(max=most - 1)), -1)
    history = s["lens"].long() - (s["starts"][1:] - s["starts"][:-1]).long()
    move = live & (path != j)
    whose, to = move.nonzero(as_tuple=True)
    source, target = history[whose] + path[whose, to], history[whose] + to
    ps, table = s["page"], s["table"].long()
    for x in (s["k"], s["v"]):
        x[:, table[whose, target // ps], target % ps] = x[:, table[whose, source // ps], source % ps]
    s["counts"].copy_(count)
    s["paths"].copy_(path)
    s["tokens"].copy_(answer)
    s["targets"].copy_(torch.where(count > 0, history + count, -1))
    return s["counts"], s["paths"], s["tokens"], s["targets"], s["k"], s["v"]


# ---------------------------------------------------------------- exact ----
def exact(c, seed):
    if c["op"] == "plan":
        return None  # whole numbers
    s = prepare(c, seed)
    if c["op"] == "attention":
        return _exact_attention(c, s)
    if c["op"] == "logits":
        return _exact_logits(s), None
    return (None, None, None, None, *_exact_moves(s))


def _way(parents, i):
    """The nodes from the root to node i of one tree."""
    way = [i]
    while parents[way[-1]] >= 0:
        way.append(parents[way[-1]])
    return way[::-1]


def _exact_attention(c, s):
    out, lse = torch.zeros_like(s["out"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
    group, ps = c["heads"] // c["kv_heads"], c["page"]
    starts, nodes, hist = s["starts_host"].tolist(), s["nodes"].tolist(), s["hist"].tolist()
    for b in range(c["requests"]):
        pages = s["table"][b, :_ceil(hist[b] + nodes[b], ps)].long()

        def sequence(x):  # [position][head][dim]: the prefix, the history, the nodes
            front = x[s["prefix_pages"].long()].reshape(-1, *x.shape[2:])[:c["prefix"]]
            return torch.cat([front, x[pages].reshape(-1, *x.shape[2:])[:hist[b] + nodes[b]]]).double()

        k, v, past = sequence(s["k"]), sequence(s["v"]), c["prefix"] + hist[b]
        a = starts[b]
        parents = s["parents_host"][a:a + nodes[b]].tolist()
        mask = torch.full((nodes[b], len(k)), -math.inf, dtype=torch.float64)
        for i in range(nodes[b]):
            way = _way(parents, i)
            mask[i, max(0, past + len(way) - c["window"]) if c["window"] else 0:past] = 0
            mask[i, [past + x for x in way]] = 0
        mask = mask.cuda()
        for h in range(c["heads"]):
            z = s["q"][a:a + nodes[b], h].double() @ k[:, h // group].T * s["scale"] + mask
            lse[a:a + nodes[b], h] = torch.logsumexp(z, -1)
            out[a:a + nodes[b], h] = torch.softmax(z, -1) @ v[:, h // group]
    return out, lse


def _exact_logits(s):
    V, starts = s["logits"].shape[1], s["starts_host"].tolist()
    out = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
    biases = s["bias_starts"].tolist() if s["bias_starts"] is not None else None
    rep, pres, freq = (s[k].double().tolist() for k in ("repetition", "presence", "frequency"))
    for b, (a, e) in enumerate(zip(starts, starts[1:])):
        n, prompt = int(s["history_lens"][b]), int(s["prompt_lens"][b])
        words = s["history"][b, :n].long()
        asked = torch.bincount(words[:prompt], minlength=V)
        said = torch.bincount(words[prompt:], minlength=V)
        parents = s["parents_host"][a:e].tolist()
        for t in range(a, e):
            more = said
            if s["drafted"] is not None:
                way = torch.tensor(_way(parents, t - a), device="cuda") + a
                more = said + torch.bincount(s["drafted"][way].long(), minlength=V)
            z = s["logits"][t].double()
            repeated = (more + asked) > 0
            z[repeated] *= torch.where(z[repeated] > 0, 1 / rep[b], rep[b])
            z -= freq[b] * more
            z[more > 0] -= pres[b]
            if biases is not None:
                part = slice(biases[b], biases[b + 1])
                z[s["bias_tokens"][part].long()] += s["bias_values"][part].double()
            if s["allowed"] is not None and int(s["allowed_rows"][t]) >= 0:
                bits = s["allowed"][int(s["allowed_rows"][t])]
                lanes = torch.arange(32, device="cuda")
                z[((bits[:, None] >> lanes) & 1).reshape(-1)[:V] == 0] = -math.inf
            out[t] = z
    return out


def _exact_moves(s):
    k, v, ps = s["k"].double(), s["v"].double(), s["page"]
    parents, drafted, choices, starts = (s[x].tolist() for x in ("parents", "drafted", "choices", "starts"))
    for b, (a, e) in enumerate(zip(starts, starts[1:])):
        path = list(range(1 if s["given"] is None else int(s["given"][b])))
        while True:
            after = [i for i in range(len(path), e - a)
                     if parents[a + i] == path[-1] and drafted[a + i] == choices[a + path[-1]]]
            if not after:
                break
            path.append(after[0])
        history, pages = int(s["hist"][b]), s["table"][b].tolist()
        for i, j in enumerate(path):
            to, at = history + i, history + j
            for x in (k, v):
                x[:, pages[to // ps], to % ps] = x[:, pages[at // ps], at % ps].clone()
    return k, v
