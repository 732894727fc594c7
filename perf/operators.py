"""The work of a decoding step that checks drafted tokens and draws from the logits: its calls at the sizes of this repository's
configurations, tests and benchmark.

Three parts of one step.  ``sample``: a token for each row of logits, from a given random number, under a temperature, top-k, top-p
and min-p of the row's own.  ``tree``: attention of a tree of drafted tokens over the paged cache that holds the context and the
drafted tokens.  ``accept``: which drafted tokens the model's own choices confirm, and their keys and values moved side by side in
every layer's pool.

``listed()`` are the cases, ``draw`` gives more of the same ranges, ``prepare`` makes what a program has in hand before the call,
``run`` is one pass - through the framework's entry points where ``own`` is true, in elementary torch otherwise -, ``exact`` the
attention in float64 and the pools after the moves, ``work`` what a pass cannot do without.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one conversation: the engine surface's default choice (temperature 0.7, top-k 50, top-p 0.9) over the 8B shape's vocabulary
        dict(name="sample_one", kind="sample", rows=1, vocab=128256, dtype="bf16", how="chat"),
        # the headline batch, every request with settings of its own: greedy rows, all four limits, masked tokens
        dict(name="sample_batch", kind="sample", rows=64, vocab=128256, dtype="bf16", how="mixed"),
        # the nodes of many draft trees, logits in 32 bits, a nucleus of a flat distribution: thousands of tokens are kept
        dict(name="sample_nucleus", kind="sample", rows=256, vocab=128256, dtype="fp32", how="nucleus"),
        # an odd vocabulary, no limit but a temperature: the draw goes over all tokens
        dict(name="sample_open", kind="sample", rows=37, vocab=32003, dtype="fp16", how="open"),
        # one sequence, a small tree over a short context: latency
        dict(name="tree_one", kind="tree", batch=1, nodes=8, heads=32, kv_heads=8, dim=128, context=160, page=16, ragged=False, dtype="bf16"),
        # the headline batch: 64 sequences at 2k, trees of 8
        dict(name="tree_batch", kind="tree", batch=64, nodes=8, heads=32, kv_heads=8, dim=128, context=2048, page=16, ragged=True, dtype="bf16"),
        # long contexts under wide trees in the 70B head layout: 512 query rows share a key
        dict(name="tree_long", kind="tree", batch=8, nodes=64, heads=64, kv_heads=8, dim=128, context=32768, page=16, ragged=False, dtype="bf16"),
        # heads with keys of their own, an odd number of nodes and odd contexts, larger pages
        dict(name="tree_own_keys", kind="tree", batch=16, nodes=5, heads=16, kv_heads=16, dim=64, context=3001, page=32, ragged=True, dtype="fp16"),
        # the small model of the parity path, 32 bits
        dict(name="tree_parity", kind="tree", batch=4, nodes=13, heads=8, kv_heads=2, dim=64, context=160, page=16, ragged=True, dtype="fp32"),
        # one sequence of the small model: 4 layers
        dict(name="accept_one", kind="accept", batch=1, nodes=8, accepted=3, layers=4, kv_heads=2, dim=64, page=16, dtype="fp32"),
        # the headline batch: 64 sequences, 32 layers of the 8B shape
        dict(name="accept_batch", kind="accept", batch=64, nodes=24, accepted=6, layers=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("sample", "sample", "tree", "tree", "tree", "accept"))
    if kind == "sample":
        dtype, vocab = rng.choice(("bf16", "bf16", "fp16", "fp32")), _spread(rng, 1000, 160000)
        return dict(kind=kind, rows=_spread(rng, 1, min(512, 32000000 // vocab)), vocab=vocab, dtype=dtype,
                    how=rng.choice(("chat", "mixed", "mixed", "nucleus", "open")))
    if kind == "accept":
        nodes = _spread(rng, 2, 64)
        return dict(kind=kind, batch=_spread(rng, 1, 64), nodes=nodes, accepted=rng.randint(1, min(nodes, 9)), layers=rng.choice((4, 16, 32)),
                    kv_heads=rng.choice((2, 8)), dim=rng.choice((64, 128)), page=rng.choice((16, 16, 32)), dtype=rng.choice(("bf16", "fp16")))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    kv, rep = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 5, 8))
    batch, nodes = _spread(rng, 1, 64), _spread(rng, 1, 64)
    context = _spread(rng, 30, max(64, min(32768, 2097152 // (kv * batch), 134217728 // (kv * rep * batch * nodes))))
    return dict(kind=kind, batch=batch, nodes=nodes, heads=kv * rep, kv_heads=kv, dim=rng.choice((64, 128, 128)), context=context,
                page=rng.choice((16, 16, 16, 32, 64)), ragged=rng.random() < 0.7, dtype=dtype)


# ---- inputs: made from the seed ---------------------------------------------------------------------------------------------------

def _settings(how, rows, rng):
    """(temperature, top-k, top-p, min-p) of each row."""
    if how == "chat":
        return [(0.7, 50, 0.9, 0.0)] * rows
    if how == "nucleus":
        return [(1.0, 0, 0.95, 0.0)] * rows
    if how == "open":
        return [(rng.uniform(0.6, 1.2), 0, 1.0, 0.0) for _ in range(rows)]
    return [(rng.choice((0.0, 0.3, 0.7, 1.0, 1.0, 1.5)), rng.choice((0, 0, 1, 20, 50, 1000)), rng.choice((1.0, 0.5, 0.9, 0.95, 0.99)),
             rng.choice((0.0, 0.0, 0.02, 0.1))) for _ in range(rows)]


def _trees(batch, nodes, rng):
    """Parents of each tree's nodes (-1: the root, node 0), children after parents; recent nodes have more children."""
    return [[-1] + [t - 1 - int((t - 1) * rng.random() ** 2.5) if rng.random() < 0.7 else rng.randrange(t) for t in range(1, nodes)]
            for _ in range(batch)]


def _ancestors(parents):
    """Bit masks: each node and those above it."""
    rows = []
    for tree in parents:
        seen = []
        for t, p in enumerate(tree):
            seen.append((1 << t) | (seen[p] if p >= 0 else 0))
        rows.append([m - (1 << 64) if m >> 63 else m for m in seen])
    return rows


def _pages(case, lens, most, g):
    """Block tables over pages in random order, and the number of pages: enough for sequences of `most` tokens."""
    per = -(-most // case["page"])
    need = [-(-n // case["page"]) for n in lens]
    pages = per * len(lens) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables, at = torch.zeros((len(lens), per), dtype=torch.int32, device=DEV), 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, pages


def prepare(case, seed):
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a bulk of unlikely tokens and a few that stand out; flat where the nucleus is to be wide
        x = torch.randn((rows, vocab), generator=g, device=DEV)
        x *= torch.empty((rows, 1), device=DEV).uniform_(1.0, 2.5, generator=g)
        if case["how"] != "nucleus":
            at = torch.randint(0, vocab, (rows, 24), generator=g, device=DEV)
            x.scatter_(1, at, 6.0 + 6.0 * torch.rand((rows, 24), generator=g, device=DEV))
        if case["how"] == "mixed":      # a grammar forbids some tokens of some rows
            x[::5].masked_fill_(torch.rand((len(range(0, rows, 5)), vocab), generator=g, device=DEV) < 0.3, -math.inf)
        t, k, p, m = zip(*_settings(case["how"], rows, rng))
        return dict(kind="sample", x=x.to(dtype), u=torch.rand(rows, generator=g, device=DEV), temperature=ints(t, torch.float32),
                    top_k=ints(k), top_p=ints(p, torch.float32), min_p=ints(m, torch.float32))
    batch, nodes = case["batch"], case["nodes"]
    parents = _trees(batch, nodes, rng)
    if case["kind"] == "tree":
        drafts = [rng.randint(max(1, nodes // 2), nodes) if case["ragged"] else nodes for _ in range(batch)]
        lens = [int(case["context"] * (rng.uniform(0.5, 1.0) if case["ragged"] else 1.0)) + n for n in drafts]
        tables, pages = _pages(case, lens, case["context"] + nodes, g)
        pool = (pages, case["kv_heads"], case["page"], case["dim"])
        return dict(kind="tree", q=torch.randn((batch, nodes, case["heads"], case["dim"]), generator=g, device=DEV).to(dtype),
                    k_pool=torch.randn(pool, generator=g, device=DEV, dtype=dtype), v_pool=torch.randn(pool, generator=g, device=DEV, dtype=dtype),
                    tables=tables, lens=ints(lens), visible=ints(_ancestors(parents), torch.int64), drafts=ints(drafts), longest=max(lens))
    # drafted tokens of which the model's choices confirm `accepted`, the root among them
    lens = [rng.randint(20, 60) + nodes for _ in range(batch)]
    tables, pages = _pages(case, lens, 60 + nodes, g)
    tokens = [[rng.randrange(1000, 100000) for _ in range(nodes)] for _ in range(batch)]
    chosen = [[rng.randrange(1000) for _ in range(nodes)] for _ in range(batch)]
    for b in range(batch):
        at, left = 0, case["accepted"] - 1
        while left > 0:
            children = [t for t in range(at + 1, nodes) if parents[b][t] == at]
            if not children:        # the tree ends here: its next node continues the path
                if at + 1 >= nodes:
                    break
                parents[b][at + 1] = at
                children = [at + 1]
            t = rng.choice(children)
            chosen[b][at] = tokens[b][t]
            at, left = t, left - 1
    pools = torch.randn((case["layers"], 2, pages, case["kv_heads"], case["page"], case["dim"]), generator=g, device=DEV, dtype=dtype)
    return dict(kind="accept", parents=ints(parents), tokens=ints(tokens, torch.int64), chosen=ints(chosen, torch.int64), tables=tables,
                lens=ints(lens), pools=pools, shape=tuple(pools.shape[2:]),
                k_ptrs=ints([pools[i, 0].data_ptr() for i in range(case["layers"])], torch.int64),
                v_ptrs=ints([pools[i, 1].data_ptr() for i in range(case["layers"])], torch.int64))


# ---- plain forms ------------------------------------------------------------------------------------------------------------------

def _plain_sample(s):
    """Weights exp((x - max) / temperature); the first k of the descending order, of these the first whose weights before them are below
    p of the sum, of these the ones of min_p of the largest weight at least; the first token in the row's order whose sum of kept weights
    passes u of the whole.  In 64 bits: the draw is next to a border between two tokens more often than 32 bits tell them apart."""
    x, u = s["x"].double(), s["u"].double()
    rows, vocab = x.shape
    top = x.max(1, keepdim=True).values
    t = s["temperature"].double()[:, None]
    w = torch.where(x == -math.inf, 0.0, torch.exp((x - top) / torch.where(t > 0, t, 1.0)))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = s["top_k"][:, None]
    place = torch.arange(vocab, device=x.device)[None]
    ws = torch.where((k <= 0) | (place < k), ws, 0.0)
    before = torch.cumsum(ws, 1) - ws
    p = s["top_p"].double()[:, None]
    ws = torch.where((p >= 1) | (before < p * ws.sum(1, keepdim=True)) | (place == 0), ws, 0.0)
    ws = torch.where((ws >= s["min_p"].double()[:, None]) | (place == 0), ws, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    total = torch.cumsum(kept, 1)
    drawn = (total <= u[:, None] * total[:, -1:]).sum(1)
    return torch.where(t[:, 0] > 0, drawn, order[:, 0])


def _plain_tree(s):
    """softmax(q k / sqrt(dim)) v over the context and the drafted tokens that a node sees; 0 for the rows behind a sequence's last node."""
    q, page = s["q"].float(), s["k_pool"].shape[2]
    batch, nodes, heads, dim = q.shape
    kv, pages = s["k_pool"].shape[1], -(-s["longest"] // page)
    k, v = (x[s["tables"][:, :pages].long()].float().transpose(2, 3).reshape(batch, pages * page, kv, dim) for x in (s["k_pool"], s["v_pool"]))
    n = s["drafts"][:, None, None]
    j = torch.arange(pages * page, device=q.device)[None, None] - (s["lens"][:, None, None] - n)      # the key's number among the drafted tokens
    keep = (j < 0) | ((j < n) & (s["visible"][:, :, None] >> j.clamp(0, 63) & 1 != 0))
    keep = keep & (torch.arange(nodes, device=q.device)[None, :, None] < n)
    scores = torch.einsum("bngrd,bkgd->bgrnk", q.view(batch, nodes, kv, heads // kv, dim) * dim ** -0.5, k)
    scores = scores.masked_fill(~keep[:, None, None], -math.inf)
    top = scores.max(-1, keepdim=True).values
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1)
    out = torch.einsum("bgrnk,bkgd->bngrd", w, v) / torch.where(total == 0, 1.0, total).permute(0, 3, 1, 2)[..., None]
    return out.reshape(batch, nodes, heads, dim).to(s["q"].dtype)


def _plain_accept(s):
    """A node is confirmed if its token is its parent's choice (of equal siblings the first) and all above it are; the i-th confirmed
    node's keys and values go to the i-th place behind the context."""
    parents, tokens, chosen, pools = s["parents"].long(), s["tokens"], s["chosen"], s["pools"]
    batch, nodes = parents.shape
    node = torch.arange(nodes, device=tokens.device)
    one_up = (parents[:, :, None] == node).float() + torch.eye(nodes, device=tokens.device)
    above = torch.linalg.matrix_power(one_up, 64) > 0       # up to 64 steps up
    visible = (above.long() << node).sum(-1)
    depth = (above.sum(-1) - 1).int()
    fits = (parents >= 0) & (tokens == chosen.gather(1, parents.clamp_min(0)))
    twin = (parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (node < node[:, None])
    fits = (fits & ~twin.any(-1)) | (node == 0)
    taken = ~(above & ~fits[:, None]).any(-1)
    count = taken.sum(1)
    path = torch.sort(torch.where(taken, node, nodes), 1).values
    live = path < nodes
    at = path.clamp_max(nodes - 1)
    out = torch.where(live, chosen.gather(1, at), -1)
    base = (s["lens"] - nodes).long()[:, None]
    page = pools.shape[4]

    def slot(place):
        return s["tables"].gather(1, place // page).long()[live], (place % page)[live]

    (sp, so), (dp, do) = slot(base + at), slot(base + torch.where(live, node, 0))
    pools[:, :, dp, :, do] = pools[:, :, sp, :, so]
    return dict(visible=visible, depth=depth, count=count.int(), path=torch.where(live, path, -1).int(), tokens=out,
                lens=(base[:, 0] + count).int(), pools=pools)


def run(state):
    s = state
    if own:
        import dgi_b200  # noqa: F401
        from dgi_b200 import ops

        if s["kind"] == "sample":
            return ops.sample_rows(s["x"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        if s["kind"] == "tree":
            return ops.paged_tree_attention(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["lens"], s["visible"], draft_lens=s["drafts"])
        visible, depth = ops.draft_tree(s["parents"])
        count, path, tokens, lens = ops.accept_drafts(s["tokens"], s["chosen"], s["parents"], visible, s["k_ptrs"], s["v_ptrs"], s["shape"],
                                                      s["pools"].dtype, s["tables"], s["lens"])
        return dict(visible=visible, depth=depth, count=count, path=path, tokens=tokens, lens=lens, pools=s["pools"])
    if s["kind"] == "sample":
        return _plain_sample(s)
    if s["kind"] == "tree":
        return _plain_tree(s)
    return _plain_accept(s)


def exact(case, seed):
    """The attention in 64 bits, a kv head and a sequence at a time; the pools after a walk down each tree and a copy per token.  Tokens
    and places are whole numbers and have no such value."""
    if case["kind"] == "sample":
        return None
    s = prepare(case, seed)
    if case["kind"] == "accept":
        tokens, chosen, parents, tables = (s[n].tolist() for n in ("tokens", "chosen", "parents", "tables"))
        pools, page = s["pools"].double(), case["page"]
        for b, length in enumerate(s["lens"].tolist()):
            at, place = 0, length - case["nodes"]
            while at is not None:
                src, dst = length - case["nodes"] + at, place
                if src != dst:
                    pools[:, :, tables[b][dst // page], :, dst % page] = pools[:, :, tables[b][src // page], :, src % page]
                at = next((t for t in range(at + 1, case["nodes"]) if parents[b][t] == at and tokens[b][t] == chosen[b][at]), None)
                place += 1
        return dict(visible=None, depth=None, count=None, path=None, tokens=None, lens=None, pools=pools)
    q, page, group = s["q"].double(), case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    lens, drafts, visible = s["lens"].tolist(), s["drafts"].tolist(), s["visible"].tolist()
    for b, (length, n) in enumerate(zip(lens, drafts)):
        where = torch.arange(length, device=DEV)
        rows = s["tables"][b].long()[where // page] * page + where % page
        hidden = torch.zeros((n, length), dtype=torch.float64, device=DEV)
        hidden[:, length - n:] = torch.tensor([[0.0 if visible[b][t] >> j & 1 else -math.inf for j in range(n)] for t in range(n)],
                                              dtype=torch.float64, device=DEV)
        for h in range(case["kv_heads"]):
            k = s["k_pool"][:, h].reshape(-1, case["dim"])[rows].double()
            v = s["v_pool"][:, h].reshape(-1, case["dim"])[rows].double()
            mine = q[b, :n, h * group:(h + 1) * group].reshape(n * group, -1)
            weights = torch.softmax(mine @ k.T / math.sqrt(case["dim"]) + hidden.repeat_interleave(group, 0), -1)
            out[b, :n, h * group:(h + 1) * group] = (weights @ v).view(n, group, -1)
    return out


def work(case):
    """Bytes that have to be read and written once, operations of the products or of the weights."""
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * 28, "flops": 4 * n}
    size, batch, nodes, row = SIZE[case["dtype"]], case["batch"], case["nodes"], case["kv_heads"] * case["dim"]
    if case["kind"] == "accept":
        return {"bytes": batch * (case["accepted"] - 1) * case["layers"] * 4 * row * size + batch * nodes * 44, "flops": batch * nodes}
    drafts, lens = (0.75 * nodes, 0.75 * case["context"]) if case["ragged"] else (nodes, case["context"])
    q = batch * drafts * case["heads"] * case["dim"]
    return {"bytes": 2 * batch * (lens + drafts) * row * size + 2 * q * size, "flops": 4 * q * (lens + drafts)}
