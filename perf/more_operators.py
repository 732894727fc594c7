"""A key/value cache held in 8 bits, with a scale for each page of tokens and kv head: its calls at the sizes of this repository's
configurations, tests and benchmark.

Four operators that one layer uses.  ``write``: queries and keys rotated, keys and values quantised into the pages behind a block table (whose
scales grow where a new token needs it), and the written pages read back.  ``read``: the first tokens of each sequence as dense keys and values.
``decode``: attention of one token per sequence over such a cache.  ``prompt``: causal attention of several new tokens per sequence.

``listed()`` are the cases, ``draw`` gives more of the same ranges, ``prepare`` makes what a program has in hand before the call,
``run`` is one pass - through the framework's entry points where ``own`` is true, in elementary torch otherwise -, ``exact`` the same by the
definition in float64, ``work`` what a pass cannot do without.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "e4m3": 448.0}      # the largest code
LEAST = 2.0 ** -60                         # the smallest scale


def listed():
    return [
        # one conversation's next token in the 8B head layout: latency
        dict(name="write_one", kind="write", batch=1, new=1, heads=32, kv_heads=8, dim=128, context=160, page=16, ragged=False, dtype="bf16", codes="int8"),
        # the headline batch's decode step: 64 tokens, most of them into pages that hold others already
        dict(name="write_batch", kind="write", batch=64, new=1, heads=32, kv_heads=8, dim=128, context=2048, page=16, ragged=True, dtype="bf16", codes="int8"),
        # the prompt pass of 8 sequences of the headline length
        dict(name="write_prompt", kind="write", batch=8, new=2048, heads=32, kv_heads=8, dim=128, context=0, page=16, ragged=False, dtype="bf16", codes="int8"),
        # heads with keys of their own, odd portions behind odd contexts, larger pages
        dict(name="write_odd", kind="write", batch=16, new=201, heads=16, kv_heads=16, dim=64, context=1001, page=32, ragged=True, dtype="fp16", codes="e4m3"),
        # a short cached prompt of one sequence
        dict(name="read_one", kind="read", batch=1, kv_heads=8, dim=128, context=160, page=16, dtype="bf16", codes="int8"),
        # the cached prompts of a batch, read for a pass that continues them
        dict(name="read_batch", kind="read", batch=8, kv_heads=8, dim=128, context=4096, page=16, dtype="bf16", codes="int8"),
        # one sequence, a short context: latency
        dict(name="decode_one", kind="decode", batch=1, heads=32, kv_heads=8, dim=128, context=160, page=16, ragged=False, dtype="bf16", codes="int8"),
        # the headline batch: 64 sequences at 2k
        dict(name="decode_batch", kind="decode", batch=64, heads=32, kv_heads=8, dim=128, context=2048, page=16, ragged=False, dtype="bf16", codes="int8"),
        # long contexts in the 70B head layout
        dict(name="decode_long", kind="decode", batch=8, heads=64, kv_heads=8, dim=128, context=32768, page=16, ragged=True, dtype="bf16", codes="e4m3"),
        # a portion of one long prompt: 512 tokens behind 8k
        dict(name="prompt_portion", kind="prompt", batch=1, new=512, heads=32, kv_heads=8, dim=128, context=8192, page=16, ragged=False, dtype="bf16", codes="int8"),
        # the prompts of 8 sequences of the headline length, from their first token on
        dict(name="prompt_batch", kind="prompt", batch=8, new=2048, heads=32, kv_heads=8, dim=128, context=0, page=16, ragged=False, dtype="bf16", codes="int8"),
        # a few tokens of many sequences behind odd contexts, heads with keys of their own, larger pages
        dict(name="prompt_odd", kind="prompt", batch=16, new=9, heads=16, kv_heads=16, dim=64, context=3001, page=32, ragged=True, dtype="fp16", codes="e4m3"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "write", "read", "decode", "decode", "decode", "prompt", "prompt", "prompt"))
    kv, rep = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 5, 8))
    small = rng.random() < 0.1      # the small model of the parity path, in 32 bits
    case = dict(kind=kind, kv_heads=2 if small else kv, dim=64 if small else rng.choice((64, 128, 128)), page=rng.choice((16, 16, 16, 32, 64)),
                dtype="fp32" if small else rng.choice(("bf16", "bf16", "fp16")), codes=rng.choice(("int8", "int8", "e4m3")))
    batch = _spread(rng, 1, 8 if small else 64)
    if kind == "read":
        return dict(case, batch=batch, context=_spread(rng, 20, 300 if small else 262144 // (case["kv_heads"] * batch)))
    case.update(batch=batch, heads=8 if small else kv * rep, ragged=rng.random() < 0.7)
    heads = case["heads"]
    if kind == "write":
        one = rng.random() < 0.4
        return dict(case, new=1 if one else _spread(rng, 2, 64 if small else max(2, 524288 // (heads * batch))), context=0 if rng.random() < 0.3 else _spread(rng, 1, 2048))
    if kind == "decode":
        return dict(case, context=_spread(rng, 30, 300 if small else min(32768, 2097152 // (case["kv_heads"] * batch))))
    new = _spread(rng, 2, 32 if small else max(2, min(2048, 524288 // (heads * batch))))
    return dict(case, new=new, context=0 if rng.random() < 0.3 else _spread(rng, 16, 200 if small else max(16, min(16384, 2097152 // (case["kv_heads"] * batch),
                                                                                                   1073741824 // (heads * batch * new)))))


# ---- inputs: made from the seed ---------------------------------------------------------------------------------------------------

def _pages(case, lens, most, g):
    """Block tables over pages in random order, and the number of pages: enough for sequences of `most` tokens."""
    per = max(1, -(-most // case["page"]))
    need = [-(-n // case["page"]) for n in lens]
    pages = per * len(lens) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables, at = torch.zeros((len(lens), per), dtype=torch.int32, device=DEV), 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n]
        at += n
    return tables, pages


def _cache(case, pages, g):
    """Pools as such a cache holds them: normal keys and values, each page's largest at the largest code or a little below, scales to it."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    pools = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=DEV) * (MOST[case["codes"]] / 4.0)
        pools.append(x.clamp_(-MOST[case["codes"]], MOST[case["codes"]]).round_().to(CODES[case["codes"]]))
    scales = [4.0 / MOST[case["codes"]] * torch.exp(0.3 * torch.randn((pages, case["kv_heads"]), generator=g, device=DEV)) for _ in range(2)]
    return dict(k_pool=pools[0], v_pool=pools[1], k_scale=scales[0], v_scale=scales[1])


def _lengths(case):
    """New tokens and tokens in all of each sequence; the same ones whatever the seed."""
    rng = random.Random(str([case[k] for k in sorted(case) if k != "name"]))
    part = (lambda n: int(n * rng.uniform(0.5, 1.0))) if case.get("ragged") else int  # noqa: E731
    new = [max(1, part(case.get("new", 1))) for _ in range(case["batch"])]
    if case["kind"] in ("read", "decode"):      # (the context counts the token that asks)
        return new, [max(1, part(case["context"])) for _ in range(case["batch"])]
    return new, [part(case["context"]) + n for n in new]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(dtype)  # noqa: E731
    kind, batch, dim, page = case["kind"], case["batch"], case["dim"], case["page"]
    if kind == "read":
        tables, pages = _pages(case, [case["context"]] * batch, case["context"], g)
        return dict(kind=kind, **_cache(case, pages, g), tables=tables, tokens=case["context"], dtype=dtype)
    new, lens = _lengths(case)
    if kind == "decode":
        tables, pages = _pages(case, lens, case["context"], g)
        return dict(kind=kind, q=normal(batch, case["heads"], dim), **_cache(case, pages, g), tables=tables, lens=ints(lens), longest=max(lens))
    tables, pages = _pages(case, lens, case["context"] + case["new"], g)
    starts = [sum(new[:b]) for b in range(batch + 1)]
    s = dict(kind=kind, q=normal(starts[-1], case["heads"], dim), **_cache(case, pages, g), tables=tables, lens=ints(lens),
             starts=None if kind == "write" and case["new"] == 1 else ints(starts), most=max(new), longest=max(lens), dtype=dtype)
    if kind == "write":
        s["k"], s["v"] = normal(starts[-1], case["kv_heads"], dim), normal(starts[-1], case["kv_heads"], dim)
        # where a channel stands out, as keys' do
        s["k"][..., 3::32] *= 4
        pos = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in zip(lens, new)]).double()
        angle = pos[:, None] * 500000.0 ** (-torch.arange(0, dim, 2, device=DEV).double() / dim)
        s["cos"], s["sin"] = (torch.cat((t, t), 1).to(dtype) for t in (angle.cos(), angle.sin()))
        first = [(n - m) // page for n, m in zip(lens, new)]
        wide = max((n - 1) // page + 1 - f for n, f in zip(lens, first))
        at = torch.stack([torch.arange(f, f + wide, device=DEV).clamp(max=(n - 1) // page) for f, n in zip(first, lens)])
        s["written"] = tables.gather(1, at).contiguous()
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------------

def _values(s, tables, tokens):
    """Keys and values [batch, kv heads, tokens, dim] in 32 bits: code times its page's scale."""
    page, dim = s["k_pool"].shape[2:]
    at = tables[:, :-(-tokens // page)].long()
    return tuple((pool.view(torch.uint8)[at].view(pool.dtype).float() * scale[at][..., None, None]).transpose(1, 2).reshape(
        tables.shape[0], pool.shape[1], -1, dim)[:, :, :tokens] for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])))


def _rows(s):
    """Sequence and position of each row."""
    lens = s["lens"].long()
    starts = torch.arange(lens.shape[0] + 1, device=DEV) if s["starts"] is None else s["starts"].long()
    row = torch.arange(s["q"].shape[0], device=DEV)
    b = torch.searchsorted(starts[1:], row, right=True)
    return b, lens[b] - starts[b + 1] + row, starts


def _to_codes(y, dtype):
    return y.round().clamp(-127, 127).to(dtype) if dtype == torch.int8 else y.to(dtype)


def _plain_write(s):
    """Rotation in 32 bits; a page's scale the largest magnitude of its new tokens over the largest code, or the one it had where it holds
    earlier tokens and that was larger - then what they hold is put into the new scale's codes."""
    cos, sin, dim, page = s["cos"].float()[:, None], s["sin"].float()[:, None], s["q"].shape[2], s["k_pool"].shape[2]
    turned = lambda x: x * cos + torch.cat((-x[..., dim // 2:], x[..., :dim // 2]), -1) * sin  # noqa: E731
    b, pos, starts = _rows(s)
    lens = s["lens"].long()
    held = lens - (starts[1:] - starts[:-1])      # tokens before
    first, wide = held // page, s["written"].shape[1]
    slots = s["written"].long()
    live = (first[:, None] + torch.arange(wide, device=DEV) <= (lens[:, None] - 1) // page)
    unit = b * wide + pos // page - first[b]
    earlier = torch.zeros(live.shape, dtype=torch.bool, device=DEV)
    earlier[:, 0] = held % page > 0
    for pool, scale, x in ((s["k_pool"], s["k_scale"], turned(s["k"].float())), (s["v_pool"], s["v_scale"], s["v"].float())):
        most = torch.zeros((slots.numel(), x.shape[1]), device=DEV).scatter_reduce_(0, unit[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        had = torch.where(earlier[..., None], scale[slots], 0.0).view(slots.numel(), -1)
        now = torch.maximum(torch.maximum(had, most * (1.0 / MOST["int8" if pool.dtype == torch.int8 else "e4m3"])), torch.tensor(LEAST, device=DEV))
        inverse = 1.0 / now
        raw = pool.view(torch.uint8)
        # (a page that several rows of `slots` name: all but the first are not live, and write nothing)
        mine = slots[live]
        pages = raw[mine].view(pool.dtype)
        again = _to_codes(pages.float() * (had * inverse).view(*live.shape, -1)[live][..., None, None], pool.dtype)
        before = (torch.arange(page, device=DEV)[None] < (held % page)[:, None])[:, None, :] & earlier[..., None]
        raw[mine] = torch.where(before[live][:, None, :, None], again.view(torch.uint8), pages.view(torch.uint8))
        raw[slots.view(-1)[unit], :, pos % page] = _to_codes(x * inverse[unit][..., None], pool.dtype).view(torch.uint8)
        scale[mine] = now.view(*live.shape, -1)[live]
    k, v = _values(s, s["written"], wide * page)
    return dict(q=turned(s["q"].float()).to(s["dtype"]), k=k.to(s["dtype"]), v=v.to(s["dtype"]), k_scale=s["k_scale"], v_scale=s["v_scale"])


def _plain_attention(s):
    """softmax(q k / sqrt(dim)) v over the keys up to each token's own position."""
    q, lens = s["q"].float(), s["lens"].long()
    heads, dim = q.shape[1:]
    k, v = _values(s, s["tables"], s["longest"])
    batch, kv, keys = k.shape[:3]
    if s["kind"] == "decode":
        b, n, pos, most = torch.arange(batch, device=DEV), torch.zeros(batch, dtype=torch.long, device=DEV), lens - 1, 1
    else:
        b, pos, starts = _rows(s)
        n, most = torch.arange(q.shape[0], device=DEV) - starts[b], s["most"]
    padded = torch.zeros((batch, most, heads, dim), device=DEV)
    padded[b, n] = q
    seen = torch.zeros((batch, most), dtype=torch.long, device=DEV)
    seen[b, n] = pos + 1
    scores = torch.einsum("bngrd,bgkd->bgrnk", padded.view(batch, most, kv, heads // kv, dim) * dim ** -0.5, k)
    scores.masked_fill_((torch.arange(keys, device=DEV) >= seen[:, :, None])[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = w.sum(-1)
    out = torch.einsum("bgrnk,bgkd->bngrd", w, v) / torch.where(total == 0, 1.0, total).permute(0, 3, 1, 2)[..., None]
    return out.reshape(batch, most, heads, dim)[b, n].to(s["q"].dtype)


def run(state):
    s = state
    if own:
        import dgi_b200  # noqa: F401
        from dgi_b200 import ops

        cache = (s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
        if s["kind"] == "write":
            q = ops.rope_kv_append_q8(s["q"], s["k"], s["v"], s["cos"], s["sin"], *cache, s["tables"], s["lens"], row_starts=s["starts"], max_new=s["most"])
            k, v = ops.kv_gather_dense_q8(*cache, s["written"], s["written"].shape[1] * s["k_pool"].shape[2], s["dtype"])
            return dict(q=q, k=k, v=v, k_scale=s["k_scale"], v_scale=s["v_scale"])
        if s["kind"] == "read":
            return ops.kv_gather_dense_q8(*cache, s["tables"], s["tokens"], s["dtype"])
        if s["kind"] == "decode":
            return ops.paged_decode_attention_q8(s["q"], *cache, s["tables"], s["lens"], s["longest"])
        return ops.paged_prompt_attention_q8(s["q"], *cache, s["tables"], s["lens"], s["starts"], s["most"], s["longest"])
    if s["kind"] == "write":
        return _plain_write(s)
    if s["kind"] == "read":
        return tuple(x.to(s["dtype"]) for x in _values(s, s["tables"], s["tokens"]))
    return _plain_attention(s)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------

def _exact_write(case, s):
    page, dim, top = case["page"], case["dim"], MOST[case["codes"]]
    cos, sin = s["cos"].double()[:, None, :dim // 2], s["sin"].double()[:, None, :dim // 2]

    def turned(x):
        a, b = x.double().chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    def coded(y):
        return torch.round(y) if case["codes"] == "int8" else y.float().to(torch.float8_e4m3fn).double()

    lens, tables = s["lens"].tolist(), s["tables"].tolist()
    starts = list(range(len(lens) + 1)) if s["starts"] is None else s["starts"].tolist()
    answer = dict(q=turned(s["q"]))
    for name, x in (("k", turned(s["k"])), ("v", s["v"].double())):
        codes, scale, back = s[name + "_pool"], s[name + "_scale"].double(), []
        for b, length in enumerate(lens):
            held, mine, rows = length - (starts[b + 1] - starts[b]), [], x[starts[b]:starts[b + 1]].transpose(0, 1)
            p0, p1 = held // page, (length - 1) // page + 1
            at = torch.tensor(tables[b][p0:p1], device=DEV)
            off, n = held - p0 * page, rows.shape[1]
            # every touched page at once: the new tokens' largest, the scale that the first one had
            room = torch.zeros((rows.shape[0], (p1 - p0) * page, dim), dtype=torch.float64, device=DEV)
            room[:, off:off + n] = rows
            room = room.view(rows.shape[0], p1 - p0, page, dim).transpose(0, 1)
            new = room.abs().amax((-1, -2)) / top
            had = scale[at[0]].clone()
            if off:
                new[0] = torch.maximum(new[0], had)
            new = new.clamp_min(LEAST)
            scale[at] = new
            value = codes.view(torch.uint8)[at].view(codes.dtype).double()
            if off:
                value[0, :, :off] = coded(value[0, :, :off] * (had / new[0])[:, None, None])
            ours = torch.zeros((p1 - p0) * page, dtype=torch.bool, device=DEV)
            ours[off:off + n] = True
            value = torch.where(ours.view(p1 - p0, 1, page, 1), coded(room / new[..., None, None]), value) * new[..., None, None]
            wide = s["written"].shape[1]
            back.append(value[torch.arange(wide, device=DEV).clamp(max=p1 - p0 - 1)].transpose(0, 1).reshape(rows.shape[0], wide * page, dim))
        answer[name], answer[name + "_scale"] = torch.stack(back), scale
    return answer


def exact(case, seed):
    """The same in 64 bits, a sequence (and a kv head) at a time."""
    s = prepare(case, seed)
    if case["kind"] == "write":
        return _exact_write(case, s)
    page, dim, kv = case["page"], case["dim"], case["kv_heads"]

    def dense(name, b, h, n):
        at = s["tables"][b, :-(-n // page)].long()
        return (s[name + "_pool"][:, h].view(torch.uint8)[at].view(CODES[case["codes"]]).double() * s[name + "_scale"][at, h].double()[:, None, None]).reshape(-1, dim)[:n]

    if case["kind"] == "read":
        return tuple(torch.stack([torch.stack([dense(x, b, h, case["context"]) for h in range(kv)]) for b in range(case["batch"])]) for x in "kv")
    q, group = s["q"].double(), case["heads"] // kv
    out = torch.zeros_like(q)
    lens = s["lens"].tolist()
    starts = list(range(len(lens) + 1)) if case["kind"] == "decode" else s["starts"].tolist()
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        hidden = torch.full((r1 - r0, length), -math.inf, dtype=torch.float64, device=DEV).triu(length - (r1 - r0) + 1)
        for h in range(kv):
            k, v = dense("k", b, h, length), dense("v", b, h, length)
            scores = torch.einsum("ngd,kd->gnk", q[r0:r1, h * group:(h + 1) * group], k) / math.sqrt(dim) + hidden
            out[r0:r1, h * group:(h + 1) * group] = torch.einsum("gnk,kd->ngd", torch.softmax(scores, -1), v)
    return out


def work(case):
    """Bytes that have to be read and written once, operations of the products."""
    size, page, kv, row = SIZE[case["dtype"]], case["page"], case["kv_heads"], 2 * case["kv_heads"] * case["dim"]      # row: a token's keys and values
    new, lens = _lengths(case)
    held = sum(lens) * row + 8 * kv * sum(-(-n // page) for n in lens)      # codes and scales of all tokens
    if case["kind"] == "read":
        return {"bytes": held + sum(lens) * row * size, "flops": sum(lens) * row}
    q = sum(new) * case["heads"] * case["dim"]
    if case["kind"] == "write":
        pages = sum((n - 1) // page + 1 - (n - m) // page for n, m in zip(lens, new))
        # what comes in and the queries going out; codes; the written pages read back
        return {"bytes": 2 * q * size + sum(new) * (row * (size + 1) + 2 * case["dim"] * size) + pages * (page * row * (1 + size) + 16 * kv),
                "flops": 3 * q + 5 * sum(new) * row}
    pairs = sum(lens) if case["kind"] == "decode" else sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
    return {"bytes": held + 2 * q * size, "flops": 4 * case["heads"] * case["dim"] * pairs}
