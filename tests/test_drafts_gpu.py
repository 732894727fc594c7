"""Draft trees: masks, accepted paths and moved rows against a walk down each tree in Python."""
import random

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def trees(batch, nodes, seed, chain=False):
    rng = random.Random(seed)
    return [[-1] + [t - 1 if chain else rng.randrange(max(0, t - 9), t) for t in range(1, nodes)] for _ in range(batch)]


def signed(m):
    return m - (1 << 64) if m >> 63 else m


@pytest.mark.parametrize("nodes", [1, 2, 3, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("batch,chain", [(1, True), (1, False), (5, False), (70, False)])
def test_masks_and_depths(batch, nodes, chain):
    rng = random.Random(nodes)
    par, lens = trees(batch, nodes, nodes, chain), [rng.randint(0, nodes) for _ in range(batch)]
    if nodes > 4:
        par[0][3] = 3           # parents that do not come before their children
        par[-1][4] = nodes + 5
        par[-1][2] = -7
    wide = torch.full((batch, nodes + 3), 99, dtype=torch.int32, device=DEV)
    wide[:, :nodes] = torch.tensor(par, dtype=torch.int32, device=DEV)
    for cut in (None, lens):
        visible, depth = ops.draft_tree(wide[:, :nodes], None if cut is None else torch.tensor(cut, dtype=torch.int32, device=DEV))
        for b in range(batch):
            seen, deep = [], []
            for t in range(nodes):
                p = par[b][t]
                up = t > 0 and 0 <= p < t
                seen.append((1 << t) | (seen[p] if up else 0))
                deep.append(deep[p] + 1 if up else 0)
            n = nodes if cut is None else cut[b]
            assert visible[b].tolist() == [signed(m) if t < n else 0 for t, m in enumerate(seen)]
            assert depth[b].tolist() == [d if t < n else 0 for t, d in enumerate(deep)]


def case(batch, nodes, seed, page, layers, kv, dim, dtype, accepted, chain=False, ragged=False):
    rng = random.Random(seed)
    par = trees(batch, nodes, seed, chain)
    lens = [rng.randint(1, nodes) if ragged else nodes for _ in range(batch)]
    tokens = [[rng.randrange(50) for _ in range(nodes)] for _ in range(batch)]      # siblings with equal tokens among them
    chosen = [[rng.randrange(50) for _ in range(nodes)] for _ in range(batch)]
    for b in range(batch):
        at = 0
        for _ in range(accepted):
            kids = [t for t in range(at + 1, lens[b]) if par[b][t] == at]
            if not kids:
                break
            at, before = rng.choice(kids), at
            chosen[b][before] = tokens[b][at]
    context = [rng.randint(0, 3 * page) for _ in range(batch)]
    cols = -(-(max(context) + nodes) // page)
    order = list(range(batch * cols + 2))
    rng.shuffle(order)
    tables = [order[b * cols:(b + 1) * cols] for b in range(batch)]
    g = torch.Generator(device=DEV).manual_seed(seed)
    pools = [torch.randn((len(order), kv, page, dim), generator=g, device=DEV).to(dtype) for _ in range(2 * layers)]
    return par, lens, tokens, chosen, context, tables, pools


def walk(par, n, tokens, chosen):
    path = [0] if n > 0 else []
    while path:
        at = next((t for t in range(path[-1] + 1, n) if par[t] == path[-1] and tokens[t] == chosen[path[-1]]), None)
        if at is None:
            break
        path.append(at)
    return path


def run(c, **kw):
    par, lens, tokens, chosen, context, tables, pools = c
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    i64 = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    drafts = i32(lens)
    visible, _ = ops.draft_tree(i32(par), drafts)
    k, v = ops.pool_pointer_array(pools[0::2]), ops.pool_pointer_array(pools[1::2])
    return ops.accept_drafts(i64(tokens), i64(chosen), i32(par), visible, k, v, tuple(pools[0].shape), pools[0].dtype, i32(tables),
                             i32([n + x for n, x in zip(lens, context)]), draft_lens=drafts, **kw)


@pytest.mark.parametrize("batch,nodes,page,layers,kv,dim,dtype,accepted,ragged", [
    (1, 1, 16, 1, 1, 64, torch.float32, 0, False), (1, 8, 16, 4, 2, 64, torch.float32, 3, False), (3, 2, 16, 2, 2, 128, torch.bfloat16, 1, False),
    (7, 24, 16, 3, 8, 128, torch.bfloat16, 6, True), (64, 64, 32, 2, 4, 64, torch.float16, 12, True), (5, 33, 5, 2, 3, 20, torch.float16, 9, True),
    (4, 40, 7, 1, 1, 3, torch.bfloat16, 9, True), (2, 64, 16, 40, 1, 256, torch.float32, 30, False),
])
@pytest.mark.parametrize("chain", [False, True])
def test_accepted_path_and_moved_rows(batch, nodes, page, layers, kv, dim, dtype, accepted, ragged, chain):
    c = case(batch, nodes, nodes + batch, page, layers, kv, dim, dtype, accepted, chain, ragged)
    par, lens, tokens, chosen, context, tables, pools = c
    want = [p.clone() for p in pools]
    count, path, new_tokens, new_lens = run(c)
    for b in range(batch):
        taken = walk(par[b], lens[b], tokens[b], chosen[b])
        tail = [-1] * (nodes - len(taken))
        assert int(count[b]) == len(taken) and path[b].tolist() == taken + tail
        assert new_tokens[b].tolist() == [chosen[b][t] for t in taken] + tail and int(new_lens[b]) == context[b] + len(taken)
        for k, t in enumerate(taken):
            src, dst = context[b] + t, context[b] + k
            for p in want:
                p[tables[b][dst // page], :, dst % page] = p[tables[b][src // page], :, src % page].clone()
    for got, w in zip(pools, want):       # every other row as it was
        assert torch.equal(got.view(torch.uint8), w.view(torch.uint8))


def test_no_drafts_no_pools_and_pages_outside():
    c = case(3, 6, 1, 16, 2, 2, 64, torch.bfloat16, 4, chain=True)
    par, lens, tokens, chosen, context, tables, pools = c
    lens[1] = 0
    before = [p.clone() for p in pools]
    tables[0] = [-5] * len(tables[0])
    tables[2] = [10 ** 6] * len(tables[2])
    count, path, _, new_lens = run(c)
    assert count.tolist()[1] == 0 and path[1].tolist() == [-1] * 6 and int(new_lens[1]) == context[1]
    assert count.tolist()[0] == 5       # the path does not depend on the pages
    for got, w in zip(pools, before):
        assert torch.equal(got, w)
    i32, i64 = (lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)), (lambda v: torch.tensor(v, dtype=torch.int64, device=DEV))
    visible, _ = ops.draft_tree(i32(par))
    out = ops.accept_drafts(i64(tokens), i64(chosen), i32(par), visible, None, None, (1, 1, 16, 64), torch.bfloat16, i32(tables), i32([9, 0, 4]))
    # contexts shorter than the trees: as many nodes as there are tokens
    assert out[0].tolist() == [len(walk(par[b], n, tokens[b], chosen[b])) for b, n in enumerate((6, 0, 4))]
    assert out[3].tolist() == [3 + int(out[0][0]), 0, int(out[0][2])]


def test_values_that_are_the_keys_move_once():
    c = case(3, 16, 4, 16, 1, 1, 64, torch.bfloat16, 7)
    alone = [p.clone() for p in c[6]]
    run(c[:6] + ([alone[0], alone[1]],))
    both = c[6][0].clone()
    run(c[:6] + ([both, both],))
    assert torch.equal(both, alone[0])


def test_captured_and_replayed():
    c = case(4, 16, 3, 16, 2, 2, 64, torch.bfloat16, 5)
    par, lens, tokens, chosen, context, tables, pools = c
    start = [p.clone() for p in pools]
    i32, i64 = (lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)), (lambda v: torch.tensor(v, dtype=torch.int64, device=DEV))
    a = [i64(tokens), i64(chosen), i32(par)]
    k, v = ops.pool_pointer_array(pools[0::2]), ops.pool_pointer_array(pools[1::2])
    t, n = i32(tables), i32([16 + x for x in context])

    def call():
        visible, _ = ops.draft_tree(a[2])
        return ops.accept_drafts(*a, visible, k, v, tuple(pools[0].shape), torch.bfloat16, t, n)

    want = [x.clone() for x in call()]
    moved = [p.clone() for p in pools]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for p, s in zip(pools, start):
        p.copy_(s)
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(p, m) for p, m in zip(pools, moved))
