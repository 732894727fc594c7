"""Attention of drafted tokens over paged KV against the formula in 64 bits.

Bound per element, with e = half a step of the type relative to a value, A = sum_j w_j |v_j| / sum_j w_j:  the output's rounding e |o|; the weights' rounding to
16 bits e A; sums in 32 bits 2^-24 (keys + 8) A; scores off by d = (D + 8) 2^-24 scale sum |q k| change a weight by 2 d of itself at most (its own score and the
maximum's share of the sum), and exponentials by 2^-21 of themselves: (2 d + 2^-21) 2 A."""
import random

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64


def build(B, nodes, Hq, Hkv, D, bs, context, dtype, seed=0, ragged=True, tree=True, stale=float("nan")):
    """Context lengths up to `context`, pages in random order, slots that nobody owns filled with `stale`."""
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    drafts = [rng.randint(0 if b == 1 else 1, nodes) if ragged else nodes for b in range(B)]
    past = [0 if ragged and b == 2 else rng.randint(0, context) if ragged else context for b in range(B)]
    lens = [p + n for p, n in zip(past, drafts)]
    cols = max(1, -(-max(lens) // bs))
    need = [-(-n // bs) for n in lens]
    order = list(range(sum(need) + 2))
    rng.shuffle(order)
    tables = torch.full((B, cols), -1, dtype=torch.int32)
    k = torch.full((len(order), Hkv, bs, D), stale, device=DEV)
    v = torch.full_like(k, stale)
    at = 0
    for b in range(B):
        tables[b, :need[b]] = torch.tensor(order[at:at + need[b]], dtype=torch.int32)
        for i in range(need[b]):
            n = min(bs, lens[b] - i * bs)
            k[order[at + i], :, :n] = torch.randn((Hkv, n, D), generator=g, device=DEV)
            v[order[at + i], :, :n] = torch.randn((Hkv, n, D), generator=g, device=DEV)
        at += need[b]
    q = torch.randn((B, nodes, Hq, D), generator=g, device=DEV) * 1.5
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    if tree:
        visible, _ = ops.draft_tree(i32([[-1] + [rng.randrange(max(0, t - 6), t) for t in range(1, nodes)] for _ in range(B)]))
    else:       # any masks, empty ones among them
        visible = torch.tensor([[rng.choice((0, -1, rng.getrandbits(63), -rng.getrandbits(62))) for _ in range(nodes)] for _ in range(B)],
                               dtype=torch.int64, device=DEV)
    return dict(q=q.to(dtype), k_pool=k.to(dtype), v_pool=v.to(dtype), block_tables=tables.to(DEV), context_lens=i32(lens), visible=visible,
                draft_lens=i32(drafts))


def reference(c, scale=None):
    """(values, bound) in 64 bits; what no row sees is left out of the sums."""
    q, bs, D = c["q"], c["k_pool"].shape[2], c["q"].shape[3]
    B, nodes, Hq, _ = q.shape
    Hkv, blocks = c["k_pool"].shape[1], c["k_pool"].shape[0]
    scale = D ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=F64, device=DEV), torch.zeros(q.shape, dtype=F64, device=DEV)
    e = torch.finfo(q.dtype).eps / 2
    lens = c["context_lens"].tolist()
    drafts = c["draft_lens"].tolist() if c["draft_lens"] is not None else [nodes] * B
    for b in range(B):
        length = min(lens[b], c["block_tables"].shape[1] * bs)
        n = min(drafts[b], length)
        if n == 0:
            continue
        pos = torch.arange(length, device=DEV)
        page = c["block_tables"][b].long()[pos // bs]
        bad = (page < 0) | (page >= blocks)
        kk, vv = (torch.where(bad[:, None, None], 0.0, p[page.clamp(0, blocks - 1), :, pos % bs].to(F64)) for p in (c["k_pool"], c["v_pool"]))
        for t in range(n):
            m = c["visible"][b, t].item()
            see = torch.tensor([j < length - n or bool(m >> (j - length + n) & 1) for j in range(length)], device=DEV)
            if not see.any():
                continue
            k, v = (x[see].repeat_interleave(Hq // Hkv, 1) for x in (kk, vv))
            qt = q[b, t].to(F64)
            s = torch.einsum("hd,khd->hk", qt, k) * scale
            w = torch.softmax(s, 1)
            out[b, t] = torch.einsum("hk,khd->hd", w, v)
            A = torch.einsum("hk,khd->hd", w, v.abs())
            d = (D + 8) * 2.0 ** -24 * scale * torch.einsum("hd,khd->hk", qt.abs(), k.abs()).amax(1, keepdim=True)
            bound[b, t] = e * out[b, t].abs() + A * (e + 2.0 ** -24 * (length + 8) + 2 * (2 * d + 2.0 ** -21)) + torch.finfo(q.dtype).tiny
    return out, bound


def check(c, flags=0, scale=None, **kw):
    got = ops.paged_tree_attention(c["q"], c["k_pool"], c["v_pool"], c["block_tables"], c["context_lens"], c["visible"],
                                   draft_lens=c["draft_lens"], scale=scale, flags=flags, **kw)
    want, bound = reference(c, scale)
    off = (got.to(F64) - want).abs()
    assert bool((off <= bound).all()), f"{(off / bound.clamp_min(1e-300)).max().item():.3f} of the bound"
    return got


SHAPES = [  # B, nodes, Hq, Hkv, D, page, context
    (1, 1, 1, 1, 64, 16, 0), (1, 1, 8, 8, 128, 16, 1), (3, 8, 32, 8, 128, 16, 160), (4, 13, 8, 2, 64, 16, 200), (3, 64, 16, 2, 128, 16, 700),
    (5, 5, 16, 16, 64, 32, 333), (3, 7, 10, 2, 128, 64, 500), (3, 33, 6, 2, 64, 8, 129), (4, 3, 20, 4, 128, 128, 777), (3, 9, 64, 1, 64, 16, 250),
    (3, 4, 12, 4, 96, 16, 100), (3, 6, 4, 2, 20, 5, 90), (3, 6, 4, 2, 64, 24, 300), (3, 5, 3, 1, 256, 16, 100), (3, 2, 2, 1, 7, 1, 40),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,nodes,Hq,Hkv,D,page,context", SHAPES)
def test_against_the_formula(B, nodes, Hq, Hkv, D, page, context, dtype):
    c = build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=nodes + D)
    check(c)
    check(c, flags=ops.ATTN_FORCE_GENERIC)
    check(build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=nodes, tree=False))
    even = build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=1, ragged=False)
    even["draft_lens"] = None
    check(even, scale=0.3)


SHARED = [  # types and sizes without tensor cores, tables of many tokens or many rows
    (1, 1, 4, 2, 64, 16, 2500), (2, 3, 8, 2, 96, 24, 1300), (1, 4, 16, 4, 128, 16, 5000), (3, 13, 8, 2, 64, 5, 700), (2, 64, 16, 2, 256, 16, 600),
    (40, 8, 32, 8, 64, 16, 70), (5, 2, 6, 3, 20, 7, 900), (64, 1, 2, 2, 200, 16, 640), (2, 16, 4, 4, 256, 16, 1000), (7, 9, 9, 3, 128, 16, 530),
    (300, 2, 2, 2, 40, 16, 3), (1, 64, 64, 1, 64, 16, 1),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,nodes,Hq,Hkv,D,page,context", SHARED)
def test_rows_that_share_their_keys_without_tensor_cores(B, nodes, Hq, Hkv, D, page, context, dtype):
    check(build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=nodes + D), flags=ops.ATTN_FORCE_GENERIC)
    check(build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=nodes, tree=False), flags=ops.ATTN_FORCE_GENERIC)
    even = build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=1, ragged=False)
    even["draft_lens"] = None
    check(even, scale=0.3, flags=ops.ATTN_FORCE_GENERIC)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_no_numbers_among_rows_that_share_their_keys(D, dtype):
    """A node without numbers, and what stands behind the last node: rows that do not see them stay as they are."""
    B, nodes, page = 2, 20, 16
    c = build(B, nodes, 8, 2, D, page, 900, dtype, seed=5, ragged=False)
    clean = ops.paged_tree_attention(**c, flags=ops.ATTN_FORCE_GENERIC)
    lens, seen = c["context_lens"].tolist(), c["visible"].tolist()
    for b in range(B):
        for place in [lens[b] - nodes + 7] + list(range(lens[b], -(-lens[b] // page) * page)):
            at = int(c["block_tables"][b, place // page])
            c["k_pool"][at, :, place % page] = float("nan")
            c["v_pool"][at, :, place % page] = float("inf")
    got = ops.paged_tree_attention(**c, flags=ops.ATTN_FORCE_GENERIC)
    for b in range(B):
        for t in range(nodes):
            if seen[b][t] >> 7 & 1:
                assert got[b, t].isnan().all()
            else:
                assert torch.equal(got[b, t], clean[b, t])


@pytest.mark.parametrize("context", [63, 64, 65, 127, 128, 129, 4000, 20001])
@pytest.mark.parametrize("nodes", [1, 16, 63, 64])
def test_lengths_around_a_tile(nodes, context):
    check(build(2, nodes, 4, 1, 128, 16, context, torch.bfloat16, seed=context, ragged=False))


@pytest.mark.parametrize("flags", [0, ops.ATTN_FORCE_GENERIC])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(flags):
    c = build(2, 40, 8, 2, 128, 16, 100, torch.bfloat16, seed=3, ragged=False)
    inf, nan = float("inf"), float("nan")
    lens, B, nodes = c["context_lens"].tolist(), 2, 40
    where = {}
    for b in range(B):
        for t, d, what in ((3, 5, inf), (7, 100, nan), (11, 5, -inf), (39, 127, inf)):
            j = lens[b] - nodes + t
            c["v_pool"][int(c["block_tables"][b, j // 16]), 1, j % 16, d] = what
            where[(b, t, d)] = what
    clean = dict(c, v_pool=torch.where(torch.isfinite(c["v_pool"]), c["v_pool"], 0.0))
    got = ops.paged_tree_attention(c["q"], c["k_pool"], c["v_pool"], c["block_tables"], c["context_lens"], c["visible"], flags=flags)
    want, bound = reference(clean)
    hit = torch.zeros(got.shape, dtype=F64, device=DEV)
    for (b, t, d), what in where.items():
        for row in range(nodes):
            if c["visible"][b, row].item() >> t & 1:
                hit[b, row, 4:, d] += what
    plain = hit == 0
    assert bool(((got.to(F64) - want).abs() <= bound)[plain].all())
    assert torch.equal(torch.nan_to_num(got.to(F64)[~plain], nan=7.0), torch.nan_to_num(hit[~plain], nan=7.0))


@pytest.mark.parametrize("flags", [0, ops.ATTN_FORCE_GENERIC])
def test_keys_that_are_no_numbers_stay_behind_their_mask(flags):
    c = build(1, 12, 4, 2, 64, 16, 50, torch.float16, seed=5, ragged=False)
    c["visible"][0] &= ~(1 << 4)          # nobody sees node 4
    j = 50 + 4
    page = int(c["block_tables"][0, j // 16])
    c["k_pool"][page, :, j % 16] = float("nan")
    c["v_pool"][page, :, j % 16] = float("inf")
    check(c, flags=flags)


@pytest.mark.parametrize("flags", [0, ops.ATTN_FORCE_GENERIC])
def test_pages_outside_the_pool_read_as_zeros(flags):
    c = build(2, 6, 8, 2, 128, 16, 200, torch.bfloat16, seed=6, ragged=False)
    c["block_tables"][0, 3] = -1
    c["block_tables"][1, 5] = 2 ** 31 - 1
    c["block_tables"][1, -1] = c["k_pool"].shape[0]
    check(c, flags=flags)
    short = dict(c, block_tables=c["block_tables"][:, :4].contiguous())       # lengths beyond the table: its pages only
    check(short, flags=flags)


def test_large_scores_and_a_maximum_that_grows_along_the_keys():
    c = build(2, 16, 8, 2, 128, 16, 1500, torch.bfloat16, seed=7, ragged=False, stale=0.0)
    for b in range(2):
        for i in range(c["block_tables"].shape[1]):
            c["k_pool"][int(c["block_tables"][b, i])] *= (0.2 + 0.04 * i)
    check(c)
    c["q"] = c["q"] * -1
    check(c)


@pytest.mark.parametrize("flags", [0, ops.ATTN_FORCE_GENERIC])
@pytest.mark.parametrize("nodes", [3, 40])
def test_a_scale_that_is_no_number(nodes, flags):
    q, k, v = (torch.randn(s, device="cuda").bfloat16() for s in ((2, nodes, 8, 128), (20, 2, 16, 128), (20, 2, 16, 128)))
    tables, lens = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10), torch.tensor([nodes + 70, nodes], dtype=torch.int32, device="cuda")
    visible, _ = ops.draft_tree(torch.arange(-1, nodes - 1, dtype=torch.int32, device="cuda").expand(2, -1))
    assert ops.paged_tree_attention(q, k, v, tables, lens, visible, scale=float("nan"), flags=flags).isnan().all()


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("nodes", [3, 12, 40])
def test_scales_below_and_at_zero(nodes, scale):
    check(build(2, nodes, 8, 2, 64, 16, 700, torch.bfloat16, seed=nodes, stale=0.0), scale=scale)


def test_many_sequences_and_groups_of_odd_size():
    """More sequences than a look-up of lengths holds; heads whose rows straddle warps and blocks."""
    check(build(150, 3, 6, 2, 64, 16, 90, torch.bfloat16, seed=2))
    wide = build(140, 2, 5, 1, 128, 16, 700, torch.float16, seed=3)
    check(wide)
    check(build(2, 61, 21, 3, 128, 16, 900, torch.bfloat16, seed=5))


def test_a_context_that_is_infinite_somewhere_is_no_number_there():
    c = build(2, 6, 8, 2, 128, 16, 900, torch.bfloat16, seed=11, ragged=False, stale=0.0)
    c["v_pool"][int(c["block_tables"][1, 3]), 0, 5, 9] = float("inf")
    got = ops.paged_tree_attention(c["q"], c["k_pool"], c["v_pool"], c["block_tables"], c["context_lens"], c["visible"])
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[1, :, :4, 9] = True
    assert torch.equal(bad, want)


def test_strided_queries_tables_and_masks():
    c = build(3, 10, 8, 2, 64, 16, 150, torch.bfloat16, seed=8)
    qkv = torch.randn((3, 10, 12 * 64), device=DEV).to(torch.bfloat16)
    q = qkv[..., :8 * 64].unflatten(-1, (8, 64))
    q.copy_(c["q"])
    tables = torch.full((3, c["block_tables"].shape[1] + 5), 10 ** 8, dtype=torch.int32, device=DEV)
    tables[:, :c["block_tables"].shape[1]] = c["block_tables"]
    masks = torch.full((3, 64), -1, dtype=torch.int64, device=DEV)
    masks[:, :10] = c["visible"]
    a = check(c)
    b = check(dict(c, q=q, block_tables=tables[:, :c["block_tables"].shape[1]], visible=masks[:, :10]))
    assert torch.equal(a, b)
    odd = torch.randn((3, 10, 8 * 64 + 3), device=DEV).to(torch.bfloat16)[..., 1:8 * 64 + 1].unflatten(-1, (8, 64))      # off the 16-byte grid
    odd.copy_(c["q"])
    check(dict(c, q=odd))


def test_own_workspaces_streams_and_graphs():
    """Two captured calls with workspaces of their own, replayed side by side; a workspace's contents do not matter."""
    cases = [build(4, 8, 32, 8, 128, 16, 2000, torch.bfloat16, seed=s) for s in (1, 2)]
    size = lambda c: ops.tree_attention_workspace(8, 32, 8, 128, 16, torch.bfloat16)  # noqa: E731
    want = [check(c) for c in cases]
    spaces = [torch.full((max(16, size(c)),), 255, dtype=torch.uint8, device=DEV) for c in cases]
    graphs, outs = [], []
    for c, ws in zip(cases, spaces):
        out = torch.full_like(c["q"], 3.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_tree_attention(c["q"], c["k_pool"], c["v_pool"], c["block_tables"], c["context_lens"], c["visible"], draft_lens=c["draft_lens"],
                                     out=out, workspace=ws)
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for st, graph in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_the_same_bits_every_time():
    c = build(3, 24, 32, 8, 128, 16, 5000, torch.bfloat16, seed=4)
    first = check(c)
    for _ in range(5):
        assert torch.equal(first, check(c))


def test_one_node_is_a_decode_step():
    """A tree of one node against the decode attention of the same library."""
    c = build(5, 1, 32, 8, 128, 16, 900, torch.bfloat16, seed=9, ragged=False)
    tree = check(c)
    decode = ops.paged_decode_attention(c["q"][:, 0], c["k_pool"], c["v_pool"], c["block_tables"], c["context_lens"], 901)
    want, bound = reference(c)
    assert bool(((decode.to(F64) - tree[:, 0].to(F64)).abs() <= 2 * bound[:, 0] + 2.0 ** -8 * want[:, 0].abs()).all())


def test_a_workspace_that_is_too_small_is_refused():
    need = ops.tree_attention_workspace(8, 32, 8, 128, 16, torch.bfloat16)
    if need == 0:
        pytest.skip("no workspace is needed")
    c = build(4, 8, 32, 8, 128, 16, 200, torch.bfloat16)
    with pytest.raises(_lib.B200LibraryError, match="workspace"):
        check(c, workspace=torch.empty(need - 1, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,nodes,Hq,Hkv,D,page,context", [(1, 8, 32, 8, 128, 16, 160), (40, 3, 8, 8, 64, 16, 300), (3, 64, 16, 2, 128, 16, 400),
                                                           (5, 20, 12, 4, 64, 32, 100), (3, 33, 6, 2, 128, 64, 448)])
def test_short_tables_and_the_same_behind_long_ones(B, nodes, Hq, Hkv, D, page, context, dtype):
    """Tables of up to 512 keys are walked in one piece: the same formula, rows behind the last node 0, sequences without one."""
    for tree in (True, False):
        c = build(B, nodes, Hq, Hkv, D, page, context, dtype, seed=B + nodes, tree=tree)
        out = torch.full_like(c["q"], 7.0)
        check(c, out=out)
        for b, n in enumerate(c["draft_lens"].tolist()):
            assert bool((out[b, n:] == 0).all())
        wide = torch.full((B, 600 // page + 9), -3, dtype=torch.int32, device=DEV)
        wide[:, :c["block_tables"].shape[1]] = c["block_tables"]
        check(dict(c, block_tables=wide))
    c["draft_lens"].zero_()
    assert bool((check(c) == 0).all()) and bool((check(dict(c, block_tables=wide)) == 0).all())
