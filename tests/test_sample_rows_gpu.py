"""Drawn tokens against the definition in 64 bits (numpy, one row at a time): the same token, always.  Rows of one element to 2^20, off the 16-byte
grid, ties at every limit, masked and infinite logits, numbers at the ends of [0, 1), the cluster forms, a captured call."""
import numpy as np
import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SETTINGS = [  # temperature, top-k, top-p, min-p
    (1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (0.0, 50, 0.9, 0.0), (1.3, 0, 0.95, 0.0), (0.5, 3, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 1.0, 0.05),
    (2.0, 1000, 0.999, 0.001), (1.0, 20, 0.3, 0.5), (1.5, 0, 0.5, 0.02), (0.9, 200, 0.0, 0.0), (1.0, -1, -1.0, 2.0), (30.0, 0, 0.9, 0.0), (1e-3, 0, 0.9, 0.0),
]


def token(x, u, t, k, p, m):
    """The definition, for one row."""
    x, t, p, m, u = x.astype(np.float64), *(float(np.float32(v)) for v in (t, p, m, u))
    if np.isnan(x).any():
        return int(np.flatnonzero(np.isnan(x))[0])
    top = x.max()
    if not t > 0 or not np.isfinite(top):
        return int(np.argmax(x))
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == -np.inf, 0.0, np.exp((x - top) / t))
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        ws = w[order]
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        order = order[np.maximum(before < p * ws.sum(), np.arange(len(ws)) == 0)]
    if m > 0:
        order = order[(w[order] >= min(m, 1.0))]
    kept = np.zeros_like(w)
    kept[order] = w[order]
    total = np.cumsum(kept)
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -53)
    return int(np.flatnonzero(total > u * total[-1])[0])


def check(x, u, settings, **kw):
    cols = list(zip(*settings))
    f = [torch.tensor(c, dtype=ty, device=DEV) for c, ty in zip(cols, (torch.float32, torch.int32, torch.float32, torch.float32))]
    got = ops.sample_rows(x, u, temperature=f[0], top_k=f[1], top_p=f[2], min_p=f[3], **kw).tolist()
    rows, us = x.float().cpu().numpy(), u.cpu().numpy()
    want = [token(r, v, *s) for r, v, s in zip(rows, us, settings)]
    assert got == want


def logits(rows, cols, dtype, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((rows, cols), generator=g, device=DEV) * spread
    x[:, :: max(1, cols // 5)] += 5.0
    return x.to(dtype), torch.rand(rows, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 255, 256, 257, 1000, 4099, 32003, 128256])
def test_against_the_definition(cols, dtype):
    x, u = logits(len(SETTINGS), cols, dtype, cols)
    check(x, u, SETTINGS)
    for s in SETTINGS[:2] + SETTINGS[3:4]:        # a row alone: another number of CTAs
        check(x[3:4], u[3:4], [s])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [300001, 1 << 20])
def test_rows_of_several_ctas_and_beyond_shared_memory(cols, dtype):
    x, u = logits(3, cols, dtype, 5, spread=1.0)
    for part in ([SETTINGS[0], SETTINGS[1], SETTINGS[3]], [SETTINGS[7], SETTINGS[9], SETTINGS[6]]):
        check(x, u, part)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_tokens_kept_than_a_list_holds(dtype):
    """k beyond 2048, and ranges with more equal logits than are listed: the last key by its digits."""
    x, u = logits(6, 50001, dtype, 21)
    more = [(1.0, 2049, 1.0, 0.0), (1.0, 5000, 0.9, 0.0), (1.5, 49999, 0.99, 1e-4), (0.7, 2048, 1.0, 0.0), (1.0, 50000, 0.5, 0.0), (2.0, 30000, 1.0, 0.01)]
    check(x, u, more)
    check((x * 0.25).round() * 4, u, more)
    check((x * 0.25).round() * 4, u, [(1.0, 0, 0.9, 0.0), (1.0, 700, 1.0, 0.0), (1.0, 2000, 0.99, 0.0), (3.0, 0, 0.999, 0.0), (1.0, 0, 0.3, 0.1), (1.0, 9, 0.9, 0.0)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_off_the_16_byte_grid_and_apart(dtype):
    wide, u = logits(len(SETTINGS), 5003, dtype, 1)
    for first in (1, 3, 5, 8):
        check(wide[:, first:first + 4097], u, SETTINGS)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 640, 70000])
def test_ties_go_to_the_lowest_index(cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(7)
    u = torch.rand(len(SETTINGS), generator=g, device=DEV)
    check(torch.zeros((len(SETTINGS), cols), dtype=dtype, device=DEV), u, SETTINGS)
    two = (torch.rand((len(SETTINGS), cols), generator=g, device=DEV) < 0.3).to(dtype)
    check(two, u, SETTINGS)
    few = torch.randint(-3, 3, (len(SETTINGS), cols), generator=g, device=DEV).to(dtype)
    check(few, u, SETTINGS)
    signed = torch.where(two > 0, -0.0, 0.0).to(dtype)         # one zero
    check(signed, u, SETTINGS)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_lowest_logits(dtype):
    x, u = logits(len(SETTINGS), 3001, dtype, 11)
    low, inf = torch.finfo(dtype).min, float("inf")
    keep = torch.rand(x.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV) < 0.01
    check(x.masked_fill(~keep, -inf), u, SETTINGS)
    check(x.masked_fill(~keep, low), u, SETTINGS)
    one = torch.full_like(x, -inf)
    one[:, 1777] = -3.0
    check(one, u, SETTINGS)
    check(torch.full_like(x, -inf), u, SETTINGS)
    check(torch.full_like(x, low), u, SETTINGS)
    for at, what in ((5, float("nan")), (2999, inf), (0, float("nan"))):
        y = x.clone()
        y[:, at] = what
        y[::2, at + 1 if at < 2999 else 7] = what
        check(y, u, SETTINGS)


def test_numbers_at_the_ends():
    x, _ = logits(7, 1003, torch.bfloat16, 2)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan"), 2.0 ** -60], device=DEV)
    for s in SETTINGS:
        check(x, u, [s] * 7)
    x[:, -1] = x[:, 0] = -float("inf")      # neither end may be drawn
    for s in SETTINGS:
        check(x, u, [s] * 7)


@pytest.mark.parametrize("t", [float("inf"), 1e-38, 1e30, -1.0, float("nan"), 1e-45])
def test_temperatures_at_the_ends(t):
    x, u = logits(4, 777, torch.float32, 4)
    x[:, 5] = -float("inf")
    if t == float("inf"):        # every finite logit weighs the same
        finite = [i for i in range(777) if i != 5]
        want = [finite[int(float(v) * 776)] for v in u.tolist()]
        assert ops.sample_rows(x, u, temperature=t).tolist() == want
        return
    check(x, u, [(t, 0, 1.0, 0.0), (t, 9, 1.0, 0.0), (t, 0, 0.9, 0.0), (t, 0, 1.0, 0.1)])


@pytest.mark.parametrize("offset", [0.0, 7.0, -40.0, 330.0, 709.0, 711.0, -700.0, -730.0, 12000.0, -3e6, 1e30])
def test_logits_far_from_zero(offset):
    """Weights are of differences, wherever the logits lie; the largest weight is 1."""
    x, u = logits(24, 3001, torch.float32, 31)
    x += offset
    check(x, u, [((0.05, 0.37, 1.0, 3.3)[i % 4], (0, 50)[i // 4 % 2], (1.0, 0.9)[i // 8 % 2], (0.0, 0.01, 1.0)[i // 8]) for i in range(24)])


def test_only_the_largest_weight_is_one():
    x, u = logits(400, 700, torch.float32, 32)
    x *= torch.logspace(-3, 3, 400, device=DEV)[:, None]
    t = torch.logspace(-2, 2, 400, device=DEV)[torch.randperm(400, device=DEV)]
    assert torch.equal(ops.sample_rows(x, u, t, min_p=1.0), ops.argmax_rows(x))


def test_every_token_gets_its_share():
    """Numbers one step apart: a token of probability p is drawn n p times, to within one (its part of [0, 1) holds the steps that fit)."""
    n, cols = 4096, 50
    x, _ = logits(1, cols, torch.float32, 9)
    u = (torch.arange(n, device=DEV) + 0.5) / n
    got = torch.bincount(ops.sample_rows(x.expand(n, cols).contiguous(), u, top_k=20), minlength=cols).double()
    kept = torch.zeros(cols, dtype=torch.float64, device=DEV)
    top = x[0].topk(20).indices
    kept[top] = torch.softmax(x[0, top].double(), 0)
    assert (got - n * kept).abs().max() <= 1 + 1e-6


def test_numbers_for_all_rows_and_a_row_among_many():
    """The same settings as numbers or per row; a row's token does not depend on the rows beside it."""
    x, u = logits(300, 9000, torch.bfloat16, 8)
    full = lambda v, ty: torch.full((300,), v, dtype=ty, device=DEV)  # noqa: E731
    a = ops.sample_rows(x, u, 0.8, 40, 0.9, 0.01)
    b = ops.sample_rows(x, u, full(0.8, torch.float32), full(40, torch.int32), full(0.9, torch.float32), full(0.01, torch.float32))
    assert torch.equal(a, b)
    assert a[:5].tolist() == [int(ops.sample_rows(x[i:i + 1], u[i:i + 1], 0.8, 40, 0.9, 0.01)) for i in range(5)]
    assert ops.sample_rows(x[:0], u[:0]).shape == (0,)
    assert torch.equal(ops.sample_rows(x, u, 0.0), ops.argmax_rows(x))
    assert torch.equal(ops.sample_rows(x, u, 1.0, top_k=-2 ** 40), ops.sample_rows(x, u)) and torch.equal(ops.sample_rows(x, u, top_k=2 ** 40), ops.sample_rows(x, u))
    nan = float("nan")
    assert torch.equal(ops.sample_rows(x, u, top_p=nan, min_p=nan), ops.sample_rows(x, u))


@pytest.mark.parametrize("cols", [1000, 128256])
def test_many_tokens_of_one_row(cols):
    x, _ = logits(1, cols, torch.float32, 21)
    u = torch.arange(40, device=DEV) / 40
    assert torch.equal(ops.sample_rows(x.expand(40, -1), u, 0.8, 0, 0.9), ops.sample_rows(x.repeat(40, 1), u, 0.8, 0, 0.9))
    rows = x[0].as_strided((3, cols - 20), (10, 1))
    assert torch.equal(ops.sample_rows(rows, u[5:8], np.float32(0.8), np.int32(30)), ops.sample_rows(rows.clone(), u[5:8], 0.8, 30))


def test_captured_on_another_stream_and_replayed():
    x, u = logits(6, 4000, torch.bfloat16, 12)
    out = torch.empty(6, dtype=torch.int64, device=DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_rows(x, u, 0.8, 40, 0.9, out=out)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        ops.sample_rows(x, u, 0.8, 40, 0.9, out=out)
    for seed in (13, 14):
        y, v = logits(6, 4000, torch.bfloat16, seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        assert out.tolist() == [token(r, w, 0.8, 40, 0.9, 0.0) for r, w in zip(y.float().cpu().numpy(), v.cpu().numpy())]
