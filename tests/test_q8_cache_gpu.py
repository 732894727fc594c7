"""A cache in 8 bits against its definition: writing it (in elementary 32-bit operations, each rounded, so that codes and scales are equal) and
attention over it (in 64 bits).

Bounds per element of the attention, with e half a step of the type relative to a value, A = sum_j w_j |v_j| / sum_j w_j:  the output's rounding e |o|, at least
half a step of the numbers below the type's smallest normal one n, e n (fp16 2^-25: there steps do not shrink with the value); the weights'
rounding to fp16 2^-11 A, and 2^-31 of the largest weighted step for each that lies below fp16's normal numbers (the largest weight times scale is 2^6 at least):
keys 2^-31 c s, c the largest code and s the largest scale; sums in 32 bits 2^-24 (keys + 8) A; scores off by d = (D + 8) 2^-24 scale sum |q k| + 2^-38 scale
max|q| sum |k| (queries in fp16, the largest between 2^14 and 2^15) change a weight by 2 d of itself at most, and exponentials and logarithms of scales by 2^-19 of
themselves: (2 d + 2^-19) 2 A; weights below 2^-126 of the largest (scores 87 below it) are no normal fp32 numbers and may be lost: keys 2^-126 max|v|.  In fp32 arithmetic the weights' and queries' roundings fall away."""
import random

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CODES = (torch.int8, torch.float8_e4m3fn)
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731


def raw(t):
    return t.view(torch.uint8)


def tables_for(lens, bs, rng, spare=2, cols=None):
    need = [-(-n // bs) for n in lens]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    cols = max(1, max(need)) if cols is None else cols
    rows, at = [], 0
    for n in need:
        rows.append((order[at:at + n] + [-1] * (cols - n))[:cols])
        at += n
    return i32(rows), len(order)


def cache(pages, Hkv, bs, D, codes, seed, nan_behind=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pools = [(torch.randn((pages, Hkv, bs, D), generator=g, device=DEV) * MOST[codes] / 4).clamp(-MOST[codes], MOST[codes]).round().to(codes) for _ in range(2)]
    scales = [4 / MOST[codes] * torch.exp(torch.randn((pages, Hkv), generator=g, device=DEV)) for _ in range(2)]
    return [*pools, *scales]


# ---- writing --------------------------------------------------------------------------------------------------------------------------

def coded(y, codes):
    return y.round().clamp(-127, 127).to(codes) if codes == torch.int8 else y.to(codes)


def write_reference(k, v, cos, sin, k_pool, v_pool, k_scale, v_scale, tables, lens, starts):
    """The pools and scales afterwards, a sequence, a page and a kv head at a time."""
    Hkv, bs, D = k_pool.shape[1:]

    def turned(x):
        x, c, s = x.float(), cos.float()[:, None], sin.float()[:, None]
        return x * c + torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1) * s

    out = [t.clone() for t in (k_pool, v_pool, k_scale, v_scale)]
    for pool, scale, x in ((out[0], out[2], turned(k) if cos is not None else k.float()), (out[1], out[3], v.float())):
        for b, length in enumerate(lens):
            n = starts[b + 1] - starts[b]
            held = length - n
            for p in range(held // bs, -(-length // bs) if n else 0):
                if p >= tables.shape[1]:
                    continue
                slot = int(tables[b, p])
                if not 0 <= slot < pool.shape[0]:
                    continue
                t0, t1 = max(held, p * bs), min(length, (p + 1) * bs)
                rows = x[starts[b] + t0 - held:starts[b] + t1 - held].transpose(0, 1)       # [Hkv, t, D]
                had = scale[slot].clone() if t0 > p * bs else torch.zeros(Hkv, device=DEV)
                now = torch.maximum(torch.maximum(had, rows.abs().amax((1, 2)) * (1.0 / MOST[pool.dtype])), torch.tensor(2.0 ** -60, device=DEV))
                inverse = 1.0 / now
                grew = now != had
                old = raw(pool)[slot, :, :t0 - p * bs].clone()
                again = coded(old.view(pool.dtype).float() * (had * inverse)[:, None, None], pool.dtype)
                raw(pool)[slot, :, :t0 - p * bs] = torch.where(grew[:, None, None], raw(again), old)
                raw(pool)[slot, :, t0 - p * bs:t1 - p * bs] = raw(coded(rows * inverse[:, None, None], pool.dtype))
                scale[slot] = now
    return out


def write_case(new, lens, Hq, Hkv, D, bs, dtype, codes, seed=0, padding=0, cols=None, big=1.0):
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    starts = [sum(new[:b]) + padding for b in range(len(new) + 1)]
    n = starts[-1] + padding
    tables, pages = tables_for(lens, bs, rng, cols=cols)
    normal = lambda h: (torch.randn((n, h, D), generator=g, device=DEV) * big).to(dtype)  # noqa: E731
    angle = torch.rand((n, D // 2), generator=g, device=DEV) * 6.28
    cos, sin = (torch.cat((t, t), 1).to(dtype) for t in (angle.cos(), angle.sin()))
    return dict(q=normal(Hq), k=normal(Hkv), v=normal(Hkv), cos=cos, sin=sin, cache=cache(pages, Hkv, bs, D, codes, seed + 1), tables=tables, lens=lens, starts=starts)


def check_write(c, rope=True, starts=True, max_new=None):
    want = write_reference(c["k"], c["v"], c["cos"] if rope else None, c["sin"], *c["cache"], c["tables"], c["lens"], c["starts"])
    got = [t.clone() for t in c["cache"]]
    row_starts = i32(c["starts"]) if starts else None
    if rope:
        q = ops.rope_kv_append_q8(c["q"], c["k"], c["v"], c["cos"], c["sin"], *got, c["tables"], i32(c["lens"]), row_starts=row_starts, max_new=max_new)
        D = q.shape[2]
        x, co, si = c["q"].float(), c["cos"].float()[:, None], c["sin"].float()[:, None]
        assert torch.equal(q, (x * co + torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1) * si).to(q.dtype))
    else:
        ops.kv_append_q8(c["k"], c["v"], *got, c["tables"], i32(c["lens"]), row_starts=row_starts, max_new=max_new)
    for a, b, name in zip(got, want, ("k_pool", "v_pool", "k_scale", "v_scale")):
        same = torch.equal(raw(a), raw(b)) if a.dtype != torch.float32 else torch.equal(a, b)
        assert same, f"{name}: {int((raw(a) != raw(b)).sum())} bytes differ"
    return got


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(8, 2, 128, 16), (6, 6, 64, 32), (5, 1, 128, 64), (4, 2, 96, 16), (3, 1, 34, 5), (2, 2, 64, 8), (2, 1, 256, 16)])
def test_written_codes_are_the_definitions(Hq, Hkv, D, bs, dtype, codes):
    new = [1, 0, 37, 16, 5, 130]
    lens = [1, 9, 37, 48, 21, 200]
    check_write(write_case(new, lens, Hq, Hkv, D, bs, dtype, codes, seed=D + bs, padding=2))
    check_write(write_case(new, lens, Hq, Hkv, D, bs, dtype, codes, seed=D, padding=0), rope=False)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 32), (80, 16)])
def test_single_tokens_share_and_grow_a_pages_scale(D, bs, codes):
    """One row per sequence, without row_starts: first places, places inside a page, large numbers behind small ones, empty sequences."""
    lens = [1, 2, 16, 17, 31, 32, 33, 64, 65, 100, 7, 8]
    c = write_case([1] * len(lens), lens, 4, 2, D, bs, torch.bfloat16, codes, seed=5)
    c["k"][::3] *= 100
    c["v"][1::3] *= 0.001
    c["v"][4] = 0
    check_write(c, starts=False)
    none = write_case([1, 1], [3, 20], 4, 2, D, bs, torch.bfloat16, codes, seed=6)
    before = [t.clone() for t in none["cache"]]
    ops.kv_append_q8(none["k"], none["v"], *none["cache"], none["tables"], i32([0, -5]))
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(none["cache"], before))


@pytest.mark.parametrize("D,bs,B", [(128, 16, 10), (64, 32, 12), (64, 64, 12)])
def test_queries_among_keys_and_values(D, bs, B):
    """So many rows that the CTAs of queries lie among the others; the last ones of both kinds included."""
    check_write(write_case([700] * (B - 1) + [691], [700 + 3 * b for b in range(B - 1)] + [691], 16, 8, D, bs, torch.bfloat16, torch.int8, seed=D + bs, padding=5))


@pytest.mark.parametrize("D", [128, 48])
def test_token_by_token_like_the_definition(D):
    """A sequence of 40 tokens, one at a time, then the same in portions: each step is the definition's; the values it ends with are the tokens' up to half a
    step for each time that the scale grew."""
    torch.manual_seed(0)
    k, v = (torch.randn(40, 2, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    tables = i32([[2, 0, 1]])
    got = [torch.zeros(4, 2, 16, D, device=DEV).to(torch.int8) for _ in range(2)] + [torch.zeros(4, 2, device=DEV) for _ in range(2)]
    want = [t.clone() for t in got]
    for t in range(40):
        want = write_reference(k[t:t + 1], v[t:t + 1], None, None, *want, tables, [t + 1], [0, 1])
        ops.kv_append_q8(k[t:t + 1], v[t:t + 1], *got, tables, i32([t + 1]))
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(got, want))
    dense = ops.kv_gather_dense_q8(*got, tables, 40, torch.float32)
    for x, y, scale in ((dense[0], k, got[2]), (dense[1], v, got[3])):
        step = scale[tables[0].long()].repeat_interleave(16, 0)[:40].T[..., None]        # [Hkv, 40, 1]
        assert ((x[0] - y.float().transpose(0, 1)).abs() <= 0.5 * step * 16).all()


def test_rows_of_nobody_pages_outside_and_short_tables_are_left_alone():
    c = write_case([20, 3, 40], [30, 50, 60], 4, 2, 128, 16, torch.bfloat16, torch.int8, seed=3, padding=4, cols=3)      # 50 and 60 tokens in 3 pages
    c["tables"][0, 1] = 10 ** 6
    c["tables"][2, 0] = -7
    check_write(c)
    # starts that go backwards, beyond the rows, or have more rows than tokens: no rows
    for starts in ([0, 70, 20, 66], [-3, 20, 23, 63], [0, 20, 23, 10 ** 6]):
        got = [t.clone() for t in c["cache"]]
        ops.kv_append_q8(c["k"], c["v"], *got, c["tables"], i32(c["lens"]), row_starts=i32(starts))
    got = [t.clone() for t in c["cache"]]
    ops.kv_append_q8(c["k"], c["v"], *got, c["tables"], i32([5, 2, 7]), row_starts=i32(c["starts"]))
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(got, c["cache"]))


def test_a_bound_of_new_tokens_may_be_exact_or_loose():
    c = write_case([17, 33, 1], [17, 40, 90], 8, 4, 128, 16, torch.float16, torch.float8_e4m3fn, seed=8)
    for most in (33, 34, 51, 4096):
        check_write(c, max_new=most)


def test_strided_rows_in_place_queries_and_other_streams():
    c = write_case([5, 30], [50, 30], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=9)
    n = c["q"].shape[0]
    fused = torch.cat([c["q"].reshape(n, -1), c["k"].reshape(n, -1), c["v"].reshape(n, -1)], 1)
    want_cache = [t.clone() for t in c["cache"]]
    want = ops.rope_kv_append_q8(c["q"], c["k"], c["v"], c["cos"], c["sin"], *want_cache, c["tables"], i32(c["lens"]), row_starts=i32(c["starts"]))
    q, k, v = fused[:, :1024].unflatten(1, (8, 128)), fused[:, 1024:1280].unflatten(1, (2, 128)), fused[:, 1280:].unflatten(1, (2, 128))
    got = [t.clone() for t in c["cache"]]
    args = (i32(c["lens"]), i32(c["starts"]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.rope_kv_append_q8(q, k, v, c["cos"], c["sin"], *got, c["tables"], args[0], row_starts=args[1], q_out=q)
    torch.cuda.current_stream().wait_stream(side)
    assert out.data_ptr() == fused.data_ptr() and torch.equal(q, want)
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(got, want_cache))
    # odd strides: rows that start at no multiple of 16 bytes
    wide = torch.zeros(n, 8 * 128 + 3, dtype=torch.bfloat16, device=DEV)
    wide[:, :256] = c["k"].reshape(n, -1)
    got = [t.clone() for t in c["cache"]]
    k = wide[:, :256].unflatten(1, (2, 128))
    assert torch.equal(ops.rope_kv_append_q8(c["q"], k, c["v"], c["cos"], c["sin"], *got, c["tables"], args[0], row_starts=args[1]), want)
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(got, want_cache))


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("D", [128, 40])
def test_numbers_that_are_none_mark_their_page_and_head_alone(D, bad):
    c = write_case([20, 20], [20, 20], 2, 2, D, 16, torch.bfloat16, torch.int8, seed=4)
    clean = [t.clone() for t in c["cache"]]
    ops.kv_append_q8(c["k"], c["v"], *clean, c["tables"], i32(c["lens"]), row_starts=i32(c["starts"]))
    c["k"][3, 1, D - 1] = bad
    c["v"][30, 0, 0] = bad
    ops.kv_append_q8(c["k"], c["v"], *c["cache"], c["tables"], i32(c["lens"]), row_starts=i32(c["starts"]))
    for scale, other, b, p, h in ((c["cache"][2], clean[2], 0, 0, 1), (c["cache"][3], clean[3], 1, 0, 0)):
        page = int(c["tables"][b, p])
        assert not torch.isfinite(scale[page, h])
        scale[page, h] = other[page, h]
        assert torch.equal(scale, other)


# ---- reading back ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hkv,D,bs,n", [(2, 128, 16, 100), (3, 64, 32, 64), (1, 128, 64, 1), (2, 36, 5, 33), (2, 64, 16, 0), (1, 96, 16, 50), (2, 64, 8, 23)])
def test_reading_back(Hkv, D, bs, n, dtype, codes):
    rng = random.Random(n)
    tables, pages = tables_for([n + 3, n, n], bs, rng)
    c = cache(pages, Hkv, bs, D, codes, 7)
    tables[1, 0] = -1 if n else tables[1, 0]
    k, v = ops.kv_gather_dense_q8(*c, tables, n, dtype)
    t = torch.arange(n, device=DEV)
    for got, pool, scale in ((k, c[0], c[2]), (v, c[1], c[3])):
        page = tables.long()[:, t // bs]
        at = page.clamp(0, pages - 1)
        x = raw(pool)[at, :, t % bs].view(codes).float() * scale[at][..., None]        # [B, n, Hkv, D]
        x = torch.where((page < 0)[..., None, None], 0.0, x)
        assert torch.equal(got, x.transpose(1, 2).to(dtype))


# ---- attention --------------------------------------------------------------------------------------------------------------------------

def attention_reference(q, k_pool, v_pool, k_scale, v_scale, tables, lens, starts, scale, half):
    """(values, bound) in 64 bits; `half`: weights and queries in fp16."""
    Hkv, bs, D = k_pool.shape[1:]
    Hq, G = q.shape[1], q.shape[1] // Hkv
    out, bound = torch.full(q.shape, float("nan"), dtype=F64, device=DEV), torch.zeros(q.shape, dtype=F64, device=DEV)
    e = torch.finfo(q.dtype).eps / 2
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        keys = max(0, min(length, tables.shape[1] * bs))
        pos = torch.arange(keys, device=DEV)
        page = tables[b].long()[pos // bs]
        bad, at = (page < 0) | (page >= k_pool.shape[0]), page.clamp(0, k_pool.shape[0] - 1)
        k, v = (torch.where(bad[:, None, None], 0.0, raw(p)[at, :, pos % bs].view(p.dtype).to(F64) * s[at][..., None].to(F64)).repeat_interleave(G, 1)
                for p, s in ((k_pool, k_scale), (v_pool, v_scale)))
        qq = q[starts[b]:starts[b + 1]].to(F64)
        see = pos[None] <= (length - n + torch.arange(n, device=DEV))[:, None]
        s = torch.einsum("nhd,khd->nhk", qq, k) * scale
        w = torch.where(see[:, None], s, -float("inf"))
        w = torch.softmax(w, -1) if keys else w
        o, A = torch.einsum("nhk,khd->nhd", w, v), torch.einsum("nhk,khd->nhd", w, v.abs())
        d = (D + 8) * 2.0 ** -24 * abs(scale) * torch.einsum("nhd,khd->nhk", qq.abs(), k.abs())
        if half:
            d = d + 2.0 ** -38 * abs(scale) * qq.abs().amax(-1, keepdim=True) * k.abs().sum(-1).T[None]
        d = torch.where(see[:, None], d, 0.0).amax(-1) if keys else torch.zeros(n, Hq, dtype=F64, device=DEV)
        t = e * o.abs().clamp_min(torch.finfo(q.dtype).smallest_normal) + 2.0 ** -24 * (keys + 8) * A + ((2 * d + 2.0 ** -19) * 2)[..., None] * A + keys * 2.0 ** -126 * (v.abs().max() if keys else 0.0)
        if half and keys:
            t = t + 2.0 ** -11 * A + keys * 2.0 ** -31 * MOST[v_pool.dtype] * v_scale[at].max()
        out[starts[b]:starts[b + 1]], bound[starts[b]:starts[b + 1]] = o, t
    return out, bound


def attention_case(new, lens, Hq, Hkv, D, bs, dtype, codes, seed=0, cols=None, gap=0):
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    tables, pages = tables_for(lens, bs, rng, cols=cols)
    starts = [gap + sum(new[:b]) for b in range(len(new) + 1)]
    q = (torch.randn((starts[-1] + gap, Hq, D), generator=g, device=DEV) * 1.5).to(dtype)
    c = cache(pages, Hkv, bs, D, codes, seed)
    if codes == torch.float8_e4m3fn:        # what is behind a sequence's last token may be no number
        for b, n in enumerate(lens):
            if n % bs and n // bs < tables.shape[1]:
                for p in c[:2]:
                    raw(p)[int(tables[b, n // bs]), :, n % bs:] = 0x7f
    return dict(q=q, cache=c, tables=tables, lens=lens, starts=starts)


def near(got, want, bound, what=""):
    off = (got.to(F64) - want).abs()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), f"{what}: off by {off.max().item():.3g}, {worst:.3g} over the bound"


SIZES = [(32, 8, 128, 16), (8, 8, 64, 16), (16, 2, 64, 32), (10, 2, 128, 64), (12, 1, 128, 16), (32, 2, 128, 32), (4, 2, 96, 16), (3, 1, 33, 5), (4, 4, 256, 16), (4, 2, 128, 8)]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,bs", SIZES)
def test_decode_attention(Hq, Hkv, D, bs, dtype, codes):
    lens = [1, 16, 17, 0, 250, 64, 333, 1000]
    c = attention_case([1] * len(lens), lens, Hq, Hkv, D, bs, dtype, codes, seed=D + Hq)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, dtype != torch.float32)
    got = ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), max(lens))
    assert (got[3] == 0).all()
    keep = [b for b in range(len(lens)) if b != 3]
    near(got[keep], want[keep], bound[keep])
    plain = ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), max(lens), flags=ops.ATTN_FORCE_GENERIC)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, False)
    near(plain[keep], want[keep], bound[keep], "fp32 arithmetic")


@pytest.mark.parametrize("B,context", [(1, 5000), (1, 40000), (3, 9001), (40, 700), (64, 130)])
@pytest.mark.parametrize("codes", CODES)
def test_decode_attention_of_few_long_and_many_short_sequences(B, context, codes):
    rng = random.Random(B)
    lens = [context] + [rng.randint(1, context) for _ in range(B - 1)]
    c = attention_case([1] * B, lens, 16, 4, 128, 16, torch.bfloat16, codes, seed=B)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], 128 ** -0.5, True)
    near(ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), context), want, bound)
    near(ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), 4 * context), want, bound, "a loose bound of the lengths")


PORTIONS = [([1, 1, 1], [1, 40, 300]), ([5, 0, 33, 2], [5, 7, 100, 64]), ([150], [150]), ([129, 64], [700, 64]), ([300, 1, 17, 63], [300, 999, 17, 1500])]


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,bs", SIZES)
def test_prompt_attention(Hq, Hkv, D, bs, dtype, codes):
    for i, (new, lens) in enumerate(PORTIONS):
        c = attention_case(new, lens, Hq, Hkv, D, bs, dtype, codes, seed=D + Hq + i, gap=i)
        want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, dtype != torch.float32)
        out = torch.full_like(c["q"], 7.0)
        ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(new), max(lens), out=out)
        a, e = c["starts"][0], c["starts"][-1]
        near(out[a:e], want[a:e], bound[a:e], str(new))
        assert (out[:a] == 7).all() and (out[e:] == 7).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("new,lens", [([600], [9000]), ([40], [30000]), ([2000, 3], [2000, 5000]), ([9] * 30, list(range(300, 3300, 100)))])
def test_prompt_attention_of_long_contexts(new, lens, codes):
    c = attention_case(new, lens, 8, 2, 128, 16, torch.bfloat16, codes, seed=len(new))
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], 128 ** -0.5, True)
    near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(new), max(lens)), want, bound)
    near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(new) + 100, max(lens) * 2), want, bound, "loose bounds")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_any_scale(scale, dtype):
    new, lens = [1, 30], [200, 90]
    c = attention_case(new, lens, 8, 2, 128, 16, dtype, torch.int8, seed=1)
    c["q"] *= 0.3
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], scale, dtype != torch.float32)
    near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), 30, 200, scale=scale), want, bound)
    one = attention_case([1, 1], lens, 8, 2, 128, 16, dtype, torch.int8, seed=1)
    want, bound = attention_reference(one["q"], *one["cache"], one["tables"], lens, one["starts"], scale, dtype != torch.float32)
    near(ops.paged_decode_attention_q8(one["q"], *one["cache"], one["tables"], i32(lens), 200, scale=scale), want, bound)


def test_large_and_small_queries_and_scales():
    """Queries far above and below fp16's range, values' scales 2^40 apart, a page of zeros at the smallest scale."""
    lens = [120, 120]
    c = attention_case([1, 1], lens, 4, 2, 128, 16, torch.bfloat16, torch.int8, seed=2)
    c["q"][0] *= 2.0 ** 100
    c["cache"][2] *= 2.0 ** -100
    c["q"][1] *= 2.0 ** -20
    page = c["tables"][1].tolist()
    c["cache"][3][page[0]] *= 2.0 ** 20
    c["cache"][3][page[1]] *= 2.0 ** -20
    c["cache"][3][page[2]] = 2.0 ** -60
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], 128 ** -0.5, True)
    near(ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), 120), want, bound)
    near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), 1, 120), want, bound)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scales_that_are_no_numbers_reach_the_rows_that_see_them(which, bad):
    new, lens = [40, 40], [100, 40]
    c = attention_case(new, lens, 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=3)
    clean = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), 40, 100)
    c["cache"][which][int(c["tables"][0, 5]), 1] = bad        # tokens 80 .. 95 of sequence 0: rows 20 on see them
    got = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), 40, 100)
    assert not torch.isfinite(got[20:40, 4:]).any() if bad != bad else not torch.isfinite(got[36:40, 4:]).all()
    assert torch.equal(got[:, :4], clean[:, :4]) and torch.equal(got[40:], clean[40:])
    one = ops.paged_decode_attention_q8(c["q"][[39, 79]], *c["cache"], c["tables"], i32(lens), 100)
    assert not torch.isfinite(one[0, 4:]).all() and torch.isfinite(one[0, :4]).all() and torch.isfinite(one[1]).all()


def test_bad_tables_read_zeros_and_short_tables_end_the_context():
    new, lens = [3, 20], [90, 100]
    c = attention_case(new, lens, 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=4, cols=6)      # 96 tokens
    c["tables"][0, 2] = -3
    c["tables"][0, 4] = 2 ** 30
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], 128 ** -0.5, True)
    got = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), 20, 100)
    near(got, want, bound)
    lens = [90, 100]
    one = attention_case([1, 1], lens, 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=4, cols=6)
    one["tables"][0, 2] = -3
    want, bound = attention_reference(one["q"], *one["cache"], one["tables"], lens, one["starts"], 128 ** -0.5, True)
    near(ops.paged_decode_attention_q8(one["q"], *one["cache"], one["tables"], i32(lens), 100), want, bound)


@pytest.mark.parametrize("codes", CODES)
def test_offsets_past_32_bits(codes):
    """Pages behind the first 2^31 numbers of a pool, and behind 2^32: as in a small one."""
    pages, Hkv, bs, D = (2 ** 32 + 2 ** 28) // (8 * 16 * 128), 8, 16, 128
    shift = pages - 40
    c = write_case([50, 3], [50, 200], 16, Hkv, D, bs, torch.bfloat16, codes, seed=31)
    small = [t.clone() for t in c["cache"]]
    n = small[0].shape[0]
    big = [torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device=DEV) for t in small]
    for past in (shift, 2 ** 31 // (Hkv * bs * D) - n // 2):
        for b, t in zip(big, c["cache"]):
            raw(b)[past:past + n] = raw(t)
        far = torch.where(c["tables"] >= 0, c["tables"] + past, -1)
        outs = []
        for pools, tables in ((big, far), ([t.clone() for t in c["cache"]], c["tables"])):
            q = ops.rope_kv_append_q8(c["q"], c["k"], c["v"], c["cos"], c["sin"], *pools, tables, i32(c["lens"]), row_starts=i32(c["starts"]), max_new=50)
            outs.append((q, *ops.kv_gather_dense_q8(*pools, tables, 64), ops.paged_decode_attention_q8(q[:2], *pools, tables, i32(c["lens"]), 200),
                         ops.paged_prompt_attention_q8(q, *pools, tables, i32(c["lens"]), i32(c["starts"]), 50, 200),
                         ops.paged_prompt_attention_q8(q, *pools, tables, i32(c["lens"]), i32(c["starts"]), 50, 200, flags=ops.ATTN_FORCE_GENERIC)))
        for a, b in zip(*outs):
            assert torch.equal(a, b)


def test_lengths_that_do_not_fit_give_no_rows():
    c = attention_case([3, 20], [90, 100], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=5)
    for lens, starts in (([90, 10], [0, 3, 23]), ([90, 100], [0, 3, 10 ** 6]), ([90, 100], [0, 3, -5])):
        out = torch.full_like(c["q"], 7.0)
        ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(starts), 20, 100, out=out)
        assert (out[3:] == 7).all() and not (out[:3] == 7).all()
    assert (ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], i32([0, -9]), 100) == 0).all()


def test_captured_calls_replay_with_new_lengths_and_rows():
    c = attention_case([4, 20], [700, 900], 16, 4, 128, 16, torch.bfloat16, torch.int8, seed=6)
    lens, starts = i32([100, 200]), i32([0, 4, 24])
    out, one = torch.zeros_like(c["q"]), torch.zeros_like(c["q"][:2])
    g = torch.cuda.CUDAGraph()

    def calls():
        ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], lens, starts, 20, 900, out=out)
        ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 900, out=one)

    calls()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        calls()
    for l in ([700, 900], [4, 20], [555, 311]):
        lens.copy_(i32(l))
        g.replay()
        want, bound = attention_reference(c["q"], *c["cache"], c["tables"], l, [0, 4, 24], 128 ** -0.5, True)
        near(out, want, bound, str(l))
        want, bound = attention_reference(c["q"][:2], *c["cache"], c["tables"], l, [0, 1, 2], 128 ** -0.5, True)
        near(one, want, bound, str(l))


@pytest.mark.parametrize("bs", [16, 64])
def test_written_and_read_behind_copies_and_other_streams_calls(bs):
    """Writing and reading begin while what is ahead ends: behind a copy, a clearing, their own kernels and another stream's, launched and captured."""
    cases = [write_case([3, 1, 40], [70, 200, 40], 8, 2, 128, bs, torch.bfloat16, torch.int8, seed=s) for s in (11, 12, 13)]
    a = cases[0]
    names, tables, lens, starts = ("q", "k", "v", "cos", "sin"), a["tables"], i32(a["lens"]), i32(a["starts"])
    rows, pools, others = {x: torch.empty_like(a[x]) for x in names}, [torch.empty_like(t) for t in a["cache"]], [torch.empty_like(t) for t in a["cache"]]
    given, side = {x: torch.empty_like(a[x]) for x in names}, torch.cuda.Stream()

    def calls():
        for x in names:
            rows[x].copy_(given[x])
        for t in (*pools, *others):
            raw(t).zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.kv_append_q8(rows["k"], rows["v"], *others, tables, lens, row_starts=starts, max_new=40)
        q = ops.rope_kv_append_q8(rows["q"], rows["k"], rows["v"], rows["cos"], rows["sin"], *pools, tables, lens, row_starts=starts, max_new=40)
        torch.cuda.current_stream().wait_stream(side)
        rows["k"].zero_()
        rows["q"].copy_(q)
        read = [ops.kv_gather_dense_q8(*c, tables, 40) for c in (others, pools)]
        one = ops.paged_decode_attention_q8(q[:3], *pools, tables, lens, 200)
        ops.kv_append_q8(rows["k"], rows["v"], *pools, tables, lens, row_starts=starts, max_new=40)        # (what was read is written over)
        return [q, *read[0], *read[1], one, rows["q"]]

    def wanted(c):
        cleared = [torch.zeros_like(t) for t in c["cache"]]
        with_rope, without = (write_reference(c["k"], c["v"], cos, c["sin"], *cleared, tables, c["lens"], c["starts"]) for cos in (c["cos"], None))
        co, si, x = c["cos"].float()[:, None], c["sin"].float()[:, None], c["q"].float()
        q = (x * co + torch.cat((-x[..., 64:], x[..., :64]), -1) * si).to(x.dtype).to(torch.bfloat16)
        kv = [(pool[tables[:, 0].long()].float() * scale[tables[:, 0].long(), :, None, None])[:, :, :16] for w in (without, with_rope) for pool, scale in ((w[0], w[2]), (w[1], w[3]))]
        return q, [t.to(torch.bfloat16) for t in kv], attention_reference(q[:3], *with_rope, tables, c["lens"], [0, 1, 2, 3], 128 ** -0.5, True)

    def check(c, got):
        q, kv, (one, bound) = wanted(c)
        assert torch.equal(got[0], q) and torch.equal(got[6], q)
        for x, y in zip(got[1:5], kv):
            assert torch.equal(x[:, :, :16], y)        # the first page's, or a part of it
        near(got[5], one, bound)

    def give(c):
        for x in names:
            given[x].copy_(c[x])

    for c in cases:
        give(c)
        check(c, calls())
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = calls()
    for c in cases:
        give(c)
        g.replay()
        check(c, got)
        g.replay()
        g.replay()        # one behind the other
        check(c, got)


def test_two_streams_at_once_and_strided_queries():
    c = attention_case([64, 64], [3000, 2000], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=7)
    lens, starts = i32(c["lens"]), i32(c["starts"])
    want = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], lens, starts, 64, 3000)
    ones = ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 3000)
    wide = torch.zeros(128, 3, 8, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 1] = c["q"]
    odd = torch.zeros(128, 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)
    odd[:, 1:] = c["q"].flatten(1)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.paged_prompt_attention_q8(wide[:, 1], *c["cache"], c["tables"], lens, starts, 64, 3000),
                            ops.paged_decode_attention_q8(wide[:2, 1], *c["cache"], c["tables"], lens, 3000)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, ones) for a, b in got)
    exact, bound = attention_reference(c["q"], *c["cache"], c["tables"], c["lens"], c["starts"], 128 ** -0.5, True)
    near(ops.paged_prompt_attention_q8(odd[:, 1:].unflatten(1, (8, 128)), *c["cache"], c["tables"], lens, starts, 64, 3000), exact, bound)


def test_written_then_read_like_a_prompt_and_its_decoding():
    """Portions written and attended to, then single tokens: as attention over the tokens themselves, up to half a step of their pages' codes."""
    torch.manual_seed(3)
    B, Hq, Hkv, D, T = 3, 8, 2, 128, 70
    k, v, q = (torch.randn(B, T, h, D, device=DEV, dtype=torch.bfloat16) for h in (Hkv, Hkv, Hq))
    tables = i32([[4, 9, 2, 7, 11], [0, 1, 3, 5, 6], [8, 10, 12, 13, 14]])
    pools = [torch.zeros(15, Hkv, 16, D, device=DEV, dtype=torch.int8) for _ in range(2)] + [torch.zeros(15, Hkv, device=DEV) for _ in range(2)]
    for lo, hi in ((0, 40), (40, 53), (53, 54), (54, 70)):
        n = hi - lo
        rows = [x[:, lo:hi].reshape(B * n, -1, D).contiguous() for x in (q, k, v)]
        lens, starts = i32([hi] * B), i32([i * n for i in range(B + 1)])
        ops.kv_append_q8(rows[1], rows[2], *pools, tables, lens, row_starts=starts, max_new=n)
        if n == 1:
            got = ops.paged_decode_attention_q8(rows[0], *pools, tables, lens, hi)
        else:
            got = ops.paged_prompt_attention_q8(rows[0], *pools, tables, lens, starts, n, hi)
        kk, vv = (x[:, :hi].float().transpose(1, 2).repeat_interleave(Hq // Hkv, 1) for x in (k, v))
        s = torch.einsum("bnhd,bhkd->bhnk", q[:, lo:hi].float(), kk) * D ** -0.5
        s = s.masked_fill(torch.arange(hi, device=DEV)[None] > torch.arange(lo, hi, device=DEV)[:, None], -float("inf"))
        want = torch.einsum("bhnk,bhkd->bnhd", torch.softmax(s, -1), vv).reshape(B * n, Hq, D)
        rel = ((got.float() - want).norm() / want.norm()).item()
        # a step is max / 127 with max about 4.5 of the standard deviation: errors uniform in half a step, 4.5 / 127 / sqrt(12) = 0.0102 of the values, and the
        # scores off by as much (their deviation is 1), which moves the weights; rescaled pages twice that, bf16 0.0017
        assert rel < 0.04, rel


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------

def test_refusals():
    c = attention_case([3, 20], [90, 100], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=8)
    k_pool, v_pool, k_scale, v_scale = c["cache"]
    lens, starts = i32(c["lens"]), i32(c["starts"])
    prompt = lambda **over: ops.paged_prompt_attention_q8(**{**dict(  # noqa: E731
        q=c["q"], k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, block_tables=c["tables"], context_lens=lens, row_starts=starts, max_new=20,
        max_context_len=100), **over})
    prompt()
    with pytest.raises(TypeError):
        prompt(k_pool=k_pool.to(torch.bfloat16), v_pool=v_pool.to(torch.bfloat16))
    with pytest.raises(TypeError):
        prompt(q=c["q"].double())
    for over in (dict(v_pool=v_pool[:-1]), dict(k_scale=k_scale.half()), dict(v_scale=v_scale.T.contiguous().T), dict(k_pool=k_pool[:, :, ::2]),
                 dict(block_tables=c["tables"].long()), dict(block_tables=c["tables"][:1]), dict(context_lens=lens.long()), dict(row_starts=starts[:-1]),
                 dict(q=c["q"][..., :64]), dict(q=c["q"][:, :7]), dict(out=c["q"][:5]), dict(out=c["q"].float()), dict(block_tables=c["tables"].cpu().to(DEV)[:, :0])):
        with pytest.raises(ValueError):
            prompt(**over)
    with pytest.raises(_lib.B200LibraryError):
        prompt(q=c["q"].cpu())
    with pytest.raises(_lib.B200LibraryError):
        prompt(max_new=-1)
    with pytest.raises(ValueError):
        ops.paged_decode_attention_q8(c["q"], k_pool, v_pool, k_scale, v_scale, c["tables"], lens, 100)
    with pytest.raises(ValueError):
        ops.kv_gather_dense_q8(k_pool, v_pool, k_scale, v_scale, c["tables"], 10 ** 6)
    with pytest.raises(TypeError):
        ops.kv_gather_dense_q8(k_pool, v_pool, k_scale, v_scale, c["tables"], 5, torch.int8)
    w = write_case([3, 20], [90, 100], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=8)
    write = lambda **over: ops.rope_kv_append_q8(**{**dict(  # noqa: E731
        q=w["q"], k=w["k"], v=w["v"], cos=w["cos"], sin=w["sin"], k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, block_tables=c["tables"],
        context_lens=lens, row_starts=starts), **over})
    for over in (dict(cos=None), dict(cos=None, sin=None), dict(row_starts=None), dict(k=w["k"][:5]), dict(cos=w["cos"][:, :64]), dict(v=w["v"][:, :1]),
                 dict(k=w["k"].transpose(1, 2)), dict(q_out=w["q"][:, :4])):
        with pytest.raises(ValueError):
            write(**over)
    for over in (dict(v=w["v"].float()), dict(q_out=w["q"].float())):
        with pytest.raises(TypeError):
            write(**over)
    for over in (dict(v_pool=k_pool), dict(v_scale=k_scale)):
        with pytest.raises(_lib.B200LibraryError, match="of their own"):
            write(**over)
    with pytest.raises(TypeError):
        write(cos=w["cos"].float())
    with pytest.raises(TypeError):
        write(q=w["q"].float())


def test_calls_with_and_without_the_fast_module(monkeypatch):
    """The same outputs, bits and strides of both ways in; what the fast one does not take goes through the other."""
    assert _lib.fast_calls() is not None
    c = attention_case([4, 20], [700, 900], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=11)
    w = write_case([3, 20], [90, 100], 8, 2, 128, 16, torch.float16, torch.float8_e4m3fn, seed=12)
    lens, starts = i32(c["lens"]), i32(c["starts"])
    wide = torch.zeros(24, 3, 8, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 1] = c["q"]

    def calls():
        pools = [t.clone() for t in w["cache"]]
        plain = [t.clone() for t in w["cache"]]
        q = ops.rope_kv_append_q8(w["q"], w["k"], w["v"], w["cos"], w["sin"], *pools, w["tables"], i32(w["lens"]), row_starts=i32(w["starts"]), max_new=20)
        ops.kv_append_q8(w["k"], w["v"], *plain, w["tables"], i32(w["lens"]), row_starts=i32(w["starts"]))
        k, v = ops.kv_gather_dense_q8(*pools, w["tables"][:, :6], 90, torch.float32)
        return [q, *pools, *plain, k, v, ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 900),
                ops.paged_decode_attention_q8(wide[:2, 1], *c["cache"], c["tables"], lens, 900, scale=0.1),
                ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 900, scale=1),
                ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], lens, starts, 20, 900),
                ops.paged_prompt_attention_q8(wide[:, 1], *c["cache"], c["tables"], lens, starts, 20, 900, scale=0.1)]

    fast = calls()
    with torch.inference_mode():
        inference = calls()
    monkeypatch.setattr(_lib, "fast_calls", lambda: None)
    for got in (inference, calls()):
        assert all(a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(raw(a.contiguous()), raw(b.contiguous())) for a, b in zip(fast, got))


def test_a_workspace_of_the_callers():
    c = attention_case([100, 100], [3000, 2000], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=13)
    lens, starts = i32(c["lens"]), i32(c["starts"])
    want = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], lens, starts, 100, 3000)
    one = ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 3000)
    for call, need, expect in ((lambda **k: ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], lens, starts, 100, 3000, **k),
                                ops.prompt_attention_q8_workspace(2, 100, 8, 2, 128, 16, 3000, torch.bfloat16), want),
                               (lambda **k: ops.paged_decode_attention_q8(c["q"][:2], *c["cache"], c["tables"], lens, 3000, **k),
                                ops.decode_attention_q8_workspace(2, 8, 2, 128, 16, 3000, torch.bfloat16), one)):
        assert need > 0
        ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device=DEV)
        assert torch.equal(call(workspace=ws[:need]), expect) and (ws[need:] == 0xff).all()
        with pytest.raises(_lib.B200LibraryError, match="workspace"):
            call(workspace=ws[:need - 16])
        with pytest.raises(_lib.B200LibraryError, match="aligned"):
            call(workspace=ws[4:need + 4])
        with pytest.raises(ValueError):
            call(workspace=ws.cpu())


def test_nothing_to_do():
    """No sequences, no rows, no new tokens: empty outputs, and nothing is written."""
    c = attention_case([3, 20], [90, 100], 8, 2, 128, 16, torch.bfloat16, torch.int8, seed=14)
    none, no_tables, q0 = i32([]), c["tables"][:0], c["q"][:0]
    before = [raw(t).clone() for t in c["cache"]]
    assert ops.paged_decode_attention_q8(q0, *c["cache"], no_tables, none, 100).shape == (0, 8, 128)
    assert ops.paged_prompt_attention_q8(q0, *c["cache"], no_tables, none, i32([0]), 0, 0).shape == (0, 8, 128)
    assert ops.paged_prompt_attention_q8(q0, *c["cache"], c["tables"], i32([90, 100]), i32([0, 0, 0]), 0, 100).shape == (0, 8, 128)
    assert [t.shape for t in ops.kv_gather_dense_q8(*c["cache"], no_tables, 5)] == [(0, 2, 5, 128)] * 2
    assert [t.shape for t in ops.kv_gather_dense_q8(*c["cache"], c["tables"], 0)] == [(2, 2, 0, 128)] * 2
    kv, angle = q0[:, :2], torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.rope_kv_append_q8(q0, kv, kv, angle, angle, *c["cache"], c["tables"], i32([90, 100]), row_starts=i32([0, 0, 0])).shape == (0, 8, 128)
    ops.kv_append_q8(kv, kv, *c["cache"], no_tables, none)
    out = torch.full_like(c["q"], 7.0)
    ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32([90, 100]), i32([5, 5, 5]), 20, 100, out=out)
    assert (out == 7).all() and all(torch.equal(a, raw(b)) for a, b in zip(before, c["cache"]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("G,new", [(1, 8), (1, 9), (1, 16), (1, 17), (3, 5), (4, 4), (4, 8), (9, 1), (16, 1), (20, 1), (16, 2), (5, 13), (8, 16), (7, 37)])
def test_rows_around_the_blocks_of_the_kernels(G, new, codes, dtype):
    """Rows of a sequence and kv head on both sides of 8, 16, 32, 128 and 256; ragged, with a part of the keys that some rows do not see."""
    lens = [2000, new, new + 3, 530]
    counts = [new, new, max(1, new // 2), max(1, new - 1)]
    for Hkv, D in ((2, 128), (1, 64)):
        c = attention_case(counts, lens, G * Hkv, Hkv, D, 16, dtype, codes, seed=G * 100 + new, gap=1)
        want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
        a, e = c["starts"][0], c["starts"][-1]
        near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, 2000)[a:e], want[a:e], bound[a:e])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("G,new,D", [(1, 17, 64), (4, 8, 128), (4, 9, 128), (5, 13, 64), (12, 8, 128), (3, 32, 64), (7, 14, 128), (1, 128, 128), (1, 129, 128)])
def test_rows_of_many_sequences(G, new, D, codes, dtype):
    """Rows of 17 to 129 in nine sequences of 8 kv heads, more than are taken 16 at a time; one sequence's last page has a scale that is no number."""
    lens = [700, new, new + 3, 530, 64, 129, 1, 256, 300]
    counts = [new, new, max(1, new // 2), new - 1, min(new, 60), new, 1, min(new, 33), 16]
    c = attention_case(counts, lens, G * 8, 8, D, 32, dtype, codes, seed=G * 100 + new, gap=2)
    a, e, hurt = c["starts"][0], c["starts"][-1], lens[3] // 32
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
    kept = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(counts), 700)
    near(kept[a:e], want[a:e], bound[a:e])
    c["cache"][3][int(c["tables"][3, hurt]), 5] = float("inf")
    got = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(counts), 700)
    see = torch.zeros(got.shape[:2], dtype=torch.bool, device=DEV)
    first = c["starts"][3] + max(0, hurt * 32 - (lens[3] - counts[3]))        # the first row that sees the page
    see[first:c["starts"][4], 5 * G:6 * G] = True
    assert not torch.isfinite(got[see]).any() and torch.equal(got[a:e][~see[a:e]], kept[a:e][~see[a:e]])


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("G,new", [(3, 70), (5, 9), (6, 3)])
def test_pages_of_48_and_three_kv_heads(G, new, D, dtype):
    """Numbers that are no powers of two everywhere: pages, heads, sequences, query heads of a kv head, parts."""
    lens = [new, 1000, 47 + new, 48 + new, 333]
    counts = [new, new, new - 1, new, 1]
    c = attention_case(counts, lens, G * 3, 3, D, 48, dtype, torch.int8, seed=G + D)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
    near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, 1000), want, bound)
    want, bound = attention_reference(c["q"][:5], *c["cache"], c["tables"], lens, list(range(6)), D ** -0.5, True)
    near(ops.paged_decode_attention_q8(c["q"][:5], *c["cache"], c["tables"], i32(lens), 1000), want, bound)


@pytest.mark.parametrize("G,new,context,D", [(4, 16, 2100, 128), (4, 32, 700, 128), (1, 100, 900, 64), (3, 21, 1500, 128), (8, 8, 3000, 64)])
def test_rows_of_one_sequence_in_several_blocks(G, new, context, D):
    """Rows of up to 128 of a sequence and kv head, 16 at a time: alone, and more of them than there are keys before."""
    for lens in ([context], [new]):
        c = attention_case([new], lens, G * 8, 8, D, 16, torch.bfloat16, torch.int8, seed=G + new)
        want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
        near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, context), want, bound)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("G,new,dtype", [(2, 4, torch.bfloat16), (2, 8, torch.float16), (4, 30, torch.bfloat16), (4, 100, torch.float16), (2, 20, torch.float32)])
def test_rows_that_do_not_see_a_page_do_not_meet_its_scale(G, new, dtype, bad, which):
    """The page of the last tokens: earlier tokens' rows come out as they did, the rows behind see no number."""
    length = 96 + new if new < 16 else 160
    c = attention_case([new], [length], 2 * G, 2, 128, 16, dtype, torch.int8, seed=15)
    call = lambda: ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32([length]), i32([0, new]), new, length)  # noqa: E731
    clean = call()
    page = (length - 2) // 16
    c["cache"][which][int(c["tables"][0, page])] = bad
    got = call()
    first = max(0, page * 16 - (length - new))      # the first row that sees it
    assert torch.equal(got[:first], clean[:first])
    if bad != bad:
        assert not torch.isfinite(got[first:]).any()
    else:
        assert not torch.isfinite(got[first:]).all()


def test_numbers_that_are_none_in_a_prompt_reach_later_rows_only():
    """A key that is not finite, written among others: earlier pages' rows are as without it."""
    for codes in CODES:
        w = write_case([40], [40], 8, 2, 128, 16, torch.bfloat16, codes, seed=16)
        outs = []
        for bad in (False, True):
            if bad:
                w["k"][20, 0, 5], w["v"][37, 1, 9] = float("nan"), float("inf")
            pools = [t.clone() for t in w["cache"]]
            q = ops.rope_kv_append_q8(w["q"], w["k"], w["v"], w["cos"], w["sin"], *pools, w["tables"], i32([40]), row_starts=i32([0, 40]))
            outs.append(ops.paged_prompt_attention_q8(q, *pools, w["tables"], i32([40]), i32([0, 40]), 40, 40))
        assert torch.equal(outs[0][:16], outs[1][:16]) and torch.equal(outs[0][16:32, 4:], outs[1][16:32, 4:])
        assert not torch.isfinite(outs[1][16:, :4]).any() and not torch.isfinite(outs[1][32:, 4:]).all()


@pytest.mark.parametrize("codes,dtype", [(torch.int8, torch.bfloat16), (torch.float8_e4m3fn, torch.float16)])
@pytest.mark.parametrize("B,new,Hq,Hkv,D,context", [(1, 1301, 9, 3, 64, 0), (3, 101, 5, 1, 128, 1200), (1, 207, 5, 1, 128, 2048), (9, 127, 1, 1, 128, 1273), (5, 193, 1, 1, 64, 1217),
                                                    (23, 33, 1, 1, 64, 2267), (5, 33, 3, 1, 128, 20000)])
def test_an_odd_number_of_parts(B, new, Hq, Hkv, D, context, codes, dtype):
    """Sequences, heads, rows and parts whose product is odd, in one row block and in two: the parts' outputs lie behind an odd number of statistics.  Scratch of the allocator,
    and the caller's with something behind it."""
    lens = [new + context] + [new + context - 7 * b for b in range(1, B)]
    need = ops.prompt_attention_q8_workspace(B, new, Hq, Hkv, D, 16, lens[0], dtype)
    rows = B * new * Hq
    assert need // (rows * (8 + 4 * D)) * rows % 2 == 1 and need % 16 == 0
    c = attention_case([new] + [new - 2 * (b % 9) for b in range(1, B)], lens, Hq, Hkv, D, 16, dtype, codes, seed=new)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
    call = lambda **k: ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, lens[0], **k)  # noqa: E731
    got = call()
    near(got, want, bound)
    ws = torch.full((need + 256,), 0xff, dtype=torch.uint8, device=DEV)
    assert torch.equal(call(workspace=ws[:need]), got) and (ws[need:] == 0xff).all()


@pytest.mark.parametrize("what", ["append", "gather", "decode", "prompt"])
def test_transformed_tensors_are_refused(what):
    """Tensors without storage (their type is torch.Tensor): an error, as from the checks without the fast module, and the next plain call runs."""
    c = attention_case([2, 3], [40, 50], 8, 2, 64, 16, torch.bfloat16, torch.int8, seed=3)
    w = write_case([2, 3], [40, 50], 8, 2, 64, 16, torch.bfloat16, torch.int8, seed=3)
    lens, starts, one = i32([40, 50]), i32(c["starts"]), i32([40])
    call = dict(
        append=lambda q: ops.rope_kv_append_q8(q, w["k"], w["v"], w["cos"], w["sin"], *w["cache"], w["tables"], lens, row_starts=starts, max_new=3),
        gather=lambda s: ops.kv_gather_dense_q8(c["cache"][0], c["cache"][1], s, c["cache"][3], c["tables"], 20)[0],
        decode=lambda q: ops.paged_decode_attention_q8(q[:1], *c["cache"], c["tables"][:1], one, 40),
        prompt=lambda q: ops.paged_prompt_attention_q8(q, *c["cache"], c["tables"], lens, starts, 3, 50))[what]
    x = c["cache"][2] if what == "gather" else c["q"]
    want = call(x)
    before = [raw(t).clone() for t in w["cache"]]
    for transformed in (lambda: torch.vmap(call)(torch.stack((x, x))), lambda: torch.func.grad(lambda y: call(y).float().sum())(x)):
        with pytest.raises(RuntimeError, match="storage"):
            transformed()
    assert all(torch.equal(a, raw(b)) for a, b in zip(before, w["cache"])) and torch.equal(call(x), want)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("G,Hkv,D,B,lens,new", [(2, 2, 128, 3, [200, 129, 500], 1), (2, 2, 64, 3, [200, 129, 500], 1), (12, 1, 128, 2, [300, 140], 1), (1, 2, 128, 2, [3000, 5000], 1),
                                                (4, 8, 64, 80, [180], 1), (2, 2, 128, 2, [300, 150], 3), (4, 1, 64, 2, [2000, 300], 40), (5, 2, 128, 1, [3000], 300)])
def test_scores_below_all_numbers_weigh_nothing(G, Hkv, D, B, lens, new, codes):
    """The first 128 tokens' scores are below the lowest 32-bit number, the others' are 0: these weigh alike, the first nothing.  One token per sequence, and several.  Bound: the
    output's rounding, the weights' to fp16, exponentials and logarithms of scales by 2^-19 of themselves, and sums in 32 bits."""
    lens = (lens * B)[:B]
    counts = [min(new, n - 128) for n in lens]
    c = attention_case(counts, lens, G * Hkv, Hkv, D, 16, torch.bfloat16, codes, seed=D + G)
    q = torch.full_like(c["q"], 2.0 ** 60)
    k_pool, v_pool, k_scale, v_scale = c["cache"]
    raw(k_pool).zero_()
    for b in range(B):
        first = c["tables"][b, :8].long()
        raw(k_pool)[first] = raw(torch.full((1,), -100.0, device=DEV).to(codes))
        k_scale[first] = 2.0 ** 70
    for flags in (0, ops.ATTN_FORCE_GENERIC):
        if new == 1:
            got = ops.paged_decode_attention_q8(q, *c["cache"], c["tables"], i32(lens), max(lens), flags=flags).to(F64)
        else:
            got = ops.paged_prompt_attention_q8(q, *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, max(lens), flags=flags).to(F64)
        for b, n in enumerate(lens):
            pos = torch.arange(128, n, device=DEV)
            at = c["tables"][b].long()[pos // 16]
            v = (raw(v_pool)[at, :, pos % 16].view(codes).to(F64) * v_scale[at][..., None].to(F64)).repeat_interleave(G, 1)
            seen = torch.arange(1, n - 127, device=DEV, dtype=F64)[:, None, None]
            want, A = (v.cumsum(0) / seen)[-counts[b]:], (v.abs().cumsum(0) / seen)[-counts[b]:]
            near(got[c["starts"][b]:c["starts"][b + 1]], want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -18 + (n + 8) * 2.0 ** -24) * A, f"{b}, flags {flags}")


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("Hkv,G,D,bs,cols,new,lens", [(4, 2, 64, 16, 5, [1], [105]), (4, 8, 64, 16, 1, [3, 2], [44, 17]), (1, 4, 64, 48, 3, [4, 1, 3], [160, 300, 147]), (2, 4, 64, 16, 7, [30], [400]),
                                                    (2, 4, 128, 16, 5, [3, 1], [120, 90]), (1, 1, 64, 80, 1, [8, 5], [83, 400])])
def test_tables_that_end_before_the_first_new_token(Hkv, G, D, bs, cols, new, lens, codes):
    """Every row sees all that the table holds and nothing behind it, where that is no whole number of the kernels' tiles too."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        c = attention_case(new, lens, G * Hkv, Hkv, D, bs, dtype, codes, seed=D + cols, cols=cols)
        want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, dtype != torch.float32)
        near(ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), max(new), max(lens)), want, bound, str(dtype))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("power", [-34, -25, 60])
@pytest.mark.parametrize("D,new,lens", [(128, 1, [400, 90]), (64, 1, [400, 90]), (128, 3, [300, 60]), (128, 90, [400, 90]), (64, 200, [1500, 300])])
def test_pages_outside_the_pool_cost_small_and_large_values_nothing(D, new, lens, power, codes):
    """Keys of such pages are zeros and weigh in; the values of the others keep their digits, however small or large their scales are."""
    counts = [min(new, n) for n in lens]
    c = attention_case(counts, lens, 8, 2, D, 16, torch.bfloat16, codes, seed=D + new)
    c["tables"][0, 3], c["tables"][0, 9], c["tables"][1, 1] = -1, 2 ** 30, -5
    c["cache"][3].mul_(2.0 ** power)
    want, bound = attention_reference(c["q"], *c["cache"], c["tables"], lens, c["starts"], D ** -0.5, True)
    if new == 1:
        got = ops.paged_decode_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), max(lens))
    else:
        got = ops.paged_prompt_attention_q8(c["q"], *c["cache"], c["tables"], i32(lens), i32(c["starts"]), new, max(lens))
    near(got, want, bound)
