"""Passes over trees and drawn tokens between other calls of one engine: what a call leaves behind, and what it leaves alone."""
import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import ops
from dgi_b200.drafting import Sampling, pad_trees
from dgi_b200.engine import PagedDecodeEngine
from dgi_b200.testing import build_product_shards
from oracle import llama_ref as L
from test_drafted_decode_gpu import SETTINGS, Knowing, model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def adopt(eng, prompts, room):
    """The prompts in blocks of the caller's own; their first tokens."""
    blocks = [[pool.allocate_sequence(prompts.shape[1] + room) for pool in eng.pools] for _ in range(prompts.shape[0])]
    eng.adopt_sequences(blocks, [0] * prompts.shape[0])
    return blocks, [[t] for t in eng.prefill(prompts).tolist()]


@pytest.mark.parametrize("others", [1, 2])
def test_trees_of_fewer_sequences_than_the_pass_before(golden, others):
    """A step captured for one sequence, a pass over trees of four, then `others` handed over: their tokens, and nobody else's blocks."""
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), g["tokens"]
    rows = [p + t for p, t in zip(g["prompt_ids"], want)]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager", spare_blocks=40)
    assert eng.generate(prompts[:others], 6).tolist() == [t[:6] for t in want[:others]]
    assert eng.generate_drafted(prompts, 20, Knowing(rows, 9, 1), nodes=9).tolist() == [t[:20] for t in want]
    blocks, told = adopt(eng, prompts[2:2 + others], 30)
    slots = []
    for li in range(cfg.num_hidden_layers):
        mine = {blk.slot for seq in blocks for blk in seq[0][li]}
        slots.append([i for i in range(eng.pools[0].layer(li).key_pool.shape[0]) if i not in mine])
    pools = [(eng.pools[0].layer(li).key_pool, eng.pools[0].layer(li).value_pool) for li in range(cfg.num_hidden_layers)]
    before = [[p[s].clone() for p in two] for two, s in zip(pools, slots)]
    know = Knowing(rows, 9, 2)
    for _ in range(3):
        trees = [know(g["prompt_ids"][2 + b] + told[b]) for b in range(others)]
        count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees(trees, 9)))
        assert len(count) == len(new) == others
        for b in range(others):
            told[b] += new[b][:count[b]]
    assert all(torch.equal(x, p[s]) for was, two, s in zip(before, pools, slots) for x, p in zip(was, two))
    assert told == [w[:len(t)] for t, w in zip(told, want[2:])] and min(map(len, told)) >= 4
    assert eng._host_lens == [prompts.shape[1] + len(t) - 1 for t in told] + [0] * (4 - others)
    for _ in range(3):        # single steps go on from there
        eng.decode_step_device()
        for b, t in enumerate(eng.next_tokens[:others].tolist()):
            told[b].append(t)
    assert told == [w[:len(t)] for t, w in zip(told, want[2:])]


def test_trees_of_more_sequences_than_the_pass_before(golden):
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), g["tokens"]
    rows = [p + t for p, t in zip(g["prompt_ids"], want)]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager", spare_blocks=60)
    for n in (1, 4, 2, 2):
        _, told = adopt(eng, prompts[:n], 30)
        know = Knowing(rows, 8, n)
        for _ in range(2):
            count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees([know(g["prompt_ids"][b] + told[b]) for b in range(n)], 8)))
            for b in range(n):
                told[b] += new[b][:count[b]]
        assert told == [w[:len(t)] for t, w in zip(told, want)] and len(told) == n


def single_steps(eng, prompts, n):
    eng.allocate(prompts.shape[0], prompts.shape[1] + n)
    told = [[t] for t in eng.prefill(prompts).tolist()]
    for _ in range(n - 1):
        for row, t in zip(told, eng.decode_step(torch.tensor([r[-1] for r in told])).tolist()):
            row.append(t)
    return told


@pytest.mark.parametrize("graph", [True, False])
def test_a_calls_settings_end_with_it(golden, graph):
    """Behind a call that drew: prompts, single steps, sequences handed over and trees go by the engine's own settings, greedily or not."""
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), [t[:12] for t in g["tokens"]]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager", use_cuda_graph=graph, spare_blocks=60)
    drawn = eng.generate(prompts, 12, sampling=SETTINGS).tolist()
    assert drawn != want and single_steps(eng, prompts, 12) == want
    ask = [{"input_ids": p, "max_new_tokens": 12, "do_sample": True, "temperature": 1.5, "seed": i} for i, p in enumerate(g["prompt_ids"])]
    for call in (lambda: eng.generate_ragged(g["prompt_ids"], 12, sampling=SETTINGS), lambda: eng.generate_drafted(prompts, 12, sampling=SETTINGS),
                 lambda: eng.batch_inference(ask)):
        call()
        _, told = adopt(eng, prompts, 12)
        know = Knowing([p + t for p, t in zip(g["prompt_ids"], g["tokens"])], 8, 1)
        count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees([know(p + t) for p, t in zip(g["prompt_ids"], told)], 8)))
        assert [t + n[:c] for t, n, c in zip(told, new, count)] == [w[:1 + c] for w, c in zip(want, count)]
        eng.release()
    eng.set_sampling(SETTINGS)
    assert eng.generate(prompts, 12).tolist() == want
    assert single_steps(eng, prompts, 12) == drawn
    eng.generate(prompts, 5, sampling=[Sampling(2.0, 0, 1.0, 0.0, 9)] * 4)
    assert single_steps(eng, prompts, 12) == drawn
    eng.set_sampling(None)
    assert single_steps(eng, prompts, 12) == want


TEXT, FROM = 64, 40


def text_model(golden, dtype):
    """A model of 16-bit weights, four texts, and the same weights' logits in 32 bits from token FROM on."""
    g = golden("tiny_decode.json")
    cfg = L.RefConfig(**g["config"])
    sd = {name: w.to(dtype).float() for name, w in L.make_weights(cfg, seed=0).items()}
    texts = torch.tensor(g["prompt_ids"])[:, :TEXT]
    (ref,) = L.build_shards(cfg, sd, [(0, 4)])
    h, _ = ref.forward(texts, position_ids=torch.arange(TEXT)[None].expand(4, -1), use_cache=True)
    shards = build_product_shards(cfg, sd, [(0, 4)], DEV, dtype)
    return PagedDecodeEngine(shards, max_batch=4, max_seq_len=160, fuse_projections=True, use_cuda_graph=False), texts, ref.get_logits(h)[:, FROM:]


def logits_by_steps(eng, texts):
    eng.allocate(len(texts), TEXT + 2)
    eng.prefill(texts[:, :FROM])
    eng.logits_log = []
    for i in range(FROM, TEXT):
        eng.decode_step(texts[:, i])
    out = torch.stack([x for _, _, x in eng.logits_log], 1).cpu()
    eng.logits_log = None
    return out


def logits_by_trees(eng, texts, seed):
    """One pass: the text as one path, other tokens beside it."""
    rng = torch.Generator().manual_seed(seed)
    trees, paths = [], []
    for text in texts.tolist():
        tokens, parents, path = [text[FROM]], [-1], [0]
        for t in text[FROM + 1:]:
            for _ in range(int(torch.randint(0, 3, (1,), generator=rng)) if len(tokens) + 2 + TEXT - FROM - len(path) < 64 else 0):
                tokens.append(int(torch.randint(0, 1024, (1,), generator=rng)))
                parents.append(int(torch.randint(0, len(tokens) - 1, (1,), generator=rng)))
            parents.append(path[-1])
            path.append(len(tokens))
            tokens.append(t)
        trees.append((tokens, parents))
        paths.append(path)
    eng.allocate(len(texts), FROM + 66)
    eng.prefill(texts[:, :FROM])
    seen, head = [], eng.shards[-1].get_logits
    eng.shards[-1].get_logits = lambda h: seen.append(head(h)) or seen[-1]
    try:
        count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees(trees, 64)))
    finally:
        del eng.shards[-1].get_logits
    out = seen[-1].float().cpu()
    assert [r[0] for r in new] == out[:, 0].argmax(-1).tolist()         # the root's answer is always among the new tokens
    return torch.stack([out[b, path] for b, path in enumerate(paths)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_trees_agree_with_single_steps_up_to_rounding(golden, dtype):
    """Single steps and trees, four sequences or one, round at the same places (trees also the softmax's weights, whose half steps average out over the
    keys), but in other orders: logits differ, and no way may be further from 32 bits than single steps are.

    An error is a sum of many roundings: of its mean square a tree's one more rounding takes less than a half, 1.25 of its root; the largest of 10^5
    normal numbers is 4.4 deviations give or take 0.3, so twice the other's is never reached.  Greedy tokens are the same where the two largest logits are further apart than twice
    either side's largest error, four times the single steps'."""
    eng, texts, want = text_model(golden, dtype)
    steps = logits_by_steps(eng, texts) - want
    assert 0 < steps.abs().max() < 0.1 * want.std()
    two = want.topk(2, -1).values
    sure = two[..., 0] - two[..., 1] > 4 * steps.abs().max()
    assert sure.any()
    ways = [logits_by_trees(eng, texts, 1), torch.cat([logits_by_trees(eng, texts[b:b + 1], 2 + b) for b in range(4)]),
            torch.cat([logits_by_steps(eng, texts[b:b + 1]) for b in range(4)])]
    for got in ways:
        off = got - want
        print(f"{dtype}: steps {steps.square().mean().sqrt():.3e} {steps.abs().max():.3e}, here {off.square().mean().sqrt():.3e} {off.abs().max():.3e}; {sure.float().mean():.2f}")
        assert off.square().mean().sqrt() <= 1.25 * steps.square().mean().sqrt()
        assert off.abs().max() <= 2 * steps.abs().max()
        assert torch.equal(got.argmax(-1)[sure], want.argmax(-1)[sure])
    assert torch.equal((steps + want).argmax(-1)[sure], want.argmax(-1)[sure])


def test_an_engines_choice_of_kernels_counts_for_trees(golden, monkeypatch):
    """attn_flags=ATTN_FORCE_GENERIC: no tensor cores in single steps, and none in passes over trees."""
    g = golden("tiny_decode.json")
    cfg = L.RefConfig(**g["config"])
    shards = build_product_shards(cfg, L.make_weights(cfg, seed=0), [(0, 4)], DEV, torch.bfloat16)
    asked, attention = [], ops.paged_tree_attention
    monkeypatch.setattr(ops, "paged_tree_attention", lambda *a, **kw: asked.append(kw.get("flags", 0)) or attention(*a, **kw))
    for flags in (0, ops.ATTN_FORCE_GENERIC):
        eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=160, use_cuda_graph=False, attn_flags=flags)
        asked.clear()
        eng.generate_drafted(torch.tensor(g["prompt_ids"])[:, :30], 3, nodes=4)
        assert asked and set(asked) == {flags}
