"""Drawn tokens and drafted tokens through the engines: one model's tokens, whichever way they are decoded."""
import numpy as np
import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200.drafting import GREEDY, PromptLookup, Sampling, pad_trees
from dgi_b200.engine import PagedDecodeEngine
from dgi_b200.testing import build_product_shards
from dgi_b200.worker.engines.paged_engine import PagedLLMEngine
from oracle import llama_ref as L
from test_sample_rows_gpu import token

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def model(golden, ranges=((0, 4),), dtype=torch.float32):
    g = golden("tiny_decode.json")
    cfg = L.RefConfig(**g["config"])
    return g, cfg, build_product_shards(cfg, L.make_weights(cfg, seed=0), list(ranges), DEV, dtype)


class Knowing:
    """Drafts what the sequences will say (`rows`, prompts and answers) with mistakes and other branches in between."""

    def __init__(self, rows, nodes, seed):
        self.rows, self.nodes, self.rng = rows, nodes, np.random.default_rng(seed)

    def __call__(self, told):
        row = next(r for r in self.rows if r[:len(told)] == told)
        tokens, parents, at = [told[-1]], [-1], 0
        for t in row[len(told):]:
            if len(tokens) >= self.nodes - 2 or self.rng.random() < 0.15:
                break
            tokens += [int(self.rng.integers(0, 1000)), t]          # a sibling before it, seldom the same
            parents += [at, at]
            at = len(tokens) - 1
        return tokens, parents


@pytest.mark.parametrize("ranges,graph,fused,nodes", [([(0, 4)], True, False, 8), ([(0, 2), (2, 4)], True, True, 13), ([(0, 4)], False, True, 64),
                                                     ([(0, 4)], True, False, 1)])
def test_drafted_tokens_are_the_reference_tokens(golden, ranges, graph, fused, nodes):
    g, cfg, shards = model(golden, ranges)
    prompts = torch.tensor(g["prompt_ids"])
    rows = [p + t for p, t in zip(g["prompt_ids"], g["tokens"])]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=320, prefill_mode="eager", use_cuda_graph=graph, fuse_projections=fused)
    passes = []
    verify = eng.verify_trees
    eng.verify_trees = lambda *a: passes.append(1) or verify(*a)
    for drafter in (Knowing(rows, nodes, 1), None):
        passes.clear()
        assert eng.generate_drafted(prompts, 64, drafter, nodes=nodes).tolist() == g["tokens"]
        if nodes >= 8 and drafter is not None:
            assert len(passes) < 45          # several tokens a pass
    assert eng.generate(prompts, 64).tolist() == g["tokens"]         # the engine decodes singly as before


def test_trees_and_single_steps_in_turn(golden):
    """A pass over trees between single steps, a sequence that rests, rows of different lengths."""
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), g["tokens"]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=320, prefill_mode="eager")
    eng.allocate(4, prompts.shape[1] + 80)
    told = [[t] for t in eng.prefill(prompts).tolist()]
    for _ in range(3):
        for b, t in enumerate(eng.decode_step(torch.tensor([r[-1] for r in told])).tolist()):
            told[b].append(t)
    know = Knowing([p + t for p, t in zip(g["prompt_ids"], want)], 9, 3)
    trees = [know(g["prompt_ids"][b] + told[b]) for b in range(4)]
    trees[2] = None
    count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees(trees, 9)))
    assert count[2] == 0 and all(count[b] >= 1 for b in (0, 1, 3))
    for b in range(4):
        told[b] += new[b][:count[b]]
        assert told[b] == want[b][:len(told[b])] and eng._host_lens[b] == prompts.shape[1] + len(told[b]) - 1
    for _ in range(4):
        for b, t in enumerate(eng.decode_step(torch.tensor([r[-1] for r in told])).tolist()):
            told[b].append(t)
    assert all(r == w[:len(r)] for r, w in zip(told, want))


SETTINGS = [Sampling(0.9, 0, 1.0, 0.0, 1), Sampling(0.7, 50, 0.9, 0.0, 2), GREEDY, Sampling(1.2, 0, 0.8, 0.02, 3)]


def test_drawn_tokens_follow_the_definition(golden):
    g, cfg, shards = model(golden)
    prompts = torch.tensor(g["prompt_ids"])
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=192, prefill_mode="eager", use_cuda_graph=False)
    eng.logits_log = []
    toks = eng.generate(prompts, 24, sampling=SETTINGS)
    P, numbers = prompts.shape[1], [s.numbers(193) for s in SETTINGS]
    at = {}
    for lo, hi, logits in eng.logits_log:
        for b in range(lo, hi):
            i = at.get(b, 0)
            s = SETTINGS[b]
            assert int(toks[b, i]) == token(logits[b - lo].cpu().numpy(), numbers[b][P + i], s.temperature, s.top_k, s.top_p, s.min_p)
            at[b] = i + 1
    assert set(at.values()) == {24} and toks[2].tolist() == g["tokens"][2][:24]
    assert any(toks[b].tolist() != g["tokens"][b][:24] for b in (0, 1, 3))


def test_drawn_tokens_are_a_requests_own(golden):
    """Alone, in a batch, captured or not, with drafted tokens or without: the same."""
    g, cfg, shards = model(golden)
    prompts = torch.tensor(g["prompt_ids"])
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager")
    want = eng.generate(prompts, 40, sampling=SETTINGS)
    assert eng.generate(prompts[1:2], 40, sampling=SETTINGS[1:2]).tolist() == want[1:2].tolist()
    assert eng.generate(prompts, 40).tolist() == [t[:40] for t in g["tokens"]]
    rows = [p + t for p, t in zip(g["prompt_ids"], want.tolist())]
    for drafter in (Knowing(rows, 8, 5), PromptLookup(8)):
        assert eng.generate_drafted(prompts, 40, drafter, sampling=SETTINGS).tolist() == want.tolist()
    ragged = eng.generate_ragged([g["prompt_ids"][3][:20], g["prompt_ids"][0], g["prompt_ids"][1][:33]], 12, sampling=[SETTINGS[3], SETTINGS[0], SETTINGS[1]])
    assert ragged[1] == want[0, :12].tolist()
    assert ragged[0] == eng.generate(prompts[3:4, :20], 12, sampling=SETTINGS[3:]).tolist()[0]


def test_trees_of_a_16_bit_model_captured_and_not(golden):
    g, cfg, _ = model(golden)
    prompts = torch.tensor(g["prompt_ids"])
    out = []
    for graph in (True, False):
        _, _, shards = model(golden, dtype=torch.bfloat16)
        eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, use_cuda_graph=graph, fuse_projections=True)
        out.append((eng.generate_drafted(prompts, 48, PromptLookup(16, branches=3), nodes=16).tolist(),
                    eng.generate_drafted(prompts, 48, PromptLookup(16), sampling=SETTINGS, nodes=16).tolist()))
    assert out[0] == out[1] and all(len(r) == 48 for r in out[0][0])


@pytest.mark.parametrize("graph", [True, False])
def test_behind_a_shared_prefix_and_steps_on_the_device(golden, graph):
    """Prompts whose first blocks are one sequence's; after a pass over trees steps go on where it ended."""
    g, cfg, shards = model(golden)
    head = g["prompt_ids"][0][:32]
    prompts = torch.tensor([head + p[:9] for p in g["prompt_ids"]])
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager", use_cuda_graph=graph)
    want = eng.generate(prompts, 30)
    rows = [p + t for p, t in zip(prompts.tolist(), want.tolist())]
    eng.allocate(4, prompts.shape[1] + 40, shared_prefix_len=32)
    told = [r + [t] for r, t in zip(prompts.tolist(), eng.prefill(prompts).tolist())]
    know = Knowing(rows, 9, 4)
    for rest in (None, 2):
        trees = [None if b == rest else know(t) for b, t in enumerate(told)]
        count, new = eng.verify_trees(*(torch.from_numpy(x) for x in pad_trees(trees, 9)))
        for b in range(4):
            told[b] += new[b][:count[b]]
    for _ in range(5):
        eng.decode_step_device()
        for b, t in enumerate(eng.next_tokens[:4].tolist()):
            told[b].append(t)
    assert all(t == r[:len(t)] for t, r in zip(told, rows)) and min(map(len, told)) >= prompts.shape[1] + 7


def test_drafts_that_are_no_tokens(golden):
    """Drafted numbers outside the vocabulary and whatever stands behind the last node are not taken, and read nothing."""
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), g["tokens"]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=320, prefill_mode="eager")
    eng.allocate(4, prompts.shape[1] + 20)
    first = eng.prefill(prompts).cpu()
    tokens = torch.full((4, 5), -1, dtype=torch.int64)
    tokens[:, 0] = first
    tokens[0, 1:] = 10 ** 12
    tokens[1, 1] = want[1][1]
    parents = torch.tensor([-1, 0, 1, 0, 90], dtype=torch.int32).expand(4, -1)
    lens = torch.tensor([5, 2, 1, 0])
    with pytest.raises(ValueError, match="root"):
        eng.verify_trees(tokens.roll(1, 1), parents, lens)
    for on in ("cpu", "cuda"):
        count, new = eng.verify_trees(tokens.to(on), parents.to(on), lens)
        assert count == [1, 2, 1, 0]
        assert [r[:n] for r, n in zip(new, count)] == [want[b][1:1 + n] for b, n in enumerate(count)]
        eng.allocate(4, prompts.shape[1] + 20)
        eng.prefill(prompts)


def test_trees_at_the_end_of_the_room(golden):
    g, cfg, shards = model(golden)
    prompts, want = torch.tensor(g["prompt_ids"]), [t[:40] for t in g["tokens"]]
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=prompts.shape[1] + 40, prefill_mode="eager")
    know = Knowing([p + t for p, t in zip(g["prompt_ids"], g["tokens"])], 16, 1)
    assert eng.generate_drafted(prompts, 40, know, nodes=16).tolist() == want
    assert eng.generate_drafted(prompts, 40, nodes=8).tolist() == want
    with pytest.raises(ValueError):
        eng.generate_drafted(prompts, 41, nodes=8)


def test_settings_of_fewer_sequences_than_before(golden):
    g, cfg, shards = model(golden)
    prompts = torch.tensor(g["prompt_ids"])
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=256, prefill_mode="eager")
    want = eng.generate(prompts, 10, sampling=SETTINGS)
    for call in (eng.generate, eng.generate_drafted):
        with pytest.raises(ValueError):
            call(prompts, 10, sampling=SETTINGS[:2])
    eng.set_sampling(SETTINGS)
    with pytest.raises(ValueError):
        eng.set_sampling(SETTINGS * 2)
    assert eng.sampling == SETTINGS
    eng.set_sampling(SETTINGS[:1])      # the others are greedy from now on
    eng.allocate(4, prompts.shape[1] + 10)
    told = [[t] for t in eng.prefill(prompts).tolist()]
    for _ in range(9):
        for row, t in zip(told, eng.decode_step(torch.tensor([r[-1] for r in told])).tolist()):
            row.append(t)
    assert told[0] == want[0].tolist() and told[1:] == [t[:10] for t in g["tokens"][1:]]


def test_refusals(golden):
    g, cfg, shards = model(golden)
    eng = PagedDecodeEngine(shards, max_batch=4, max_seq_len=192, prefill_mode="eager")
    prompts = torch.tensor(g["prompt_ids"])
    eng.allocate(4, prompts.shape[1] + 4)
    eng.prefill(prompts)
    one = torch.zeros((4, 1), dtype=torch.int64)
    for tokens, parents, lens in ((one[:2], one[:2], None), (one, one[:, :0], None), (torch.zeros((4, 65)), torch.zeros((4, 65)), None),
                                  (one, one, torch.tensor([1, 1, 1])), (one, one, torch.tensor([2, 1, 1, 1])), (torch.zeros((4, 40)), torch.zeros((4, 40)), None)):
        with pytest.raises(ValueError):
            eng.verify_trees(tokens, parents, lens)
    with pytest.raises(ValueError):
        eng.generate_ragged([[1, 2], [3]], 4, sampling=SETTINGS)
    with pytest.raises(ValueError):
        eng.set_sampling(SETTINGS * 2)


def test_engine_surface_draws_on_request(golden):
    g, cfg, shards = model(golden)
    e = PagedLLMEngine({"shards": shards, "device": DEV, "dtype": torch.float32, "max_model_len": 192, "max_batch_size": 4, "prefill_mode": "eager"})
    e.load_model()
    ids = g["prompt_ids"][0]
    plain = e.inference({"input_ids": ids, "max_tokens": 12})["output_ids"]
    assert e.inference({"input_ids": ids, "max_tokens": 12, "temperature": 0.9, "top_k": 5})["output_ids"] == plain
    ask = {"input_ids": ids, "max_tokens": 12, "do_sample": True, "temperature": 1.3, "top_p": 0.95, "seed": 7}
    drawn = e.inference(ask)["output_ids"]
    assert drawn != plain and e.inference(ask)["output_ids"] == drawn
    both = e.batch_inference([ask, {"input_ids": ids, "max_tokens": 12}, {"input_ids": ids, "do_sample": True, "top_p": 7.0}])
    assert both[0]["output_ids"] == drawn and both[1]["output_ids"] == plain and isinstance(both[2], ValueError)


def test_step_engine_draws_on_request():
    from test_petipel_gpu import CFG_B, build

    eng, _ = build(CFG_B, bias_rows=7)
    prompts = [[3, 5, 7, 9, 11], [2] * 40, [8, 1]]
    greedy = eng.generate(prompts, 10)
    assert eng.generate(prompts, 10, sampling=[Sampling(1.0, 1, 1.0, 0.0, 4)] * 3) == greedy
    assert eng.generate(prompts, 10, sampling=[GREEDY] * 3) == greedy
    mixed = [Sampling(1.5, 0, 0.95, 0.0, 1), GREEDY, Sampling(2.0, 30, 1.0, 0.0, 2)]
    drawn = eng.generate(prompts, 10, sampling=mixed)
    assert drawn[1] == greedy[1] and drawn != greedy and drawn == eng.generate(prompts, 10, sampling=mixed, prefill_chunk=3)
    assert drawn[2] == eng.generate(prompts[2:], 10, sampling=mixed[2:])[0]
