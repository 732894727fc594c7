"""What the paged engine keeps between calls, without a GPU: its tables and pools on the CPU, a recorder in the place of a pass over trees."""
import types

import pytest
import torch

import dgi_b200  # noqa: F401
from dgi_b200 import engine as E
from dgi_b200.drafting import GREEDY, Sampling
from dgi_b200.paged_layer import PagedBatchState
from dgi_b200.worker.distributed.kv_cache import KVCachePool

MAX_BATCH, BLOCK, PER_SEQ, VOCAB = 4, 4, 8, 50


@pytest.fixture
def engine():
    """A whole model's engine of four sequences of 32 tokens; what would need a GPU (prompts, steps) is not called."""
    e = object.__new__(E.PagedDecodeEngine)
    e.max_batch, e.block_size, e.blocks_per_seq, e.max_seq_len = MAX_BATCH, BLOCK, PER_SEQ, BLOCK * PER_SEQ
    e.device, e.dtype, e.use_cuda_graph, e.logits_log = torch.device("cpu"), torch.float32, True, None
    e.is_first = e.is_last = True
    e.external_head = False
    e.Hq, e.Hkv, e.D = 4, 2, 8
    e.shards = [types.SimpleNamespace(embed_tokens=torch.nn.Embedding(VOCAB, 4))]
    e.pools = [KVCachePool(num_layers=2, num_heads=2, head_dim=8, block_size=BLOCK, max_blocks_per_layer=MAX_BATCH * PER_SEQ, device="cpu", dtype=torch.float32)]
    e.block_tables = torch.zeros((MAX_BATCH, PER_SEQ), dtype=torch.int32)
    e.context_lens = torch.zeros(MAX_BATCH, dtype=torch.int32)
    e.state = PagedBatchState(e.block_tables, e.context_lens, torch.zeros(MAX_BATCH, dtype=torch.int64), BLOCK * PER_SEQ)
    e._seq_blocks, e._host_lens = [None] * MAX_BATCH, [0] * MAX_BATCH
    e._graph = e._graph_chained = e.prefix_index = e._numbers = e.sampling = None
    e._trees, e._borrowed, e.batch = {}, False, 0
    e._temperature, e._top_p, e._min_p = (torch.zeros(MAX_BATCH) for _ in range(3))
    e._top_k = torch.zeros(MAX_BATCH, dtype=torch.int32)
    return e


@pytest.fixture
def passes(monkeypatch):
    """(sequences that the step was made for, nodes, shape of the tokens, how many steps had been made before it) of each pass over trees."""
    made, steps = [], []

    class Step:
        def __init__(self, engine, nodes):
            self.batch, self.nodes, self.number = engine.batch, nodes, len(steps)
            steps.append(nodes)

        def run(self, tokens, parents, lens):
            made.append((self.batch, self.nodes, tuple(tokens.shape), self.number))
            return [0] * tokens.shape[0], [[-1] * self.nodes] * tokens.shape[0]

    monkeypatch.setattr(E, "_TreeStep", Step)
    return made


def adopt(e, n, tokens=9):
    e.adopt_sequences([[pool.allocate_sequence(tokens + 8) for pool in e.pools] for _ in range(n)], [tokens] * n)


def verify(e, nodes=3):
    n = e.batch
    return e.verify_trees(torch.zeros((n, nodes), dtype=torch.int64), torch.full((n, nodes), -1, dtype=torch.int32))


def test_a_pass_over_trees_is_of_its_batch(engine, passes):
    """A step holds buffers and a captured pass of one number of sequences: it serves no other number, whatever single steps were captured for."""
    engine._graph_key = (1, 0)          # a single step of one sequence had been captured
    engine.allocate(4, 20)
    verify(engine)
    adopt(engine, 1)
    verify(engine)
    adopt(engine, 3)
    verify(engine)
    engine._graph_key = (2, 0)
    adopt(engine, 2)
    verify(engine)
    assert [p[:3] for p in passes] == [(n, 3, (n, 3)) for n in (4, 1, 3, 2)]


def test_a_pass_over_trees_is_kept_for_its_batch(engine, passes):
    """Sequences handed over in turn, as many as before: the captured pass serves them, though no single step was captured."""
    for _ in range(3):
        adopt(engine, 2)
        verify(engine)
        verify(engine, 5)
    assert [p[3] for p in passes] == [0, 1] * 3


OWN, CALL = [Sampling(0.9, 0, 1.0, 0.0, 1), GREEDY], [Sampling(1.2, 7, 0.8, 0.1, 2), Sampling(0.5, 0, 1.0, 0.0, 3)]


@pytest.fixture
def told(engine, passes):
    """The settings that the engine's passes found, in turn: temperatures of the first two sequences, None where it decoded greedily."""
    seen = []

    def record(n):
        seen.append(None if engine.sampling is None else engine._temperature[:2].tolist())
        return torch.zeros(n, dtype=torch.int64)

    engine.prefill = lambda prompts: record(len(prompts))
    engine.prefill_chunk = lambda lo, hi, ids, past_len=0: record(hi - lo)
    engine.decode_step = lambda tokens: record(len(tokens))
    engine.prefill_chunk_size = 8
    engine._shared_blocks = engine.cached_blocks = 0

    def verify(tokens, parents, lens):
        n = tokens.shape[0]
        return [1] * n, record(n)[:, None].tolist()

    engine.verify_trees = verify
    return seen


def calls(e, sampling):
    prompts = torch.zeros((2, 5), dtype=torch.int64)
    ask = [{"input_ids": [0] * 5, "max_new_tokens": 3, "do_sample": s.temperature > 0, "temperature": s.temperature} for s in sampling or [GREEDY] * 2]
    return [lambda: e.generate(prompts, 3, sampling=sampling), lambda: e.generate_drafted(prompts, 3, sampling=sampling),
            lambda: e.generate_ragged([[0] * 5, [0] * 6], 3, sampling=sampling), lambda: e.batch_inference(ask)]


@pytest.mark.parametrize("which", range(4))
def test_a_calls_settings_end_with_it(engine, told, which):
    want = [pytest.approx(s.temperature) for s in CALL]
    for own in (None, OWN):
        engine.set_sampling(own)
        buffers = (engine._temperature, engine._top_k, engine._top_p, engine._min_p)
        before = [b.clone() for b in buffers], None if own is None else engine._numbers.clone()
        for sampling in (CALL, None):
            told.clear()
            calls(engine, sampling)[which]()
            assert len(told) >= 3 and all(t == (None if sampling is None else want) for t in told)
            assert engine.sampling == own
            if own is not None:
                assert all(torch.equal(a, b) for a, b in zip(buffers, before[0])) and torch.equal(engine._numbers[:2], before[1][:2])


@pytest.mark.parametrize("which", range(3))
def test_a_calls_settings_end_with_it_when_it_fails(engine, told, which):
    def fails(*a, **kw):
        raise RuntimeError("no room")

    engine.allocate = fails
    for own in (None, OWN):
        engine.set_sampling(own)
        with pytest.raises(RuntimeError, match="no room"):
            calls(engine, CALL)[which]()
        assert engine.sampling == own


def test_settings_that_are_refused_change_nothing(engine, told):
    engine.set_sampling(OWN)
    engine.external_head = True
    with pytest.raises(RuntimeError, match="whole model"):
        engine.generate(torch.zeros((2, 5), dtype=torch.int64), 3, sampling=CALL)
    assert engine.sampling == OWN and not told


def test_settings_as_other_engines_write_no_limit():
    """Requests that were served before their settings counted are served: -1 for no limit of k and for no seed, 0 for the smallest nucleus."""
    ask = {"do_sample": True, "temperature": 0.8, "top_k": 40, "top_p": 0.95, "min_p": 0.05, "seed": 6}
    plain = Sampling(0.8, 40, 0.95, 0.05, 6)
    assert Sampling.of_request(ask) == plain
    assert Sampling.of_request({**ask, "top_k": -1}) == Sampling(0.8, 0, 0.95, 0.05, 6)
    assert Sampling.of_request({**ask, "seed": -1}) == Sampling(0.8, 40, 0.95, 0.05, 0)
    first = Sampling.of_request({**ask, "top_p": 0})        # the order's first is always kept: it alone
    assert first.top_k == 1 and first.temperature > 0
    for bad in (dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=2.0), dict(temperature=-1.0), dict(top_k="many")):
        with pytest.raises(ValueError):
            Sampling.of_request({**ask, **bad})


def test_a_drafter_without_a_draft(engine, told):
    """No tree, or an empty one, is the last token alone: decoding goes on, a token a pass."""
    checked = []
    verify_root = engine.verify_trees

    def verify(tokens, parents, lens):
        checked.append((lens.tolist(), tokens[:, 0].tolist(), parents[:, 0].tolist()))
        assert len(checked) < 10
        return verify_root(tokens, parents, lens)

    engine.verify_trees = verify
    prompts = torch.tensor([[3, 4, 5], [6, 7, 8]])
    for nothing in (None, ([], []), ()):
        checked.clear()
        assert engine.generate_drafted(prompts, 3, lambda told: nothing).tolist() == [[0, 0, 0]] * 2
        assert checked == [([1, 1], [0, 0], [-1, -1])] * 2


def test_a_drafter_whose_root_is_another_token(engine, told):
    """The root stands for the last token, whose keys and values the pass appends: another one would be decoded in its place."""
    with pytest.raises(ValueError, match="root"):
        engine.generate_drafted(torch.tensor([[3, 4, 5]]), 3, lambda told: ([told[-1] + 1, 7], [-1, 0]))
    assert len(told) == 1           # the prompt; no pass over trees
